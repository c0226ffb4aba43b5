"""The serving operators' order of allocations, waits and launches on streams, on the CPU: the streams are stand-ins
that write down what is asked of them, and no kernel is launched."""
from __future__ import annotations

import contextlib

import pytest
import torch

from tensorlisp_amd import native as N


class Stream:
    def __init__(self, log, name):
        self.log, self.name = log, name

    def wait_stream(self, other):
        self.log.append(f"{self.name} waits for {other}")

    def __str__(self):
        return self.name


class Library:
    """The library, with the launches written down instead."""

    def __init__(self, real, log):
        self.real, self.log = real, log

    def __getattr__(self, name):
        if name in ("tlh_packed_attention", "tlh_tree_attention", "tlh_token_logprobs"):
            return lambda *a: self.log.append("launch") or 0
        return getattr(self.real, name)


@pytest.fixture
def log(monkeypatch):
    out, lib, empty = [], N.lib(), torch.empty
    monkeypatch.setattr(N, "lib", lambda: Library(lib, out))
    monkeypatch.setattr(N, "_on", lambda device, stream: contextlib.nullcontext(0 if stream is None else stream))
    monkeypatch.setattr(N, "_torch_stream", lambda stream, device: Stream(out, f"stream {stream}"))
    monkeypatch.setattr(N, "_capturing", lambda stream: False, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "the current stream")
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: out.append(f"recorded on {s.name}"))

    def logged(*a, **kw):
        out.append("allocation")
        return empty(*a, **kw)

    monkeypatch.setattr(torch, "empty", logged)
    return out


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def packed(stream, out=None):
    q, k = torch.zeros((4, 8, 64), dtype=torch.float16), torch.zeros((4, 2, 64), dtype=torch.float16)
    N.packed_attention(q, k, k, i32(0, 4), 4, 0.1, out=out, stream=stream)


def logprobs(stream):
    N.token_logprobs(torch.zeros((2, 100)), i32(1, 2), 3, stream=stream)


def tree(stream):
    kc, vc = torch.zeros((5, 2, 8, 16, 8), dtype=torch.float16), torch.zeros((5, 2, 64, 16), dtype=torch.float16)
    N.tree_attention(torch.zeros((3, 8, 64), dtype=torch.float16), kc, vc, torch.zeros((1, 4), dtype=torch.int32), i32(7),
                     i32(0, 3), torch.zeros(3, dtype=torch.int64), 3, 60, 0.1, stream=stream)


@pytest.mark.parametrize("call", [packed, logprobs, tree])
def test_new_tensors_are_used_behind_the_current_streams_work(log, call):
    """What a call allocates comes from the current stream's pool: its memory may still be in use there."""
    call(77)
    wait = log.index("stream 77 waits for the current stream")
    assert wait < log.index("launch") and "allocation" not in log[wait:]


@pytest.mark.parametrize("call", [packed, logprobs, tree])
def test_calls_on_the_current_stream_wait_for_nothing(log, call):
    call(None)
    assert "launch" in log and not [x for x in log if "waits" in x or "recorded" in x]


def test_given_outputs_need_no_wait(log):
    packed(77, out=torch.zeros((4, 8, 64), dtype=torch.float16))
    assert log == ["launch"]


def test_stream_number_zero_is_the_default_stream(monkeypatch):
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: f"the default stream of {device}")
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda n, device=None: f"stream {n} of {device}")
    assert N._torch_stream(0, "cuda:1") == "the default stream of cuda:1"
    assert N._torch_stream(5, "cuda:1") == "stream 5 of cuda:1"


def tree_node():
    kc, vc = torch.zeros((5, 2, 8, 16, 8), dtype=torch.float16), torch.zeros((5, 2, 64, 16), dtype=torch.float16)
    q, node = torch.zeros((3, 8, 64), dtype=torch.float16), N.TreeAttention(1, 3, 3, 8, 2, 64, 16, 4, 60, 0.1, device="cpu")
    args = (torch.zeros((1, 4), dtype=torch.int32), i32(7), i32(0, 3), torch.zeros(3, dtype=torch.int64))
    return lambda stream: node(q, q, kc, vc, *args, stream=stream)


def logprobs_node():
    node, x, t = N.TokenLogprobs(2, 100, 0, torch.float32, device="cpu"), torch.zeros((2, 100)), i32(1, 2)
    return lambda stream: node(x, t, torch.zeros(2), torch.zeros(2), stream=stream)


@pytest.mark.parametrize("make", [tree_node, logprobs_node])
def test_a_nodes_scratch_on_other_streams(log, make):
    """Its memory may still be in use on the stream it was allocated on, which is 0 here, and the allocator must not
    give it away while another stream uses it."""
    call = make()
    del log[:]
    call(None)
    assert log == ["launch"]
    for stream in (77, 78):
        del log[:]
        call(stream)
        assert log == [f"stream {stream} waits for stream 0", f"recorded on stream {stream}", "launch"]
    del log[:]
    call(77), call(78), call(None)
    assert log == ["launch"] * 3
