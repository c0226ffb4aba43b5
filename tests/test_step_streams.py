"""A serving step's operators' order of allocations, waits and launches on streams, on the CPU: the streams are
stand-ins that write down what is asked of them, and no kernel is launched."""
from __future__ import annotations

import pytest
import torch

from tensorlisp_amd import native as N
from test_serving_streams import Stream, i32, log  # noqa: F401 (log: a fixture)

LAUNCHES = ("tlh_chunk_attention", "tlh_head_rope", "tlh_draft_verify")


class Library:
    def __init__(self, real, out):
        self.real, self.out = real, out

    def __getattr__(self, name):
        return (lambda *a: self.out.append("launch") or 0) if name in LAUNCHES else getattr(self.real, name)


@pytest.fixture
def steps(log, monkeypatch):  # noqa: F811
    lib, zeros, full = N.lib(), torch.zeros, torch.full
    monkeypatch.setattr(N, "lib", lambda: Library(lib, log))
    monkeypatch.setattr(torch, "zeros", lambda *a, **kw: log.append("allocation") or zeros(*a, **kw))
    monkeypatch.setattr(torch, "full", lambda *a, **kw: log.append("allocation") or full(*a, **kw))
    return log


def caches():
    return torch.empty((5, 2, 8, 16, 8), dtype=torch.float16), torch.empty((5, 2, 64, 16), dtype=torch.float16)


def chunk_args():
    return (torch.empty((3, 8, 64), dtype=torch.float16), *caches(), torch.empty((1, 4), dtype=torch.int32), i32(7), i32(0, 3))


def verify_args():
    return (torch.empty((3, 100)), torch.empty((2, 100)), i32(1, 2), i32(0, 2), torch.ones(1), torch.ones(2), torch.ones(1))


def chunk(stream):
    N.chunk_attention(*chunk_args(), 3, 60, 0.1, stream=stream)


def verify(stream):
    N.draft_verify(*verify_args(), 2, stream=stream)


@pytest.mark.parametrize("call", [chunk, verify])
def test_new_tensors_are_used_behind_the_current_streams_work(steps, call):
    call(77)
    wait = steps.index("stream 77 waits for the current stream")
    assert wait < steps.index("launch") and "allocation" not in steps[wait:]
    assert any(x == "recorded on stream 77" for x in steps)


@pytest.mark.parametrize("call", [chunk, verify])
def test_calls_on_the_current_stream_wait_for_nothing(steps, call):
    call(None)
    assert "launch" in steps and not [x for x in steps if "waits" in x or "recorded" in x]


def chunk_node():
    args, node = chunk_args(), N.ChunkAttention(1, 3, 3, 8, 2, 64, 16, 4, 60, 0.1, device="cpu")
    return lambda stream: node(args[0], *args, stream=stream)


def verify_node():
    args, node = verify_args(), N.DraftVerify(1, 2, 2, 100, device="cpu")
    outs = torch.empty(1, dtype=torch.int32), torch.empty((1, 3), dtype=torch.int32)
    return lambda stream: node(*args, *outs, stream=stream)


@pytest.mark.parametrize("make", [chunk_node, verify_node])
def test_a_nodes_scratch_on_other_streams(steps, make):
    """A chunk node's counters are cleared on the stream it was made on, too: others wait for that one."""
    call = make()
    del steps[:]
    call(None)
    assert steps == ["launch"]
    for stream in (77, 78):
        del steps[:]
        call(stream)
        assert steps == [f"stream {stream} waits for stream 0", f"recorded on stream {stream}", "launch"]
    del steps[:]
    call(77), call(78), call(None)
    assert steps == ["launch"] * 3


def test_heads_on_another_stream_have_nothing_of_their_own(steps):
    q, k, f = torch.empty((3, 8, 64)), torch.empty((3, 2, 64)), torch.ones(32)
    node, out = N.HeadRope(8, 2, 64, f), torch.empty((3, 8, 64), dtype=torch.float16)
    del steps[:]
    node(q, k, k, i32(0, 1, 2), out, stream=77)
    assert steps == ["launch"]


@pytest.mark.parametrize("captured", [True, False])
def test_a_chunk_node_made_in_a_capture(steps, monkeypatch, captured):
    """Its counters are cleared in the graph: a call on another stream comes behind that, and one outside is refused."""
    monkeypatch.setattr(N, "_capturing", lambda stream: captured)
    call = chunk_node()
    node = call.__closure__[1].cell_contents
    node._captured = True
    del steps[:]
    if captured:
        call(77)
        assert steps[0] == "stream 77 waits for stream 0" and steps[-1] == "launch"
    else:
        with pytest.raises(ValueError, match="for calls in that graph"):
            call(77)
        assert steps == []


def test_every_captured_call_clears_its_counters(steps, monkeypatch):
    """Of a node made in a capture: another graph may be captured with it, and be the one that is replayed first."""
    monkeypatch.setattr(N, "_capturing", lambda stream: True)
    args, node = chunk_args(), N.ChunkAttention(1, 3, 3, 8, 2, 64, 16, 8192, 131072, 0.1, device="cpu")
    args = (*args[:3], torch.empty((1, 8192), dtype=torch.int32), *args[4:])
    node._captured = True
    for stream in (None, 77, 0):
        node.scratch.fill_(255)
        node(args[0], *args, stream=stream)
        assert steps[-1] == "launch" and (node.scratch[:N.CHUNK_COUNTER_BYTES] == 0).all()
        assert (node.scratch[N.CHUNK_COUNTER_BYTES:] == 255).all()
