"""GPU: the serving operators on other streams than the current one, with work still queued on either."""
from __future__ import annotations

import pytest
import torch

from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").half()


@pytest.fixture
def busy(gpu):
    """Queues some ms of work on the current stream."""
    m = torch.ones((4096, 4096), dtype=torch.float16, device="cuda")
    o = torch.empty_like(m)
    torch.mm(m, m, out=o)
    torch.cuda.synchronize()

    def queue():
        for _ in range(40):
            torch.mm(m, m, out=o)

    return queue


def packed_case():
    q, k, starts = normal(1, 700, 8, 128), normal(2, 700, 2, 128), i32(0, 300, 700)
    return lambda stream=None: (N.packed_attention(q, k, k, starts, 400, 0.1, stream=stream),)


def logprobs_case():
    x, t = normal(3, 64, 30000).float(), torch.arange(64, dtype=torch.int32, device="cuda")
    return lambda stream=None: N.token_logprobs(x, t, 20, stream=stream)


@pytest.mark.parametrize("case,sizes", [
    # the memory that the calls' own tensors may be given, in bytes: outputs and scratch
    (packed_case, [700 * 8 * 128 * 2]), (logprobs_case, [64 * 4, 64 * 4, 64 * 80, 64 * 80]),
], ids=["packed", "logprobs"])
def test_memory_that_queued_work_still_uses(busy, case, sizes):
    """Blocks just let go are read by work queued on the current stream while a call on another stream gets them."""
    call = case()
    want = call()
    if case is logprobs_case:
        sizes = sizes + [N.TokenLogprobs(64, 30000, 20).scratch_bytes]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    kept = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes]
    let_go = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes]
    torch.cuda.synchronize()
    for t in let_go:
        t.fill_(7)
    busy()
    for a, b in zip(kept, let_go):
        a.copy_(b)
    at = {t.data_ptr() for t in let_go}
    t = b = None
    let_go.clear()
    got = call(s)
    assert any(x.data_ptr() in at for x in got)  # the test's point
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in kept)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_views_that_the_default_stream_is_still_to_fill(busy):
    """Stream 0 by its number: the one-call form copies views there, behind the work queued there."""
    q, kc, vc = normal(4, 6, 8, 64), normal(5, 40, 2, 8, 16, 8), normal(6, 40, 2, 64, 16)
    table, masks = torch.arange(39, -1, -1, dtype=torch.int32, device="cuda")[None], torch.tensor(
        [1, 3, 7, 9, 17, 33], device="cuda")
    rest = (i32(601), i32(0, 6), masks, 6, 640, 0.1)
    want = N.tree_attention(q, kc, vc, table, *rest)
    wide, wide_table = torch.zeros((6, 16, 64), dtype=torch.float16, device="cuda"), torch.zeros(
        (1, 80), dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy()
    wide[:, ::2] = q
    wide_table[:, ::2] = table
    with torch.cuda.stream(s):
        out = N.tree_attention(wide[:, ::2], kc, vc, wide_table[:, ::2], *rest, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def tree_inputs():
    q, kc, vc = normal(7, 64, 8, 128), normal(8, 8 * 513, 2, 16, 16, 8), normal(9, 8 * 513, 2, 128, 16)
    table = torch.randperm(8 * 513, device="cuda", dtype=torch.int32).view(8, 513)
    return (q, kc, vc, table, i32(*[8200 - 100 * i for i in range(8)]), i32(*range(0, 65, 8)),
            torch.tensor([(1 << (i % 8 + 1)) - 1 for i in range(64)], device="cuda"))


def tree_node():
    """The partials of 1024 workgroups: 8 sequences x 2 kv heads in 64 partitions."""
    args = tree_inputs()
    return (lambda: N.TreeAttention(8, 64, 8, 8, 2, 128, 16, 513, 8208, 0.1),
            lambda node, outs, stream: node(outs[0], *args, stream=stream), [torch.empty_like(args[0])])


def logprobs_node():
    x, t = normal(3, 64, 30000).float(), torch.arange(64, dtype=torch.int32, device="cuda")
    outs = [torch.empty(64, device="cuda"), torch.empty(64, device="cuda"), torch.empty((64, 20), device="cuda"),
            torch.empty((64, 20), dtype=torch.int32, device="cuda")]
    return (lambda: N.TokenLogprobs(64, 30000, 20), lambda node, outs, stream: node(x, t, *outs, stream=stream), outs)


@pytest.mark.parametrize("case", [tree_node, logprobs_node])
def test_a_new_nodes_scratch_in_memory_that_queued_work_still_uses(busy, case):
    make, call, want = case()
    node = make()
    n, got = node.scratch.numel(), [torch.zeros_like(t) for t in want]
    call(node, want, None)
    node = None
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    kept = torch.zeros(n, dtype=torch.uint8, device="cuda")
    let_go = torch.empty(n, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    let_go.fill_(7)
    busy()
    kept.copy_(let_go)
    at, let_go = let_go.data_ptr(), None
    node = make()
    assert node.scratch_ptr == at  # the test's point
    call(node, got, s)
    torch.cuda.synchronize()
    assert (kept == 7).all()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("given", [True, False], ids=["given stream", "current stream"])
@pytest.mark.parametrize("case", [tree_node, logprobs_node])
def test_a_node_let_go_behind_a_call_on_another_stream(busy, case, given):
    make, call, want = case()
    node = make()
    call(node, want, None)
    n, got = node.scratch.numel(), [torch.zeros_like(t) for t in want]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        busy()
        if not given:
            call(node, got, None)
    if given:
        call(node, got, s)
    at, node = node.scratch_ptr, None
    others = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
    assert all(t.data_ptr() != at for t in others)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", [tree_node, logprobs_node])
def test_a_node_captured_before_any_call(gpu, case):
    """The first call is in a graph, on another stream than the node was made on; then eager ones on more streams."""
    make, call, want = case()
    call(make(), want, None)
    node, got = make(), [torch.zeros_like(t) for t in want]
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        call(node, got, None)
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        other = [torch.zeros_like(t) for t in want]
        torch.cuda.synchronize()
        call(node, other, s)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want))


def tree_one_call():
    args = tree_inputs()
    return lambda stream=None: (N.tree_attention(*args, 8, 8208, 0.1, stream=stream),)


@pytest.mark.parametrize("where", ["current", "number", "forked"])
@pytest.mark.parametrize("case", [packed_case, logprobs_case, tree_one_call])
def test_one_call_forms_captured(gpu, case, where):
    """On the capture's own stream, given as itself or by number, and on one that the capture forks to."""
    call = case()
    want = call()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        if where == "forked":
            side.wait_stream(here)
            got = call(side)
            here.wait_stream(side)
        else:
            got = call(here if where == "current" else here.cuda_stream)
    for _ in range(4):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
