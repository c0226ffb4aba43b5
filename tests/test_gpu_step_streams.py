"""GPU: a serving step's operators on other streams than the current one, with work still queued on either, and in
graphs."""
from __future__ import annotations

import pytest
import torch

from tensorlisp_amd import native as N
from test_gpu_serving_streams import busy, i32, normal  # noqa: F401 (busy: a fixture)

pytestmark = pytest.mark.gpu


def chunk_args():
    """Decoding sequences over long contexts, whose partitions are joined, and a piece of a prompt."""
    new = [1, 1, 1, 90, 1, 1, 1, 1]
    q, kc, vc = normal(7, sum(new), 8, 128), normal(8, 8 * 513, 2, 16, 16, 8), normal(9, 8 * 513, 2, 128, 16)
    table = torch.randperm(8 * 513, generator=torch.Generator().manual_seed(1)).int().cuda().view(8, 513)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return q, kc, vc, table, i32(*[8200 - 100 * i for i in range(8)]), i32(*starts)


def chunk_node():
    args = chunk_args()
    return (lambda: N.ChunkAttention(8, 97, 90, 8, 2, 128, 16, 513, 8208, 0.1),
            lambda node, outs, stream: node(outs[0], *args, stream=stream), [torch.empty_like(args[0])])


def verify_args():
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda n: torch.rand(n, generator=g, device="cuda")  # noqa: E731
    return (normal(3, 48, 30000).float(), normal(4, 32, 30000).float(), torch.arange(32, dtype=torch.int32, device="cuda"),
            i32(*range(0, 33, 2)), torch.full((16,), 0.8, device="cuda"), rand(32) * 1e-3, rand(16))


def verify_node():
    args = verify_args()
    outs = [torch.empty(16, dtype=torch.int32, device="cuda"), torch.empty((16, 3), dtype=torch.int32, device="cuda"),
            torch.empty(32, device="cuda")]
    return lambda: N.DraftVerify(16, 32, 2, 30000), lambda node, outs, stream: node(*args, *outs, stream=stream), outs


def chunk_one_call():
    args = chunk_args()
    return lambda stream=None: (N.chunk_attention(*args, 90, 8208, 0.1, stream=stream),)


def verify_one_call():
    args = verify_args()
    return lambda stream=None: N.draft_verify(*args, 2, stream=stream)


NODES, CALLS = [chunk_node, verify_node], [chunk_one_call, verify_one_call]


@pytest.mark.parametrize("call,node", zip(CALLS, NODES))
def test_memory_that_queued_work_still_uses(busy, call, node):  # noqa: F811
    """Blocks just let go are read by work queued on the current stream while a call on another stream gets them."""
    call, sizes = call(), [node()[0]().scratch.numel()]
    want = call()
    sizes += [t.numel() * t.element_size() for t in want]
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


@pytest.mark.parametrize("case", NODES)
def test_a_new_nodes_scratch_in_memory_that_queued_work_still_uses(busy, case):  # noqa: F811
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
@pytest.mark.parametrize("case", NODES)
def test_a_node_let_go_behind_a_call_on_another_stream(busy, case, given):  # noqa: F811
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


@pytest.mark.parametrize("case", NODES)
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


@pytest.mark.parametrize("where", ["current", "forked"])
def test_a_chunk_node_made_in_the_graph(gpu, where):
    make, call, want = chunk_node()
    call(make(), want, None)
    got, graph, side = [torch.zeros_like(t) for t in want], torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        if where == "forked":
            side.wait_stream(here)
        node = make()
        call(node, got, side if where == "forked" else None)
        if where == "forked":
            here.wait_stream(side)
    with pytest.raises(ValueError, match="for calls in that graph"):
        call(node, got, None)
    for _ in range(4):
        got[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("where", ["current", "number", "forked"])
@pytest.mark.parametrize("case", CALLS)
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


@pytest.mark.parametrize("case", NODES)
def test_two_nodes_at_once(gpu, case):
    """Each with its own scratch, on a stream each; the graphs of both replayed side by side."""
    make, call, want = case()
    call(make(), want, None)
    nodes, streams = [make(), make()], [torch.cuda.Stream(), torch.cuda.Stream()]
    gots, graphs = [[torch.zeros_like(t) for t in want] for _ in nodes], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    torch.cuda.synchronize()
    for _ in range(5):
        for node, got, s in zip(nodes, gots, streams):
            call(node, got, s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in gots for a, b in zip(got, want))
    for node, got, graph in zip(nodes, gots, graphs):
        with torch.cuda.graph(graph):
            for _ in range(3):
                call(node, got, None)
    for _ in range(4):
        for got in gots:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for got in gots for a, b in zip(got, want))


@pytest.mark.parametrize("where", ["current", "forked"])
def test_a_chunk_node_made_in_one_graph_and_called_in_another(gpu, where):
    """The second graph is replayed first, over counters that hold anything; then both in turn."""
    make, call, want = chunk_node()
    call(make(), want, None)
    gots, graphs, side = [[torch.zeros_like(t) for t in want] for _ in range(2)], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], torch.cuda.Stream()
    node = None
    torch.cuda.synchronize()
    for got, graph in zip(gots, graphs):
        with torch.cuda.graph(graph):
            here = torch.cuda.current_stream()
            if where == "forked":
                side.wait_stream(here)
            node = make() if node is None else node
            call(node, got, side if where == "forked" else None)
            if where == "forked":
                here.wait_stream(side)
    node.scratch.fill_(0xff)
    torch.cuda.synchronize()
    for _ in range(3):
        for got, graph in zip(gots[::-1], graphs[::-1]):
            got[0].zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0])
