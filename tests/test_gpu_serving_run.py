"""GPU: the serving operators together, as a server that drafts trees uses them.

Prompts are attended packed and written to the cache; a sequence is forked with its last
page copied; trees of drafted tokens are written behind the committed ones and verified by
tree attention; the accepted branch is kept and the cache closed; a later step over the
closed cache gives what it gives over a cache that held the accepted tokens from the start.
The log probabilities of the accepted tokens come from the verified rows' logits.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from serving_refs import packed_reference, random_tree, signed
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu
H, KV, D, BS, LAYERS, VOCAB = 8, 2, 128, 16, 3, 5000


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def slots(table, s, positions):
    return torch.tensor([int(table[s, p // BS]) * BS + p % BS for p in positions], dtype=torch.int64, device="cuda")


def test_prompt_fork_draft_verify_keep(gpu):
    r, g = np.random.default_rng(90), torch.Generator(device="cuda").manual_seed(90)
    f16 = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731
    lens, scale = [37, 5, 64], D ** -0.5
    blocks, width = 40, 8
    table = r.permutation(blocks)[:4 * width].reshape(4, width)
    kcs = [torch.full((blocks, KV, D // 8, BS, 8), float("nan"), dtype=torch.float16, device="cuda") for _ in range(LAYERS)]
    vcs = [torch.full((blocks, KV, D, BS), float("nan"), dtype=torch.float16, device="cuda") for _ in range(LAYERS)]
    pools = N.KVPools(kcs, vcs, KV, D, BS)

    def write(layer, k, v, s, positions):
        N.reshape_and_cache(k.reshape(len(positions), -1).contiguous(), v.reshape(len(positions), -1).contiguous(),
                            kcs[layer], vcs[layer], slots(table, s, positions), KV, BS)

    # prompts
    starts = [0] + [int(x) for x in np.cumsum(lens)]
    ks, vs = [], []
    for layer in range(LAYERS):
        rows = f16(starts[-1], (H + 2 * KV) * D)
        q, k, v = rows.split([H * D, KV * D, KV * D], 1)
        q, k, v = q.unflatten(1, (H, D)), k.unflatten(1, (KV, D)), v.unflatten(1, (KV, D))
        out = N.packed_attention(q, k, v, i32(starts), max(lens), scale)
        want, tol = packed_reference(q, k, v, starts, scale, torch.float16)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        for s, n in enumerate(lens):
            write(layer, k[starts[s]:starts[s + 1]], v[starts[s]:starts[s + 1]], s, range(n))
        ks.append([k[starts[s]:starts[s + 1]].clone() for s in range(3)])
        vs.append([v[starts[s]:starts[s + 1]].clone() for s in range(3)])

    # sequence 3 forks sequence 0: whole pages shared, the last one copied
    lens.append(lens[0])
    last = lens[0] // BS
    table[3, :last] = table[0, :last]
    pools.copy_blocks(torch.tensor([[int(table[0, last]), int(table[3, last])]], device="cuda"))
    for layer in range(LAYERS):
        ks[layer].append(ks[layer][0].clone())
        vs[layer].append(vs[layer][0].clone())

    # two rounds of drafts: trees of different sizes behind each sequence
    for step in range(2):
        drafts = [int(x) for x in r.integers(1, 12, 4)]
        trees = [random_tree(r, n) for n in drafts]
        keep = [t[int(r.integers(0, n))] for t, n in zip(trees, drafts)]  # a token and its ancestors
        dstarts = [0] + [int(x) for x in np.cumsum(drafts)]
        context = [n + d for n, d in zip(lens, drafts)]
        args = (i32(table), i32(context), i32(dstarts), signed([m for t in trees for m in t]).cuda())
        node = N.TreeAttention(4, dstarts[-1], max(drafts), H, KV, D, BS, width, max(context), scale)
        for layer in range(LAYERS):
            q, dk, dv = f16(dstarts[-1], H, D), f16(dstarts[-1], KV, D), f16(dstarts[-1], KV, D)
            for s in range(4):
                a, b = dstarts[s], dstarts[s + 1]
                write(layer, dk[a:b], dv[a:b], s, range(lens[s], context[s]))
            out = node(torch.empty_like(q), q, kcs[layer], vcs[layer], *args)
            for s in range(4):
                a = dstarts[s]
                for i, m in enumerate(trees[s]):  # each row: the tokens it sees, gathered
                    seen = [j for j in range(drafts[s]) if m >> j & 1]
                    k = torch.cat([ks[layer][s], dk[a:][seen]])
                    v = torch.cat([vs[layer][s], dv[a:][seen]])
                    qq = torch.cat([torch.zeros((len(k) - 1, H, D), device="cuda").half(), q[a + i:a + i + 1]])
                    want, tol = packed_reference(qq, k, v, [0, len(k)], scale, torch.float16)
                    assert ((out[a + i].cpu().double() - want[-1]).abs() <= tol[-1]).all(), (step, layer, s, i)
                kept = [j for j in range(drafts[s]) if keep[s] >> j & 1]
                ks[layer][s] = torch.cat([ks[layer][s], dk[a:][kept]])
                vs[layer][s] = torch.cat([vs[layer][s], dv[a:][kept]])

        # the drafted tokens' log probabilities
        logits, tokens = f16(dstarts[-1], VOCAB).float(), torch.randint(0, VOCAB, (dstarts[-1],), generator=g, device="cuda")
        lp, ent, tl, ti = N.token_logprobs(logits, tokens.int(), 4)
        ref = torch.log_softmax(logits.double(), 1)
        assert (lp.double() - ref.gather(1, tokens[:, None])[:, 0]).abs().max() < 1e-5
        assert torch.equal(ti.long(), torch.topk(logits, 4)[1])

        new = torch.empty(4, dtype=torch.int32, device="cuda")
        pools.compact(args[0], args[1], args[2], signed(keep).cuda(), new, max(drafts))
        lens = new.tolist()
        assert lens == [len(k) for k in ks[0]]
        for layer in range(LAYERS):
            for s, n in enumerate(lens):
                at = slots(table, s, range(n))
                assert torch.equal(kcs[layer][at // BS, :, :, at % BS].reshape(n, KV, D), ks[layer][s])
                assert torch.equal(vcs[layer][at // BS, :, :, at % BS].reshape(n, KV, D), vs[layer][s])


def test_a_captured_verify_step(gpu):
    """Write, verify, score and keep in one graph, replayed on other inputs."""
    g = torch.Generator(device="cuda").manual_seed(91)
    blocks, n, context = 12, 6, [40, 9]
    kc = torch.randn((blocks, KV, D // 8, BS, 8), generator=g, device="cuda").half()
    vc = torch.randn((blocks, KV, D, BS), generator=g, device="cuda").half()
    table = np.arange(12).reshape(2, 6)[:, ::-1].copy()
    k, v, q = (torch.randn((2 * n, w, D), generator=g, device="cuda").half() for w in (KV, KV, H))
    logits = torch.randn((2 * n, VOCAB), generator=g, device="cuda")
    tokens = torch.arange(2 * n, dtype=torch.int32, device="cuda")
    trees = [[1, 3, 5, 11, 17, 33], [1, 2, 6, 8, 24, 34]]
    masks, keep = signed(trees[0] + trees[1]).cuda(), signed([11, 24]).cuda()
    sl = torch.cat([slots(table, s, range(c, c + n)) for s, c in enumerate(context)])
    lens, starts, tab = i32([c + n for c in context]), i32([0, n, 2 * n]), i32(table)
    node, lpn = N.TreeAttention(2, 2 * n, n, H, KV, D, BS, 6, 60, 0.1), N.TokenLogprobs(2 * n, VOCAB, 3)
    pools = N.KVPools([kc], [vc], KV, D, BS)

    def step(out, new, lps):
        N.reshape_and_cache(k.reshape(2 * n, -1), v.reshape(2 * n, -1), kc, vc, sl, KV, BS)
        node(out, q, kc, vc, tab, lens, starts, masks)
        lpn(logits, tokens, *lps)
        pools.compact(tab, lens, starts, keep, new, n)

    def buffers():
        f = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        return (torch.zeros_like(q), torch.zeros(2, dtype=torch.int32, device="cuda"),
                [f(2 * n), f(2 * n), f(2 * n, 3), torch.zeros((2 * n, 3), dtype=torch.int32, device="cuda")])

    got, want = buffers(), buffers()
    step(*got)  # everything loaded before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*got)
    for _ in range(4):
        for t in (q, k, v, logits):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        kc0, vc0 = kc.clone(), vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        kc1, vc1 = kc.clone(), vc.clone()
        kc.copy_(kc0), vc.copy_(vc0)
        step(*want)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
        assert torch.equal(kc1, kc) and torch.equal(vc1, vc)


def test_two_nodes_at_once(gpu):
    """Two nodes of their own scratch on two streams, and a node used from the stream it is given."""
    g = torch.Generator(device="cuda").manual_seed(92)
    ins, nodes, alone = [], [], []
    for i in range(2):
        kc = torch.randn((300, KV, D // 8, BS, 8), generator=g, device="cuda").half()
        vc = torch.randn((300, KV, D, BS), generator=g, device="cuda").half()
        q = torch.randn((8, H, D), generator=g, device="cuda").half()
        ins.append((q, kc, vc, i32([np.arange(300)]), i32([4700 + i]), i32([0, 8]),
                    signed([(1 << (j + 1)) - 1 for j in range(8)]).cuda()))
        nodes.append(N.TreeAttention(1, 8, 8, H, KV, D, BS, 300, 4800, 0.1))
        alone.append(nodes[i](torch.empty_like(q), *ins[i]))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.zeros_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            nodes[i](outs[i], *ins[i], stream=streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_streams_given_by_number(gpu):
    """A hipStream_t as a number, as the other entry points take it."""
    g = torch.Generator(device="cuda").manual_seed(93)
    q = torch.randn((40, H, D), generator=g, device="cuda").half()
    k = torch.randn((40, KV, D), generator=g, device="cuda").half()
    x, t = torch.randn((3, 9000), generator=g, device="cuda"), i32([1, 2, 3])
    kc = torch.randn((8, KV, D // 8, BS, 8), generator=g, device="cuda").half()
    vc = torch.randn((8, KV, D, BS), generator=g, device="cuda").half()
    tree = (q[:4], kc, vc, i32([[3, 1, 7]]), i32([44]), i32([0, 4]), signed([1, 3, 7, 15]).cuda(), 4, 48, 0.1)
    want = (N.packed_attention(q, k, k, i32([0, 40]), 40, 0.1), N.tree_attention(*tree), *N.token_logprobs(x, t, 3))
    starts = i32([0, 40])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream):
        got = (N.packed_attention(q, k, k, starts, 40, 0.1, stream=stream), N.tree_attention(*tree, stream=stream),
               *N.token_logprobs(x, t, 3, stream=stream))
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
