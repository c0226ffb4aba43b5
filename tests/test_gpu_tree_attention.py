"""GPU: attention of drafted trees over a paged cache (tlh_tree_attention) against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from serving_refs import (attend, chain_masks, one_large_and_many_tiny, pools, random_tree, signed, tables, tiny_bound,
                          tree_reference)
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def build(heads, kv, hs, bs, contexts, drafts, seed, masks=None, width=None):
    """contexts: committed tokens; the drafted ones follow in the cache."""
    r, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    lens = [c + d for c, d in zip(contexts, drafts)]
    table, blocks = tables(r, lens, bs, width=width)
    kc, vc = pools(g, blocks, kv, hs, bs)
    starts = [0] + [int(n) for n in np.cumsum(drafts)]
    if masks is None:
        masks = [m for n in drafts for m in random_tree(r, n)]
    q = torch.randn((starts[-1], heads, hs), generator=g).half()
    return dict(q=q, kc=kc, vc=vc, table=table, lens=lens, starts=starts, masks=masks, scale=hs ** -0.5)


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def run(c, max_drafts=None, max_context=None, out=None, stream=None):
    drafts = [b - a for a, b in zip(c["starts"][:-1], c["starts"][1:])]
    rows, heads, hs = c["q"].shape
    node = N.TreeAttention(len(c["lens"]), rows, max_drafts or max(max(drafts), 1), heads, c["vc"].shape[1], hs,
                           c["vc"].shape[3], c["table"].shape[1], max_context or max(max(c["lens"]), 1), c["scale"])
    out = torch.full((rows, heads, hs), 7.0, dtype=torch.float16, device="cuda") if out is None else out
    node(out, c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), i32(c["starts"]),
         signed(c["masks"]).cuda(), stream)
    torch.cuda.synchronize()
    return out


def check(out, c, rows=slice(None)):
    want, tol = tree_reference(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c["masks"], c["scale"])
    got = out.cpu().double()[rows]
    err = (got - want[rows]).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol[rows]).all(), float((err / tol[rows]).max())


CASES = [
    # heads, kv heads, head size, block size, committed tokens, drafted tokens
    (8, 2, 128, 16, [70], [1]), (8, 2, 128, 16, [600], [7]), (32, 8, 128, 16, [0, 1, 15, 16, 17, 255], [3, 1, 2, 8, 5, 6]),
    (4, 1, 64, 8, [33, 5, 130], [5, 64, 9]), (8, 8, 128, 16, [300, 41], [64, 33]), (64, 8, 128, 16, [100], [63]),
    (8, 1, 64, 32, [500, 31], [17, 4]), (6, 2, 80, 32, [77, 9], [11, 2]), (5, 1, 96, 8, [129], [13]),
    (4, 2, 112, 16, [64, 200], [16, 32]), (4, 2, 192, 16, [90, 300], [7, 40]), (4, 1, 256, 32, [333, 0], [64, 64]),
    (4, 4, 256, 8, [50], [3]), (28, 4, 128, 16, [1100, 3], [9, 21]), (8, 2, 128, 16, [5000, 17, 2049], [4, 30, 8]),
    (32, 32, 64, 16, [40] * 9, [2] * 9), (12, 2, 128, 32, [700], [50]), (48, 1, 128, 16, [260], [2]),
]


@pytest.mark.parametrize("heads,kv,hs,bs,contexts,drafts", CASES)
def test_against_64_bits(gpu, heads, kv, hs, bs, contexts, drafts):
    c = build(heads, kv, hs, bs, contexts, drafts, 20 + heads + hs + bs + sum(drafts))
    check(run(c), c)


def test_one_token_is_the_decode_step(gpu):
    """A chain of one drafted token is paged attention's decode step (its own sum carries + 1e-6)."""
    c = build(32, 8, 128, 16, [99, 700, 1500], [1, 1, 1], 31)
    got = run(c)
    want = N.paged_attention(c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), 16,
                             max(c["lens"]), c["scale"], 8)
    _, tol = tree_reference(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c["masks"], c["scale"])
    assert ((got - want).abs().cpu().double() <= 2 * tol + 1e-6 * want.abs().cpu().double()).all()


def test_a_chain_over_nothing_is_a_prompt(gpu):
    """A chain of n tokens with no context: the packed prompt's attention."""
    c = build(8, 2, 128, 16, [0, 0], [50, 64], 32, masks=chain_masks(50) + chain_masks(64))
    check(run(c), c)


@pytest.mark.parametrize("context", [0, 130])
def test_masks_that_leave_rows_little_or_nothing(gpu, context):
    """Masks need not hold the row's own token: a row may see the context alone, or nothing (zeros)."""
    masks = [0, 1, 0, (1 << 5) - 1, 1 << 4, 0]
    c = build(8, 2, 64, 16, [context], [6], 33, masks=masks)
    out = run(c)
    check(out, c)
    if context == 0:
        assert (out[[0, 2, 5]] == 0).all()
    c = build(8, 2, 64, 16, [context], [64], 34, masks=[1 << 63 | i for i in range(64)])
    check(run(c), c)


def test_rows_behind_the_last_sequence_and_past_max_drafts(gpu):
    c = build(8, 2, 128, 16, [40, 90], [5, 6], 35)
    c["q"] = torch.cat([c["q"], c["q"]])
    c["masks"] = c["masks"] + c["masks"]
    out = run(c)
    check(out, c, slice(0, 11))
    assert (out[11:] == 7).all()
    # no more than max_drafts rows of a sequence, the last max_drafts places of its cache being theirs
    c = build(8, 2, 128, 16, [40, 90], [5, 3], 36, masks=[m for n in (5, 3) for m in chain_masks(n)])
    out = run(c, max_drafts=3)
    check(out, c, slice(5, 8))
    assert (out[3:5] == 7).all()


def test_contexts_shorter_than_their_drafts(gpu):
    """Drafted tokens at negative places are not there; a length below zero is zero."""
    c = build(8, 2, 128, 16, [40, 40, 40], [5, 6, 4], 37)
    c["lens"] = [3, 0, 44]
    check(run(c, max_context=48), c)
    c["lens"] = [3, -9, 44]
    out = run(c, max_context=48)
    assert (out[5:11] == 0).all()
    c["lens"] = [1, 0, 44]
    check(run(c, max_context=48), {**c, "lens": [1, 0, 44]})


def test_lengths_past_the_maximum_are_the_maximum(gpu):
    c = build(8, 2, 64, 16, [60], [4], 38)
    c["lens"] = [1000000]
    out = run(c, max_context=50)
    check(out, {**c, "lens": [50]})


@pytest.mark.parametrize("page", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_pages_outside_the_pools_are_not_seen(gpu, page):
    c = build(8, 2, 128, 16, [200, 40], [6, 40], 39)
    c["table"][0, 3], c["table"][0, 12], c["table"][1, 3] = page, page, page
    check(run(c), c)
    c["table"][1, :] = page  # nothing left
    out = run(c)
    check(out, c)
    assert (out[6:] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hs,bs", [(128, 16), (64, 8), (256, 32)])
def test_what_is_not_seen_does_not_reach_a_row(gpu, hs, bs, bad):
    """Slots past the context, the rest of the pool, and a rejected branch that is not finite."""
    c = build(8, 2, hs, bs, [37, 5], [6, 3], 40, masks=[1, 3, 5, 9, 25, 33, 1, 2, 5])
    for s, L in enumerate(c["lens"]):
        page, off = c["table"][s, (L - 1) // bs], (L - 1) % bs + 1
        c["kc"][page, :, :, off:] = bad
        c["vc"][page, :, :, off:] = bad
    used = {int(c["table"][s, i]) for s, L in enumerate(c["lens"]) for i in range(-(-L // bs))}
    for b in set(range(c["kc"].shape[0])) - used:
        c["kc"][b], c["vc"][b] = bad, bad
    check(run(c), c)
    clean = run(c)
    p = c["lens"][0] - 6 + 3  # drafted token 3 of sequence 0: rows 3 and 4 see it
    c["kc"][c["table"][0, p // bs], :, :, p % bs] = bad
    c["vc"][c["table"][0, p // bs], :, :, p % bs] = bad
    out = run(c)
    others = [0, 1, 2, 5, 6, 7, 8]
    assert torch.isfinite(out[others]).all()
    check(out, c, others)
    assert (out[others].double() - clean[others].double()).abs().max() <= 2.0 ** -8
    assert not torch.isfinite(out[3:5]).all(-1).any()


def test_sharp_scores(gpu):
    c = build(8, 2, 128, 16, [300], [20], 41)
    c["q"] = c["q"] * 20
    check(run(c), c)


def test_a_pool_past_32_bits(gpu):
    """Pages more than 2^32 bytes into the pools."""
    kv, hs, bs = 8, 128, 16
    blocks = (1 << 32) // (kv * hs * bs * 2) + 40
    c = build(8, kv, hs, bs, [90], [5], 42)
    n = c["kc"].shape[0]
    kc = torch.empty((blocks, kv, hs // 8, bs, 8), dtype=torch.float16, device="cuda")
    vc = torch.empty((blocks, kv, hs, bs), dtype=torch.float16, device="cuda")
    kc[-n:], vc[-n:] = c["kc"].cuda(), c["vc"].cuda()
    out = N.tree_attention(c["q"].cuda(), kc, vc, i32(c["table"] + blocks - n), i32(c["lens"]), i32(c["starts"]),
                           signed(c["masks"]).cuda(), 5, 95, c["scale"])
    check(out, c)


def test_wide_block_table_and_page_shared_by_sequences(gpu):
    """Two sequences with a common prefix read the same pages."""
    c = build(8, 2, 128, 16, [64, 64], [4, 7], 43, width=40)
    c["table"][1, :4] = c["table"][0, :4]
    check(run(c), c)


def test_the_same_result_every_time_and_a_used_scratch(gpu):
    c = build(32, 8, 128, 16, [3000, 10], [8, 3], 44)
    a = run(c)
    assert torch.equal(a, run(c))
    # one node for the largest batch, its scratch full of another call's partials
    node = N.TreeAttention(2, 11, 8, 32, 8, 128, 16, c["table"].shape[1], 3008, c["scale"])
    node.scratch.fill_(0xff)
    args = (c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), i32(c["starts"]),
            signed(c["masks"]).cuda())
    for _ in range(2):
        assert torch.equal(a, node(torch.empty_like(a), *args))


def test_on_another_stream_and_captured(gpu):
    c = build(32, 8, 128, 16, [1000, 300], [7, 30], 45)
    want = run(c)
    s = torch.cuda.Stream()
    dev = (c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), i32(c["starts"]),
           signed(c["masks"]).cuda())
    torch.cuda.synchronize()
    got = N.tree_attention(*dev, 30, 1007, c["scale"], stream=s)
    s.synchronize()
    # another split of the context (max_context_len) may add in another order
    want2 = N.tree_attention(*dev, 30, 1007, c["scale"])
    torch.cuda.synchronize()
    assert torch.equal(got, want2)
    check(got, c)
    node = N.TreeAttention(2, 37, 30, 32, 8, 128, 16, c["table"].shape[1], 1007, c["scale"])
    out = torch.zeros_like(want)
    node(out, *dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        node(out, *dev)
    for i in range(4):
        dev[0].copy_(torch.randn_like(dev[0]))
        dev[4].copy_(i32([1007 - 100 * i, 330]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, node(torch.zeros_like(out), *dev))


def test_nothing_to_do(gpu):
    c = build(8, 2, 128, 16, [40, 7], [4, 0], 46)
    check(run(c), c)
    c["starts"] = [0, 0, 0]
    assert (run(c, max_drafts=4) == 7).all()


# --------------------------------------------------- many rows share tiles
# more than 64 rows of a kv head (drafted tokens x group) and at least 512 workgroups
# of 128 rows: the form whose four waves read one tile from LDS
def shared_case(hs, bs, seed, contexts=(0, 5, 150, 64, 33, 1, 97, 40), drafts=(40, 1, 33, 64, 7, 40, 0, 35), **kw):
    n = 512 // (32 * len(contexts))
    return build(64, 32, hs, bs, list(contexts) * n, list(drafts) * n, seed, **kw)


@pytest.mark.parametrize("hs,bs", [(128, 16), (64, 8), (256, 32), (80, 16), (112, 32), (192, 8), (96, 8), (64, 32)])
def test_many_rows_against_64_bits(gpu, hs, bs):
    c = shared_case(hs, bs, 60 + hs)
    check(run(c), c)


def test_many_rows_little_or_nothing_seen_and_bad_pages(gpu):
    c = shared_case(128, 16, 61)
    r = np.random.default_rng(61)
    c["masks"] = [int(m) if i % 3 else 0 for i, m in enumerate(r.integers(0, 2 ** 62, len(c["masks"])))]
    check(run(c), c)
    c["table"][2, 1], c["table"][2, 9], c["table"][10, 0], c["table"][3, :] = -5, 10 ** 6, 2 ** 31 - 1, -1
    check(run(c), c)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_many_rows_what_is_not_seen_does_not_reach_them(gpu, bad):
    hs, bs = 128, 16
    c = shared_case(hs, bs, 62)
    for s, L in enumerate(c["lens"]):
        page, off = c["table"][s, (L - 1) // bs], (L - 1) % bs + 1
        c["kc"][page, :, :, off:], c["vc"][page, :, :, off:] = bad, bad
    check(run(c), c)
    hit = []
    for s in (0, 3):  # drafted token 4: the rows that see it are not finite, no others
        p = c["lens"][s] - (c["starts"][s + 1] - c["starts"][s]) + 4
        c["kc"][c["table"][s, p // bs], :, :, p % bs] = bad
        c["vc"][c["table"][s, p // bs], :, :, p % bs] = bad
        hit += [i for i in range(c["starts"][s], c["starts"][s + 1]) if c["masks"][i] >> 4 & 1]
    out = run(c)
    others = [i for i in range(c["starts"][-1]) if i not in hit]
    check(out, c, others)
    assert not torch.isfinite(out[hit]).all(-1).any()


def test_many_rows_long_contexts_and_max_drafts(gpu):
    c = build(64, 32, 64, 16, [1500] + [20] * 15, [36] * 16, 63)
    check(run(c), c)
    c = build(64, 32, 64, 16, [30] * 16, [40] * 16, 64, masks=chain_masks(40) * 16)
    out = run(c, max_drafts=35)  # places 5..39 of the drafted ones are rows 0..34's
    for s in range(16):
        assert (out[40 * s + 35:40 * s + 40] == 7).all()
    assert torch.equal(out, run(c, max_drafts=35))


def test_many_sequences_longest_first(gpu):
    """More workgroups than run at once: sequences go by length, whatever their order."""
    r = np.random.default_rng(65)
    c = build(32, 32, 64, 16, [int(x) for x in r.integers(0, 300, 64)], [int(x) for x in r.integers(0, 4, 64)], 65)
    check(run(c), c)
    c = build(16, 16, 64, 8, [int(x) for x in r.integers(0, 40, 130)], [2] * 130, 66)
    check(run(c), c)


def test_scales_below_zero_and_zero(gpu):
    c = build(8, 2, 128, 16, [300], [20], 67)
    c["scale"] = -0.2
    out = run(c)
    check(out, {**c, "q": -c["q"], "scale": 0.2})
    c["scale"] = 0.0
    check(run(c), {**c, "q": c["q"] * 0, "scale": 1.0})


def test_one_call_form_with_views(gpu):
    """Non-contiguous q and block tables are copied, also for a call on another stream."""
    c = build(8, 2, 128, 16, [100, 30], [5, 9], 68, width=9)
    q = torch.zeros((14, 16, 128), dtype=torch.float16, device="cuda")
    q[:, ::2] = c["q"].cuda()
    wide = i32(np.repeat(c["table"], 2, 1))[:, ::2]
    dev = (c["kc"].cuda(), c["vc"].cuda(), wide, i32(c["lens"]), i32(c["starts"]), signed(c["masks"]).cuda(), 9, 105,
           c["scale"])
    check(N.tree_attention(q[:, ::2], *dev), c)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        out = N.tree_attention(q[:, ::2], *dev, stream=s)
        torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")  # the allocator may hand out what the call let go
    s.synchronize()
    check(out, c)


def test_one_call_form_copies_on_the_calls_stream(gpu):
    """Views that the call's own stream is still to fill are copied behind that work."""
    c = build(8, 2, 128, 16, [100, 30], [5, 9], 69, width=9)
    q = torch.zeros((14, 16, 128), dtype=torch.float16, device="cuda")
    table = torch.zeros((2, 18), dtype=torch.int32, device="cuda")
    cq, ctable = c["q"].cuda(), i32(c["table"])
    dev = (c["kc"].cuda(), c["vc"].cuda(), table[:, ::2], i32(c["lens"]), i32(c["starts"]), signed(c["masks"]).cuda(), 9,
           105, c["scale"])
    busy = torch.ones((4096, 4096), dtype=torch.float16, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(40):  # some ms
            torch.mm(busy, busy)
        q[:, ::2] = cq
        table[:, ::2] = ctable
    out = N.tree_attention(q[:, ::2], *dev, stream=s)
    s.synchronize()
    check(out, c)


def test_a_node_takes_smaller_calls(gpu):
    """One node for a batch that shrinks: fewer sequences and rows each time, split more, in the same scratch."""
    contexts, drafts = [700, 30, 2000, 411, 0, 1500], [5, 1, 9, 3, 8, 2]
    node = N.TreeAttention(6, 28, 9, 8, 2, 128, 16, 200, 3200, 128 ** -0.5)
    for n in (6, 5, 3, 2, 1):
        c = build(8, 2, 128, 16, contexts[:n], drafts[:n], 70, width=200)
        out = torch.full((len(c["q"]), 8, 128), 7.0, dtype=torch.float16, device="cuda")
        node(out, c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), i32(c["starts"]),
             signed(c["masks"]).cuda())
        check(out, c)


@pytest.mark.parametrize("n,heads,kv,seqs,drafts", [
    (131072, 8, 1, 1, 4), (131072, 4, 4, 3, 1), (32768, 64, 32, 16, 64),  # the last in the form of shared tiles
])
def test_weights_below_f16s_smallest(gpu, n, heads, kv, seqs, drafts):
    """One key of weight 1 and n - 1 of 2^-25 each, which together are up to 4e-3 of the result. The sequences share
    their pages, and the heads their values."""
    D, bs = 64, 32
    k, v = one_large_and_many_tiny(n, D, 71)
    kc = k.view(n // bs, 1, bs, D // 8, 8).transpose(2, 3).expand(-1, kv, -1, -1, -1).cuda().contiguous()
    vc = v.view(n // bs, 1, bs, D).transpose(2, 3).expand(-1, kv, -1, -1).cuda().contiguous()
    q = torch.zeros((seqs * drafts, heads, D), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    masks = chain_masks(drafts) * seqs
    table = np.tile(np.arange(n // bs), (seqs, 1))
    node = N.TreeAttention(seqs, seqs * drafts, drafts, heads, kv, D, bs, n // bs, n, 1.0)
    out = node(torch.empty_like(q), q, kc, vc, i32(table), i32([n] * seqs), i32(range(0, seqs * drafts + 1, drafts)),
               signed(masks).cuda()).cpu().double()
    see = torch.arange(n)[None] <= n - drafts + torch.arange(drafts)[:, None]
    want, A, d = attend(q[:drafts, 0].cpu().double(), k.double(), v.double(), see, 1.0)
    tol = tiny_bound(want, A, d, n, float(v.abs().max()))
    for s in range(seqs):
        for h in range(heads):
            err = (out[s * drafts:(s + 1) * drafts, h] - want).abs()
            assert (err <= tol).all(), (s, h, float((err / tol).max()))


def cut(c, most):
    """The case of which only the first `most` rows of each sequence are left, and which rows those are."""
    at = [i for a, b in zip(c["starts"][:-1], c["starts"][1:]) for i in range(a, min(b, a + most))]
    counts = [min(b - a, most) for a, b in zip(c["starts"][:-1], c["starts"][1:])]
    return {**c, "q": c["q"][at], "masks": [c["masks"][i] for i in at], "starts": [0] + [int(n) for n in np.cumsum(counts)]}, at


@pytest.mark.parametrize("heads,kv,contexts,drafts,most", [
    (8, 2, [40, 90, 700], [5, 3, 9], 3), (8, 2, [0, 2, 33], [64, 40, 35], 34),
    (64, 32, [30, 0, 150, 7] * 4, [40, 64, 36, 33] * 4, 35),  # the form of shared tiles
])
def test_rows_up_to_max_drafts(gpu, heads, kv, contexts, drafts, most):
    """A sequence's first max_drafts rows are computed as if it had no others."""
    c = build(heads, kv, 128, 16, contexts, drafts, 72)
    out = run(c, max_drafts=most)
    less, at = cut(c, most)
    check(out[at], less)
    rest = [i for i in range(len(out)) if i not in at]
    assert rest and (out[rest] == 7).all()


def spoil(c, s, drafted, bad):
    """Makes drafted token `drafted` of sequence s not finite -> the rows that see it."""
    bs, n = c["vc"].shape[3], c["starts"][s + 1] - c["starts"][s]
    p = c["lens"][s] - n + drafted
    c["kc"][c["table"][s, p // bs], :, :, p % bs] = bad
    c["vc"][c["table"][s, p // bs], :, :, p % bs] = bad
    return [i for i in range(c["starts"][s], c["starts"][s + 1]) if c["masks"][i] >> drafted & 1]


def check_spoilt(out, c, hit):
    assert hit
    check(out, c, [i for i in range(c["starts"][-1]) if i not in hit])
    assert not torch.isfinite(out[hit]).all(-1).any()


@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
@pytest.mark.parametrize("hs,bs", [(64, 8), (64, 32), (80, 16), (96, 32), (112, 8), (128, 32), (192, 16), (256, 8), (256, 32)])
def test_many_rows_of_any_size_and_what_they_do_not_see(gpu, hs, bs, bad):
    """The shared tiles' careful pass in its other geometries: 32-key tiles above 128 dims, dims repeated in the last
    block, pages smaller and larger than 16 tokens."""
    c = shared_case(hs, bs, 73 + hs)
    hit = spoil(c, 0, 4, bad) + spoil(c, 3, 40, bad)
    check_spoilt(run(c), c, hit)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv,hs,bs,contexts,drafts", [
    (8, 2, 128, 16, [2000], [9]), (8, 2, 64, 8, [900, 3000], [6, 20]), (4, 2, 80, 32, [1500], [40]),
    (8, 1, 192, 8, [1111], [12]), (4, 1, 256, 16, [700, 2500], [7, 33]), (4, 4, 112, 32, [130, 5000], [5, 64]),
])
def test_split_contexts_and_what_is_not_seen(gpu, heads, kv, hs, bs, contexts, drafts, bad):
    """Own tiles over several partitions: the last one is taken carefully, the merge joins it to the others."""
    c = build(heads, kv, hs, bs, contexts, drafts, 74)
    hit = [i for s, n in enumerate(drafts) for i in spoil(c, s, n // 2, bad)]
    check_spoilt(run(c), c, hit)


@pytest.mark.parametrize("heads,kv", [(4, 2), (64, 32)])
def test_pages_outside_and_values_not_finite(gpu, heads, kv):
    """A page outside the pools in the middle of a context (its tile is taken as masked) whose neighbours are not finite:
    those are seen by every row of the sequence, and by no other sequence."""
    c = build(heads, kv, 64, 8, [300, 200] * 8, [40, 36] * 8, 75)
    c["vc"][c["table"][0, 4], :, :, 3] = float("inf")
    c["table"][0, 5] = -1
    hit = list(range(40))
    check_spoilt(run(c), c, hit)
