"""GPU: attention of new tokens over a paged cache (tlh_chunk_attention) against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from serving_refs import attend, one_large_and_many_tiny, pools, tables, tiny_bound
from step_refs import chunk_reference, new_token_starts
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def build(heads, kv, hs, bs, cached, new, seed, window=0, width=None):
    """cached: tokens before the new ones."""
    r, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    lens = [c + n for c, n in zip(cached, new)]
    table, blocks = tables(r, lens, bs, width=width)
    kc, vc = pools(g, blocks, kv, hs, bs)
    starts = new_token_starts(new)
    q = torch.randn((starts[-1], heads, hs), generator=g).half()
    return dict(q=q, kc=kc, vc=vc, table=table, lens=lens, starts=starts, scale=hs ** -0.5, window=window)


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def node_of(c, max_rows=None, max_context=None):
    new = [b - a for a, b in zip(c["starts"][:-1], c["starts"][1:])]
    rows, heads, hs = c["q"].shape
    return N.ChunkAttention(len(c["lens"]), rows, max_rows or max(max(new), 1), heads, c["vc"].shape[1], hs,
                            c["vc"].shape[3], c["table"].shape[1], max_context or max(max(c["lens"]), 1), c["scale"],
                            window=c["window"])


def on_gpu(c):
    return (c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), i32(c["starts"]))


def run(c, max_rows=None, max_context=None, out=None, stream=None):
    out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda") if out is None else out
    node_of(c, max_rows, max_context)(out, *on_gpu(c), stream=stream)
    torch.cuda.synchronize()
    return out


def check(out, c, rows=None, **kw):
    """Of the rows that belong to a sequence (or the given ones); the others are as they were."""
    want, tol = chunk_reference(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c["scale"], c["window"], **kw)
    mine = ~torch.isnan(want[:, 0, 0]) if rows is None else torch.tensor(rows)
    got = out.cpu().double()
    assert torch.isfinite(got[mine]).all()
    err = (got[mine] - want[mine]).abs()
    assert (err <= tol[mine]).all(), float((err / tol[mine]).max())
    if rows is None:
        assert (got[~mine] == 7).all()


CASES = [
    # heads, kv heads, head size, block size, cached tokens, new tokens
    (8, 2, 128, 16, [70], [1]), (32, 8, 128, 16, [0, 1, 15, 16, 17, 255, 600], [1, 1, 1, 1, 1, 1, 1]),
    (32, 8, 128, 16, [1500], [1]), (32, 8, 128, 16, [0], [1]), (8, 1, 64, 32, [4000, 3], [1, 1]),
    (32, 8, 128, 16, [0, 5, 300, 64], [77, 33, 16, 17]), (8, 2, 128, 16, [100, 2000, 7], [1, 130, 1]),
    (4, 1, 64, 8, [33, 5, 130], [65, 1, 9]), (8, 8, 128, 16, [300, 41], [64, 33]), (64, 8, 128, 16, [100], [63]),
    (6, 2, 80, 32, [77, 9], [211, 2]), (5, 1, 96, 8, [129], [113]), (4, 2, 112, 16, [64, 200], [16, 132]),
    (4, 2, 192, 16, [90, 300], [7, 140]), (4, 1, 256, 32, [333, 0], [64, 264]), (4, 4, 256, 8, [50], [33]),
    (28, 4, 128, 16, [1100, 3], [9, 121]), (8, 2, 128, 16, [5000, 17, 2049], [4, 230, 1]),
    (32, 32, 64, 16, [40] * 9, [2] * 9), (12, 2, 128, 32, [700], [350]), (48, 1, 128, 16, [260], [2]),
    (1, 1, 64, 16, [0, 31], [300, 1]), (2, 2, 128, 8, [3000], [513]),
]


@pytest.mark.parametrize("heads,kv,hs,bs,cached,new", CASES)
def test_against_64_bits(gpu, heads, kv, hs, bs, cached, new):
    c = build(heads, kv, hs, bs, cached, new, 20 + heads + hs + bs + sum(new))
    check(run(c), c)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 129, 1000])
def test_a_window_behind_each_token(gpu, window):
    c = build(8, 2, 128, 16, [0, 300, 7, 1000], [150, 1, 33, 70], 50 + window, window=window)
    check(run(c), c)


@pytest.mark.parametrize("hs,bs", [(64, 8), (256, 32), (80, 16), (192, 8)])
def test_a_window_in_other_geometries(gpu, hs, bs):
    c = build(4, 1, hs, bs, [700, 0, 65], [140, 40, 1], 60 + hs, window=77)
    check(run(c), c)


@pytest.mark.parametrize("window", [0, 900])
@pytest.mark.parametrize("bs", [8, 16, 32])
@pytest.mark.parametrize("hs", [64, 112, 192, 256])
def test_partitions_of_long_contexts(gpu, hs, bs, window):
    """A piece of a prompt, single tokens and a few, over contexts that are split, each in its own number of parts."""
    c = build(8, 2, hs, bs, [2950, 700, 5000, 40, 1030], [40, 1, 3, 1, 33], 70 + hs + bs, window=window)
    check(run(c), c)


def test_one_new_token_is_the_decode_step(gpu):
    """Paged attention's decode step (its own sum carries + 1e-6)."""
    c = build(32, 8, 128, 16, [99, 700, 1500], [1, 1, 1], 31)
    want = N.paged_attention(c["q"].cuda(), c["kc"].cuda(), c["vc"].cuda(), i32(c["table"]), i32(c["lens"]), 16,
                             max(c["lens"]), c["scale"], 8)
    _, tol = chunk_reference(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c["scale"])
    assert ((run(c) - want).abs().cpu().double() <= 2 * tol + 1e-6 * want.abs().cpu().double()).all()


def test_a_prompt_in_pieces_is_the_packed_prompt(gpu):
    """Pieces of 1, 200, 31 and 68 tokens over the cache the last ones left, against the packed prompt of 300."""
    c = build(8, 2, 128, 16, [0], [300], 32)
    at = torch.arange(300)
    page = torch.from_numpy(c["table"][0].astype(np.int64))[at // 16]
    k = c["kc"][page, :, :, at % 16].reshape(300, 2, 128).cuda()
    v = c["vc"][page, :, :, at % 16].reshape(300, 2, 128).cuda()
    want = N.packed_attention(c["q"].cuda(), k, v, i32([0, 300]), 300, c["scale"]).cpu().double()
    _, tol = chunk_reference(c["q"], c["kc"], c["vc"], c["table"], c["lens"], c["starts"], c["scale"])
    done = 0
    for n in (1, 200, 31, 68):
        piece = {**c, "q": c["q"][done:done + n], "lens": [done + n], "starts": [0, n]}
        assert ((run(piece).cpu().double() - want[done:done + n]).abs() <= 2 * tol[done:done + n]).all()
        done += n


def test_rows_behind_the_last_sequence_and_past_max_rows(gpu):
    c = build(8, 2, 128, 16, [40, 90], [105, 6], 35)
    c["q"] = torch.cat([c["q"], c["q"]])
    check(run(c), c)
    # the first max_rows rows of a sequence as if it had no others: its cache's last max_rows places are theirs
    for most in (3, 34, 70):
        check(run(c, max_rows=most), c, max_rows=most)


def test_contexts_shorter_than_their_new_tokens(gpu):
    """Rows at negative places see nothing and give zeros; a length below zero is zero."""
    for new in ([5, 6, 4], [50, 60, 140]):
        c = build(8, 2, 128, 16, [40, 40, 40], new, 37)
        c["lens"] = [3, 0, 44]
        out = run(c, max_context=48)
        check(out, c)
        assert (out[:new[0] - 3] == 0).all() and (out[new[0]:new[0] + new[1]] == 0).all()
        c["lens"] = [3, -9, 44]
        check(run(c, max_context=48), c)


def test_lengths_past_the_maximum_are_the_maximum(gpu):
    c = build(8, 2, 64, 16, [60], [4], 38)
    c["lens"] = [1000000]
    check(run(c, max_context=50), c, max_context=50)


@pytest.mark.parametrize("starts", [[0, 0, 9], [3, 5, 9], [0, 9, 9], [4, 4, 4], [-5, 4, 100], [-5, -9, 4]])
def test_starts_that_leave_rows_out(gpu, starts):
    """Gaps, empty sequences, starts outside the rows (taken as the nearer end)."""
    c = build(8, 2, 128, 16, [40, 90], [3, 6], 39)
    c["starts"] = starts
    clamped = [max(0, min(x, 9)) for x in starts]
    bounds = [(a, max(a, b)) for a, b in zip(clamped[:-1], clamped[1:])]
    out = run(c, max_rows=9)
    mine = set()
    for s, (a, b) in enumerate(bounds):
        if b > a:
            one = {**c, "lens": [c["lens"][s]], "table": c["table"][s:s + 1], "starts": [a, b]}
            check(out, one, rows=list(range(a, b)))
            mine |= set(range(a, b))
    assert (out[[i for i in range(9) if i not in mine]] == 7).all()


@pytest.mark.parametrize("page", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_pages_outside_the_pools_are_not_seen(gpu, page):
    c = build(8, 2, 128, 16, [200, 40, 300], [1, 40, 170], 39)
    c["table"][0, 3], c["table"][0, 12], c["table"][1, 3], c["table"][2, 1] = page, page, page, page
    check(run(c), c)
    c["table"][1, :] = page  # nothing left
    out = run(c)
    check(out, c)
    assert (out[1:41] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,hs,bs", [(8, 128, 16), (2, 64, 8), (4, 256, 32), (8, 80, 16), (4, 112, 8), (4, 192, 16), (6, 96, 32)])
def test_what_is_not_seen_does_not_reach_a_row(gpu, heads, hs, bs, bad):
    """Slots past the context, the rest of the pool, and a new token that is not finite: only it and later ones see it."""
    c = build(heads, 2, hs, bs, [37, 500, 70], [6, 1, 150], 40)
    for s, L in enumerate(c["lens"]):
        page, off = c["table"][s, (L - 1) // bs], (L - 1) % bs + 1
        c["kc"][page, :, :, off:], c["vc"][page, :, :, off:] = bad, bad
    used = {int(c["table"][s, i]) for s, L in enumerate(c["lens"]) for i in range(-(-L // bs))}
    for b in set(range(c["kc"].shape[0])) - used:
        c["kc"][b], c["vc"][b] = bad, bad
    check(run(c), c)
    hit = []
    for s, i in ((0, 3), (2, 90)):
        p = c["lens"][s] - (c["starts"][s + 1] - c["starts"][s]) + i
        c["kc"][c["table"][s, p // bs], :, :, p % bs] = bad
        c["vc"][c["table"][s, p // bs], :, :, p % bs] = bad
        hit += range(c["starts"][s] + i, c["starts"][s + 1])
    out = run(c)
    check(out, c, [i for i in range(c["starts"][-1]) if i not in hit])
    assert not torch.isfinite(out[hit]).all(-1).any()
    # values alone: a weight of the softmax meets them, not a score
    for s, i in ((0, 3), (2, 90)):
        p = c["lens"][s] - (c["starts"][s + 1] - c["starts"][s]) + i
        c["kc"][c["table"][s, p // bs], :, :, p % bs] = 0.0
    out = run(c)
    check(out, c, [i for i in range(c["starts"][-1]) if i not in hit])
    assert not torch.isfinite(out[hit]).all(-1).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_before_the_window_does_not_reach_a_row(gpu, bad):
    c = build(8, 2, 128, 16, [400, 300], [1, 90], 41, window=50)
    for s, p in ((0, 350), (1, 270)):  # seen by no row of 0, by rows 0..19 of 1 (places 300..319)
        c["kc"][c["table"][s, p // 16], :, :, p % 16] = bad
        c["vc"][c["table"][s, p // 16], :, :, p % 16] = bad
    out = run(c)
    check(out, c, [0] + list(range(21, 91)))
    assert not torch.isfinite(out[1:21]).all(-1).any()


def test_sharp_scores(gpu):
    for new in ([20], [200]):
        c = build(8, 2, 128, 16, [300], new, 42)
        c["q"] = c["q"] * 20
        check(run(c), c)


@pytest.mark.parametrize("new", [1, 120])
def test_a_pool_past_32_bits(gpu, new):
    """Pages more than 2^32 bytes into the pools."""
    kv, hs, bs = 8, 128, 16
    blocks = (1 << 32) // (kv * hs * bs * 2) + 40
    c = build(8, kv, hs, bs, [90], [new], 43)
    n = c["kc"].shape[0]
    kc = torch.empty((blocks, kv, hs // 8, bs, 8), dtype=torch.float16, device="cuda")
    vc = torch.empty((blocks, kv, hs, bs), dtype=torch.float16, device="cuda")
    kc[-n:], vc[-n:] = c["kc"].cuda(), c["vc"].cuda()
    out = N.chunk_attention(c["q"].cuda(), kc, vc, i32(c["table"] + blocks - n), i32(c["lens"]), i32(c["starts"]), new,
                            90 + new, c["scale"])
    check(out, c)


@pytest.mark.parametrize("new", [3, 90])
def test_views_of_wider_rows(gpu, new):
    """q and out as columns of buffers of other strides, also of one buffer; the columns beside them stay."""
    c = build(8, 2, 128, 16, [130, 20], [new, 5], 44)
    rows = c["q"].shape[0]
    q = torch.full((rows, 11, 128), 3.0, dtype=torch.float16, device="cuda")
    q[:, 2:10] = c["q"].cuda()
    out = torch.full((rows, 20, 128), 7.0, dtype=torch.float16, device="cuda")
    dev = on_gpu(c)
    node_of(c)(out[:, 4:12], q[:, 2:10], *dev[1:])
    check(out[:, 4:12], c)
    assert (out[:, :4] == 7).all() and (out[:, 12:] == 7).all()
    one = torch.full((rows, 17, 128), 5.0, dtype=torch.float16, device="cuda")
    one[:, :8] = c["q"].cuda()
    node_of(c)(one[:, 9:], one[:, :8], *dev[1:])
    check(one[:, 9:], c)
    assert (one[:, 8] == 5).all() and torch.equal(one[:, :8], c["q"].cuda())


def test_page_shared_by_sequences_and_a_wide_table(gpu):
    c = build(8, 2, 128, 16, [64, 64], [4, 107], 45, width=40)
    c["table"][1, :4] = c["table"][0, :4]
    check(run(c), c)


@pytest.mark.parametrize("cached,new", [([3000, 10], [1, 1]), ([3000, 10], [8, 300]), ([6000], [256])])
def test_the_same_result_every_time_and_a_used_scratch(gpu, cached, new):
    c = build(32, 8, 128, 16, cached, new, 46)
    a, node, dev = run(c), node_of(c), on_gpu(c)
    node.scratch[N.CHUNK_COUNTER_BYTES:].fill_(0xff)
    for _ in range(3):
        assert torch.equal(a, node(torch.empty_like(a), *dev))
        assert (node.scratch[:N.CHUNK_COUNTER_BYTES] == 0).all()


def test_a_node_for_more_takes_smaller_calls(gpu):
    """A node made for the largest batch and context: fewer sequences, rows and tokens each time, in the same scratch."""
    cached, new = [700, 30, 2000, 411, 0, 1500], [5, 200, 1, 33, 80, 2]
    node = N.ChunkAttention(9, 600, 400, 8, 2, 128, 16, 8192, 131072, 128 ** -0.5)
    for n in (6, 5, 3, 2, 1):
        c = build(8, 2, 128, 16, cached[:n], new[:n], 47, width=8192)
        out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda")
        check(node(out, *on_gpu(c)), c)
    c = build(8, 2, 128, 16, [40, 7], [4, 0], 48, width=8192)
    out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda")
    check(node(out, *on_gpu(c)), c)


@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 500])
def test_many_sequences(gpu, seqs):
    r = np.random.default_rng(seqs)
    cached = [int(x) for x in r.integers(0, 200, seqs)]
    new = [int(x) for x in r.choice([0, 1, 1, 1, 2, 40], seqs)]
    c = build(4, 2, 64, 16, cached, new, 49)
    check(run(c), c)


def test_more_sequences_than_a_plan_looks_at_once(gpu):
    """Over a thousand, some without rows or tokens, pieces and contexts that are split among them; and one node for
    these and for fewer."""
    r = np.random.default_rng(80)
    cached = [int(x) for x in r.choice([0, 3, 50, 100], 1100)]
    new = [int(x) for x in r.choice([0, 0, 1, 2], 1100)]
    for s, (c, n) in {0: (900, 1), 63: (4000, 1), 64: (700, 60), 1023: (0, 0), 1024: (3000, 1), 1099: (600, 33)}.items():
        cached[s], new[s] = c, n
    c = build(4, 2, 64, 16, cached, new, 81)
    node, dev = node_of(c), on_gpu(c)
    for S in (1100, 1025, 65, 64, 1100):
        rows = c["starts"][S]
        out = torch.full((rows, 4, 64), 7.0, dtype=torch.float16, device="cuda")
        node(out, dev[0][:rows], dev[1], dev[2], dev[3][:S], dev[4][:S], dev[5][:S + 1])
        check(out, {**c, "q": c["q"][:rows], "table": c["table"][:S], "lens": c["lens"][:S], "starts": c["starts"][:S + 1]})
        assert (node.scratch[:N.CHUNK_COUNTER_BYTES] == 0).all()


@pytest.mark.parametrize("at", [0, 64, 65, 128])
def test_starts_that_decrease_among_many_compute_nothing(gpu, at):
    c = build(4, 2, 64, 16, [600] * 130, [2] * 130, 82)
    node, dev = node_of(c), list(on_gpu(c))
    out, right = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda"), dev[5].clone()
    dev[5][at] = 259
    node(out, *dev)
    torch.cuda.synchronize()
    assert (out == 7).all() and (node.scratch[:N.CHUNK_COUNTER_BYTES] == 0).all()
    dev[5] = right
    check(node(out, *dev), c)


def test_nothing_to_do(gpu):
    c = build(8, 2, 128, 16, [40, 7], [4, 0], 50)
    c["starts"] = [0, 0, 0]
    assert (run(c, max_rows=4) == 7).all()


def test_scales_below_zero_and_zero(gpu):
    for new in (3, 120):
        c = build(8, 2, 128, 16, [300], [new], 51)
        c["scale"] = -0.2
        check(run(c), {**c, "q": -c["q"], "scale": 0.2})
        c["scale"] = 0.0
        check(run(c), {**c, "q": c["q"] * 0, "scale": 1.0})


@pytest.mark.parametrize("n,heads,kv,new", [(131072, 8, 1, 1), (131072, 4, 4, 3), (32768, 32, 1, 40)])
def test_weights_below_f16s_smallest(gpu, n, heads, kv, new):
    """One key of weight 1 and n - 1 of 2^-25 each, which together are up to 4e-3 of the result."""
    D, bs = 64, 32
    k, v = one_large_and_many_tiny(n, D, 71)
    kc = k.view(n // bs, 1, bs, D // 8, 8).transpose(2, 3).expand(-1, kv, -1, -1, -1).cuda().contiguous()
    vc = v.view(n // bs, 1, bs, D).transpose(2, 3).expand(-1, kv, -1, -1).cuda().contiguous()
    q = torch.zeros((new, heads, D), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    out = N.chunk_attention(q, kc, vc, i32(np.arange(n // bs)[None]), i32([n]), i32([0, new]), new, n, 1.0).cpu().double()
    see = torch.arange(n)[None] <= n - new + torch.arange(new)[:, None]
    want, A, d = attend(q[:, 0].cpu().double(), k.double(), v.double(), see, 1.0)
    tol = tiny_bound(want, A, d, n, float(v.abs().max()))
    for h in range(heads):
        err = (out[:, h] - want).abs()
        assert (err <= tol).all(), (h, float((err / tol).max()))


def test_captured_and_replayed(gpu):
    """A graph over inputs that change: lengths, starts, pages and queries."""
    c = build(32, 8, 128, 16, [1000, 300, 50], [1, 130, 7], 52)
    dev, node = on_gpu(c), node_of(c)
    out = torch.zeros_like(dev[0])
    node(out, *dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        node(out, *dev)
    for i in range(4):
        dev[0].copy_(torch.randn_like(dev[0]))
        dev[4].copy_(i32([1001 - 100 * i, 430, 57 - i]))
        dev[5].copy_(i32([[0, 1, 131, 138], [0, 100, 101, 138], [0, 0, 130, 131], [2, 7, 9, 130]][i]))
        out.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, node(torch.full_like(out, 7), *dev))


def test_one_call_form_on_streams(gpu):
    """Block tables that are a view are copied, on the call's stream; the result is the current stream's."""
    c = build(8, 2, 128, 16, [100, 30], [5, 99], 53, width=9)
    q, kc, vc, _, lens, starts = on_gpu(c)
    wide = i32(np.repeat(c["table"], 2, 1))[:, ::2]
    rest = (kc, vc, wide, lens, starts, 99, 130, c["scale"])
    want = N.chunk_attention(q, *rest)
    check(want, c)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream, 0):
        out = N.chunk_attention(q, *rest, stream=stream)
        torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda")  # the allocator may hand out what the call let go
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("starts", [[9, 4, 8], [0, 9, 0], [0, 9, 8]])
def test_starts_that_decrease_compute_nothing(gpu, starts):
    """Sequences that overlap would make more work than the scratch has room for; the next call is as ever."""
    c = build(8, 2, 128, 16, [4000, 2000], [3, 6], 39)
    node, dev = node_of(c, max_rows=9), list(on_gpu(c))
    out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda")
    right, dev[5] = dev[5], i32(starts)
    node(out, *dev)
    torch.cuda.synchronize()
    assert (out == 7).all() and (node.scratch[:N.CHUNK_COUNTER_BYTES] == 0).all()
    dev[5] = right
    check(node(out, *dev), c)


def close_bound(out, A, d, keys, vmax):
    """Weights of few rows: rounded to f16, plus what that took off rounded to f16, which is off by half a step of half a
    step, 2^-22 of the weight (below f16's normal range by 2^-25, 2^-32 of the largest, which is at least 2^7)."""
    eps = torch.finfo(torch.float16).eps
    return out.abs() * eps / 2 * 1.01 + A * 2.0 ** -22 * 1.01 + 2 * d * A + 2.0 ** -32 * keys * vmax + 2.0 ** -24


@pytest.mark.parametrize("heads,hs,bs,new", [(8, 64, 16, 1), (8, 128, 8, 3), (4, 128, 32, 32), (4, 80, 16, 7), (4, 192, 32, 2),
                                             (2, 256, 16, 64)])
def test_weights_of_few_rows_keep_what_f16_rounds_off(gpu, heads, hs, bs, new):
    """Sums that nearly cancel, where the weights' rounding to f16 (2^-11 of each) would be all there is to see."""
    cached = [1, 2, 3, 5, 9, 40, 300, 1500]
    c = build(heads, 2, hs, bs, cached, [new] * len(cached), 90 + hs)
    c["kc"][:, :, 1:], c["scale"] = 0.0, 0.25  # scores of eight dims, whose sums are off by little
    out = run(c).cpu().double()
    for s, L in enumerate(c["lens"]):
        at, pos = slice(c["starts"][s], c["starts"][s + 1]), np.arange(L)
        page, off = torch.from_numpy(c["table"][s, pos // bs].astype(np.int64)), torch.from_numpy(pos % bs)
        see = torch.arange(L)[None] <= L - new + torch.arange(new)[:, None]
        for h in range(heads):
            g = h // (heads // 2)
            k, v = c["kc"][page, g, :, off].reshape(L, hs)[:, :8].double(), c["vc"][page, g, :, off].reshape(L, hs).double()
            want, A, d = attend(c["q"][at, h, :8].double(), k, v, see, c["scale"])
            err, tol = (out[at, h] - want).abs(), close_bound(want, A, d, L, float(v.abs().max()))
            assert (err <= tol).all(), (s, h, float((err / tol).max()))


@pytest.mark.parametrize("hs,bs,new", [(128, 16, 1), (64, 8, 5), (256, 32, 20), (192, 16, 2)])
def test_infinite_values_that_are_seen(gpu, hs, bs, new):
    """An infinity that a row sees is its result in that dim, whatever its weight's rounding; both signs are NaN."""
    c = build(4, 2, hs, bs, [400], [new], 95)
    place = lambda p: (c["table"][0, p // bs], slice(None), p % bs)  # noqa: E731
    for p, dims, x in ((40, slice(0, 8), float("inf")), (333, slice(8, 16), -float("inf")), (41, slice(16, 20), float("inf")),
                       (42, slice(16, 20), -float("inf"))):
        page, g, off = place(p)
        c["vc"][page, g, dims, off] = x
    out = run(c).cpu()
    assert (out[..., :8] == float("inf")).all() and (out[..., 8:16] == -float("inf")).all() and torch.isnan(out[..., 16:20]).all()
    finite = {**c, "vc": torch.where(torch.isfinite(c["vc"]), c["vc"], torch.zeros_like(c["vc"]))}
    want, tol = chunk_reference(finite["q"], finite["kc"], finite["vc"], c["table"], c["lens"], c["starts"], c["scale"])
    assert ((out[..., 20:].double() - want[..., 20:]).abs() <= tol[..., 20:]).all()


@pytest.mark.parametrize("window,cached", [(64, 89), (65, 99), (1, 64), (100, 200)])
def test_a_windowed_node_for_many_rows_takes_few(gpu, window, cached):
    """Whose contexts count a tile more in blocks of few rows than in those of many."""
    whole = build(32, 8, 128, 16, [cached - 39, cached], [40, 1], 96, window=window)
    node = N.ChunkAttention(2, 41, 40, 32, 8, 128, 16, whole["table"].shape[1], cached + 1, whole["scale"], window=window)
    for new in ([40, 1], [16, 1], [1, 1], [0, 1]):
        c = {**whole, "starts": new_token_starts(new), "q": whole["q"][:sum(new)]}
        out = torch.full(c["q"].shape, 7.0, dtype=torch.float16, device="cuda")
        check(node(out, *on_gpu(c)), c)


def close(c, out, heads, kv, hs, bs, new):
    for s, L in enumerate(c["lens"]):
        at, pos = slice(c["starts"][s], c["starts"][s + 1]), np.arange(L)
        page, off = torch.from_numpy(c["table"][s, pos // bs].astype(np.int64)), torch.from_numpy(pos % bs)
        see = torch.arange(L)[None] <= L - new + torch.arange(new)[:, None]
        for h in range(heads):
            g = h // (heads // kv)
            k, v = c["kc"][page, g, :, off].reshape(L, hs)[:, :8].double(), c["vc"][page, g, :, off].reshape(L, hs).double()
            want, A, d = attend(c["q"][at, h, :8].double(), k, v, see, c["scale"])
            err, tol = (out[at, h] - want).abs(), close_bound(want, A, d, L, float(v.abs().max()))
            yield bool((err <= tol).all())


@pytest.mark.parametrize("heads,hs,bs,new", [(8, 64, 16, 33), (8, 128, 8, 90), (4, 128, 32, 130), (4, 80, 16, 70), (4, 112, 16, 40),
                                             (4, 96, 32, 200), (4, 192, 32, 50), (4, 192, 16, 140), (2, 256, 16, 65)])
def test_weights_of_many_rows_keep_what_f16_rounds_off(gpu, heads, hs, bs, new):
    """As those of few, unless the caller asks for weights in f16; contexts that are split among them."""
    cached = [1, 40, 300, 2500]
    c = build(heads, 2 if heads < 8 else 1, hs, bs, cached, [new] * len(cached), 97 + hs)
    kv = c["vc"].shape[1]
    c["kc"][:, :, 1:], c["scale"] = 0.0, 0.25
    out = run(c).cpu().double()
    assert all(close(c, out, heads, kv, hs, bs, new))
    fast = N.ChunkAttention(4, c["q"].shape[0], new, heads, kv, hs, bs, c["table"].shape[1], max(c["lens"]), 0.25, f16_weights=True)
    fast = fast(torch.empty_like(c["q"], device="cuda"), *on_gpu(c))
    assert not all(close(c, fast.cpu().double(), heads, kv, hs, bs, new))  # the test can see it
    check(fast, c)


@pytest.mark.parametrize("heads,kv,hs,bs,cached,new", [x for x in CASES if max(x[5]) * x[0] // x[1] > 64])
def test_f16_weights_against_64_bits(gpu, heads, kv, hs, bs, cached, new):
    """Few rows beside many are what they are without; the one-call form takes it too."""
    c = build(heads, kv, hs, bs, cached, new, 20 + heads + hs + bs + sum(new))
    want, dev = run(c), on_gpu(c)
    out = N.chunk_attention(*dev, max(new), max(c["lens"]), c["scale"], f16_weights=True)
    check(out, c)
    for s, n in enumerate(new):
        at = slice(c["starts"][s], c["starts"][s + 1])
        if n * heads // kv <= 64:
            assert torch.equal(out[at], want[at])
        if n * heads // kv > 64:
            assert not torch.equal(out[at], want[at])


@pytest.mark.parametrize("f16_weights", [False, True])
@pytest.mark.parametrize("hs,bs,new", [(128, 16, 40), (64, 8, 70), (256, 32, 90), (192, 16, 70), (80, 32, 50)])
def test_infinite_values_that_many_rows_see(gpu, hs, bs, new, f16_weights):
    """An infinity that a row sees is its result in that dim, both signs are NaN, and the other dims are as ever; rows
    before it do not see it."""
    c = build(4, 1, hs, bs, [400], [new], 98)
    for p, dims, x in ((40, slice(0, 8), float("inf")), (333, slice(8, 16), -float("inf")), (41, slice(16, 20), float("inf")),
                       (42, slice(16, 20), -float("inf")), (420, slice(24, 28), float("inf"))):
        c["vc"][c["table"][0, p // bs], :, dims, p % bs] = x
    node = N.ChunkAttention(1, new, new, 4, 1, hs, bs, c["table"].shape[1], 400 + new, c["scale"], f16_weights=f16_weights)
    out = node(torch.empty_like(c["q"], device="cuda"), *on_gpu(c)).cpu()
    assert (out[..., :8] == float("inf")).all() and (out[..., 8:16] == -float("inf")).all() and torch.isnan(out[..., 16:20]).all()
    assert (out[20:, :, 24:28] == float("inf")).all() and torch.isfinite(out[:20, :, 24:28]).all()
    finite = {**c, "vc": torch.where(torch.isfinite(c["vc"]), c["vc"], torch.zeros_like(c["vc"]))}
    want, tol = chunk_reference(finite["q"], finite["kc"], finite["vc"], c["table"], c["lens"], c["starts"], c["scale"])
    for dims in (slice(20, 24), slice(28, hs)):
        assert ((out[..., dims].double() - want[..., dims]).abs() <= tol[..., dims]).all()
    assert ((out[:20, :, 24:28].double() - want[:20, :, 24:28]).abs() <= tol[:20, :, 24:28]).all()
