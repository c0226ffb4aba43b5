"""GPU: page copies and the accepted branch in every layer's pools (tlh_copy_blocks, tlh_compact_cache)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from serving_refs import pools, signed, tables
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def layers(n, blocks, kv, hs, bs, seed):
    g = torch.Generator().manual_seed(seed)
    ps = [pools(g, blocks, kv, hs, bs) for _ in range(n)]
    return [p[0].cuda() for p in ps], [p[1].cuda() for p in ps]


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def i64(a):
    return torch.tensor(np.asarray(a, np.int64), device="cuda")


GEO = [(2, 64, 8, 3), (8, 128, 16, 2), (1, 80, 32, 5), (3, 112, 8, 1), (4, 256, 32, 2), (32, 192, 16, 1)]


@pytest.mark.parametrize("kv,hs,bs,n", GEO)
@pytest.mark.parametrize("count", [1, 7])
def test_copies_pages_in_every_layer(gpu, kv, hs, bs, n, count):
    kc, vc = layers(n, 24, kv, hs, bs, 50 + kv)
    r = np.random.default_rng(count)
    ids = r.permutation(24)
    pairs = np.stack([ids[r.integers(0, 8, count)], ids[8:8 + count]], 1)  # sources repeat
    want = [p.clone() for p in kc + vc]
    for p in want:
        for s, d in pairs:
            p[d] = p[s]
    N.KVPools(kc, vc, kv, hs, bs).copy_blocks(i64(pairs))
    for got, w in zip(kc + vc, want):
        assert torch.equal(got, w)


def test_pairs_outside_the_pools_and_nothing_to_copy(gpu):
    kc, vc = layers(2, 10, 2, 64, 16, 51)
    want = [p.clone() for p in kc + vc]
    p = N.KVPools(kc, vc, 2, 64, 16)
    p.copy_blocks(i64([[0, 10], [10, 1], [-1, 2], [3, -1], [4, 4], [2 ** 62, 5], [6, -2 ** 63]]))
    p.copy_blocks(i64(np.zeros((0, 2))))
    for got, w in zip(kc + vc, want):
        assert torch.equal(got, w)
    p.copy_blocks(i64([[0, 10], [1, 2]]))
    want[0][2] = want[0][1]
    assert torch.equal(kc[0], want[0])


def test_more_layers_than_one_launch_takes(gpu):
    n = 150
    kc, vc = layers(n, 6, 1, 64, 8, 52)
    want = [p.clone() for p in kc + vc]
    pl = N.KVPools(kc, vc, 1, 64, 8)
    pl.copy_blocks(i64([[1, 4], [2, 0]]))
    for w in want:
        w[4], w[0] = w[1].clone(), w[2].clone()
    for got, w in zip(kc + vc, want):
        assert torch.equal(got, w)
    new = i32([-1])
    pl.compact(i32([[3, 5]]), i32([13]), i32([0, 7]), i64([0b1010100]), new, 7)
    assert new.tolist() == [9]
    expect_compact([w for w in want[:n]], [w for w in want[n:]], [[3, 5]], [13], [7], [0b1010100], 8)
    for got, w in zip(kc + vc, want):
        assert torch.equal(got, w)


def test_pool_past_32_bits(gpu):
    kv, hs, bs = 8, 128, 16
    blocks = (1 << 32) // (kv * hs * bs * 2) + 8
    kc = torch.empty((blocks, kv, hs // 8, bs, 8), dtype=torch.float16, device="cuda")
    vc = torch.zeros((blocks, kv, hs, bs), dtype=torch.float16, device="cuda")
    kc[blocks - 1].normal_(), vc[3].normal_()
    pl = N.KVPools([kc], [vc], kv, hs, bs)
    pl.copy_blocks(i64([[blocks - 1, 1], [3, blocks - 2]]))
    assert torch.equal(kc[1], kc[blocks - 1]) and torch.equal(vc[blocks - 2], vc[3])
    vc[blocks - 1].normal_()
    kw, vw = kc[-1:].clone(), vc[-1:].clone()
    new = i32([0])
    pl.compact(i32([[blocks - 1]]), i32([9]), i32([0, 5]), i64([0b11000]), new, 5)
    expect_compact([kw], [vw], [[0]], [9], [5], [0b11000], bs)
    assert new.tolist() == [6] and torch.equal(kc[-1:], kw) and torch.equal(vc[-1:], vw)


# -------------------------------------------------------------- compaction
def expect_compact(kc, vc, table, lens, drafts, keep, bs):
    """In place on (CPU or GPU) pools: the kept tokens in order, all read before any is written."""
    new = []
    NB = kc[0].shape[0]
    for s, (L, n) in enumerate(zip(lens, drafts)):
        first = L - n
        kept = [j for j in range(n) if keep[s] >> j & 1 and first + j >= 0]
        new.append(max(first, 0) + len(kept))
        moves = []
        for i, j in enumerate(kept):
            a, b = first + j, max(first, 0) + i
            pa, pb = table[s][a // bs], table[s][b // bs]
            if a != b and 0 <= pa < NB and 0 <= pb < NB:
                moves.append((int(pa), a % bs, int(pb), b % bs))
        for k, v in zip(kc, vc):
            rows = [(k[pa, :, :, oa].clone(), v[pa, :, :, oa].clone()) for pa, oa, _, _ in moves]
            for (_, _, pb, ob), (rk, rv) in zip(moves, rows):
                k[pb, :, :, ob], v[pb, :, :, ob] = rk, rv
    return new


def compact_case(kv, hs, bs, n, contexts, drafts, keep, seed, mutate=None, max_drafts=None):
    r = np.random.default_rng(seed)
    lens = [c + d for c, d in zip(contexts, drafts)]
    table, blocks = tables(r, lens, bs)
    kc, vc = layers(n, blocks, kv, hs, bs, seed)
    if mutate:
        table, lens = mutate(table, lens)
    kw, vw = [k.clone() for k in kc], [v.clone() for v in vc]
    new = torch.full((len(lens),), -5, dtype=torch.int32, device="cuda")
    starts = [0] + [int(x) for x in np.cumsum(drafts)]
    lens_d = i32(lens)
    N.KVPools(kc, vc, kv, hs, bs).compact(i32(table), lens_d, i32(starts), signed(keep).cuda(), new,
                                          max_drafts or max(drafts))
    want = expect_compact(kw, vw, table.tolist(), [max(x, 0) for x in lens], drafts, keep, bs)
    assert new.tolist() == want
    assert lens_d.tolist() == list(lens)
    for got, w in zip(kc + vc, kw + vw):
        assert torch.equal(got, w)


@pytest.mark.parametrize("kv,hs,bs,n", GEO)
def test_keeps_the_accepted_branch(gpu, kv, hs, bs, n):
    # chains of moves, where a place is one token's source and another's destination, across pages
    compact_case(kv, hs, bs, n, [30, 0, 7, 61], [9, 64, 5, 33],
                 [0b101101010, (1 << 64) - 1 - 0b10010, 0b11111, 0xAAAAAAAA | 1 << 32], 60 + kv)


def test_nothing_kept_everything_kept_and_single_tokens(gpu):
    compact_case(2, 128, 16, 2, [30, 31, 32, 0, 15], [4, 4, 1, 1, 64], [0, 15, 1, 0, 1 << 63], 61)


def test_bits_past_the_drafts_and_sequences_without_any(gpu):
    compact_case(2, 64, 8, 1, [30, 10, 5], [4, 0, 2], [0xfff0 | 0b1010, 0xff, 1 << 63 | 0b10], 62)


def test_lengths_shorter_than_the_drafts(gpu):
    compact_case(2, 64, 8, 1, [30, 10, 5, 9], [6, 5, 64, 3], [0b110101, 0b11111, (1 << 64) - 1, 0b110], 63,
                 mutate=lambda t, lens: (t, [4, 0, 8, -3]))


def test_bad_pages_are_left_out(gpu):
    def bad(t, lens):
        t[0, 3], t[1, 1] = -1, 10 ** 6
        return t, lens
    compact_case(2, 64, 8, 2, [20, 6], [10, 8], [0b1011010101, 0b11011010], 64, mutate=bad)


def test_compact_captured(gpu):
    kv, hs, bs = 2, 128, 16
    table, blocks = tables(np.random.default_rng(65), [40, 50], bs)
    kc, vc = layers(2, blocks, kv, hs, bs, 65)
    save = [p.clone() for p in kc + vc]
    pl = N.KVPools(kc, vc, kv, hs, bs)
    t, lens, starts, keep, new = i32(table), i32([40, 50]), i32([0, 8, 20]), i64([0b10010110, 0b101010101010]), i32([0, 0])
    pairs = i64([[int(table[0, 0]), blocks - 1]])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pl.compact(t, lens, starts, keep, new, 12)
        pl.copy_blocks(pairs)
    for i in range(3):
        for p, s in zip(kc + vc, save):
            p.copy_(s)
        keep.copy_(i64([0b10010110 + i, 0b101010101010 + 2 * i]))
        graph.replay()
        torch.cuda.synchronize()
        want = [s.clone() for s in save]
        n = expect_compact(want[:2], want[2:], table.tolist(), [40, 50], [8, 12], keep.tolist(), bs)
        for w in want:
            w[blocks - 1] = w[int(table[0, 0])]
        assert new.tolist() == n
        for got, w in zip(kc + vc, want):
            assert torch.equal(got, w)
