"""GPU: causal attention of packed prompts (tlh_packed_attention) against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from serving_refs import attend, one_large_and_many_tiny, packed_reference, tiny_bound
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def inputs(heads, kv, hs, tokens, dtype, seed, std=1.0):
    """q, k and v as views of one fused projection's rows."""
    g = torch.Generator().manual_seed(seed)
    rows = (torch.randn((tokens, (heads + 2 * kv) * hs), generator=g) * std).to(dtype).cuda()
    q, k, v = rows.split([heads * hs, kv * hs, kv * hs], 1)
    return q.unflatten(1, (heads, hs)), k.unflatten(1, (kv, hs)), v.unflatten(1, (kv, hs))


def starts_of(lens, first=0):
    return [first] + [first + int(n) for n in np.cumsum(lens)]


def dev(starts):
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def check(out, q, k, v, starts, scale):
    want, tol = packed_reference(q, k, v, starts, scale, q.dtype)
    got = out.cpu().double()
    live = slice(starts[0], starts[-1])
    err = (got - want).abs()[live]
    assert torch.isfinite(got[live]).all()
    assert (err <= tol[live]).all(), float((err / tol[live]).max())


CASES = [
    # heads, kv heads, head size, lengths
    (8, 2, 128, [77]), (8, 2, 128, [1]), (4, 4, 64, [1, 2, 3, 31, 32, 33, 63, 64, 65]), (8, 1, 128, [127, 128, 129]),
    (6, 2, 128, [200, 0, 15, 0, 0, 290]), (3, 1, 64, [257, 40]), (28, 4, 64, [100, 33]), (1, 1, 256, [130, 5]),
    (4, 2, 256, [66, 97]), (4, 1, 192, [65, 130]), (5, 5, 80, [96, 33, 1]), (4, 2, 96, [140]), (2, 1, 112, [191, 64]),
    (16, 16, 128, [48, 16]), (64, 8, 64, [37]), (8, 2, 128, [513, 700, 8]), (2, 2, 64, [1500]),
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,hs,lens", CASES)
def test_against_64_bits(gpu, heads, kv, hs, lens, dtype):
    q, k, v = inputs(heads, kv, hs, sum(lens), dtype, 10 + heads + hs + len(lens))
    starts = starts_of(lens)
    out = N.packed_attention(q, k, v, dev(starts), max(lens), hs ** -0.5)
    check(out, q, k, v, starts, hs ** -0.5)


@pytest.mark.parametrize("hs", [64, 128, 192])
@pytest.mark.parametrize("std", [4.0, 0.05])
def test_sharp_and_flat_scores(gpu, hs, std):
    """Scores of some tens (a softmax of few keys, the running maximum moves) and all alike."""
    q, k, v = inputs(4, 2, hs, 300, F16, 3, std)
    out = N.packed_attention(q, k, v, dev([0, 300]), 300, hs ** -0.5)
    check(out, q, k, v, [0, 300], hs ** -0.5)


def test_growing_scores(gpu):
    """Every key scores higher than the ones before it, so each tile moves the maximum."""
    q, k, v = (t.clone() for t in inputs(4, 2, 128, 400, F16, 4))
    q[:] = 1.0
    k[:] = (torch.arange(400, device="cuda", dtype=torch.float32) / 16)[:, None, None].half()
    out = N.packed_attention(q, k, v, dev([0, 400]), 400, 128 ** -0.5)
    check(out, q, k, v, [0, 400], 128 ** -0.5)


def test_negative_scores_of_great_size(gpu):
    """Scores around -3000: the softmax is of their differences."""
    q, k, v = (t.clone() for t in inputs(4, 1, 64, 150, F16, 5))
    q[:, :, 0], k[:, :, 0] = 150.0, -160.0
    out = N.packed_attention(q, k, v, dev([0, 150]), 150, 0.125)
    check(out, q, k, v, [0, 150], 0.125)


def test_rows_outside_the_sequences_are_left_alone(gpu):
    q, k, v = inputs(8, 2, 128, 300, F16, 6)
    starts = [40, 100, 100, 230]
    out = torch.full((300, 8, 128), 7.0, dtype=F16, device="cuda")
    N.packed_attention(q, k, v, dev(starts), 130, 0.1, out=out)
    check(out, q, k, v, starts, 0.1)
    assert (out[:40] == 7).all() and (out[230:] == 7).all()


def test_tokens_past_max_seq_len_are_left_alone(gpu):
    q, k, v = inputs(8, 2, 64, 300, F16, 7)
    out = torch.full((300, 8, 64), 7.0, dtype=F16, device="cuda")
    N.packed_attention(q, k, v, dev([0, 200, 300]), 70, 0.1, out=out)
    check(out[:70], q[:70], k[:70], v[:70], [0, 70], 0.1)
    check(out[200:270], q[200:270], k[200:270], v[200:270], [0, 70], 0.1)
    assert (out[70:200] == 7).all() and (out[270:] == 7).all()


def test_starts_outside_the_tokens_are_the_nearer_end(gpu):
    q, k, v = inputs(4, 2, 64, 90, F16, 8)
    out = torch.full((90, 4, 64), 7.0, dtype=F16, device="cuda")
    N.packed_attention(q, k, v, dev([-50, 30, 20, 1000000, 2000000000]), 2000, 0.1, out=out)
    # 0..30, then a decreasing pair (nothing), 20..90, and nothing. Starts that decrease are not
    # allowed: tokens 20..29 are two sequences' and hold either's result, the others theirs
    want = torch.full_like(out, 7.0)
    N.packed_attention(q, k, v, dev([0, 30]), 30, 0.1, out=want)
    check(want, q, k, v, [0, 30], 0.1)
    assert torch.equal(out[:20], want[:20])
    out[20:30] = N.packed_attention(q[20:], k[20:], v[20:], dev([0, 70]), 70, 0.1)[:10]
    check(out[20:], q[20:], k[20:], v[20:], [0, 70], 0.1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hs", [64, 128, 256])
def test_later_tokens_reach_nothing(gpu, hs, bad):
    """A token that is not finite in k and v changes no row before it, in its own tile or another."""
    q, k, v = (t.clone() for t in inputs(4, 2, hs, 200, F16, 9))
    clean = N.packed_attention(q, k, v, dev([0, 200]), 200, 0.1)
    k[37], v[37] = bad, bad
    out = N.packed_attention(q, k, v, dev([0, 200]), 200, 0.1)
    assert torch.isfinite(out[:37]).all()
    check(out[:37], q[:37], k[:37], v[:37], [0, 37], 0.1)
    assert (out[:37].double() - clean[:37].double()).abs().max() <= 2.0 ** -8
    assert not torch.isfinite(out[37:]).all(-1).any()  # the rows that see it are not finite
    v2 = v.clone()
    v2[37] = 1.0
    k[37] = 0.0
    v2[37, :, 5] = bad  # one dim of v alone: the others stay finite in every row
    out = N.packed_attention(q, k, v2, dev([0, 200]), 200, 0.1)
    assert torch.isfinite(out[:37]).all() and torch.isfinite(out[:, :, :5]).all() and torch.isfinite(out[:, :, 6:]).all()
    seen = out[37:, :, 5].double()
    assert (torch.isnan(seen) if bad != bad else seen == bad).all()


def test_sequences_do_not_see_each_other(gpu):
    q, k, v = (t.clone() for t in inputs(4, 2, 128, 150, BF16, 11))
    k[70:], v[70:] = float("nan"), float("inf")
    out = N.packed_attention(q, k, v, dev([0, 70, 150]), 80, 0.1)
    check(out[:70], q[:70], k[:70], v[:70], [0, 70], 0.1)
    q, k, v = (t.clone() for t in inputs(4, 2, 128, 150, BF16, 11))
    k[:70], v[:70] = float("nan"), float("inf")
    out = N.packed_attention(q, k, v, dev([0, 70, 150]), 80, 0.1)
    check(out[70:], q[70:], k[70:], v[70:], [0, 80], 0.1)


def test_strided_out_and_padded_rows(gpu):
    q, k, v = inputs(4, 2, 128, 100, F16, 12)
    wide = torch.full((100, 4 * 128 + 24), 7.0, dtype=F16, device="cuda")
    out = wide[:, 8:8 + 512].unflatten(1, (4, 128))
    N.packed_attention(q, k, v, dev([0, 100]), 100, 0.1, out=out)
    check(out, q, k, v, [0, 100], 0.1)
    assert (wide[:, :8] == 7).all() and (wide[:, 520:] == 7).all()


def test_offsets_past_32_bits(gpu):
    """Token strides of 2^28 elements: the last token lies 4 GiB from the first."""
    n, hs, stride = 9, 128, 1 << 28
    base = torch.empty(((n - 1) * stride + 2 * hs,), dtype=F16, device="cuda")
    g = torch.Generator().manual_seed(13)
    k, v = (base.as_strided((n, 1, hs), (stride, hs, 1), o) for o in (0, hs))
    src = torch.randn((3, n, 1, hs), generator=g).half().cuda()
    k.copy_(src[0]), v.copy_(src[1])
    out = N.packed_attention(src[2], k, v, dev([0, n]), n, 0.1)
    check(out, src[2], k, v, [0, n], 0.1)


def test_many_short_sequences(gpu):
    r = np.random.default_rng(14)
    lens = [int(n) for n in r.integers(0, 12, 700)]
    q, k, v = inputs(2, 1, 64, sum(lens), F16, 14)
    out = N.packed_attention(q, k, v, dev(starts_of(lens)), 12, 0.125)
    check(out, q, k, v, starts_of(lens), 0.125)


def test_the_same_result_every_time(gpu):
    q, k, v = inputs(8, 2, 128, 700, F16, 15)
    a = N.packed_attention(q, k, v, dev([0, 333, 700]), 400, 0.1)
    for _ in range(5):
        assert torch.equal(a, N.packed_attention(q, k, v, dev([0, 333, 700]), 400, 0.1))


def test_on_another_stream_and_captured(gpu):
    q, k, v = inputs(8, 2, 128, 500, F16, 16)
    starts = dev([0, 123, 500])
    want = N.packed_attention(q, k, v, starts, 400, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = N.packed_attention(q, k, v, starts, 400, 0.1, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        N.packed_attention(q, k, v, starts, 400, 0.1, out=out)
    for i in range(4):  # each replay on other inputs
        q.copy_(torch.randn_like(q))
        starts.copy_(dev([0, 100 + i, 500]))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, N.packed_attention(q, k, v, starts, 400, 0.1))


def test_numbers_of_sequences_and_tokens_at_zero(gpu):
    q, k, v = inputs(4, 2, 64, 10, F16, 17)
    out = torch.full((10, 4, 64), 7.0, dtype=F16, device="cuda")
    N.packed_attention(q, k, v, dev([0]), 10, 0.1, out=out)
    N.packed_attention(q, k, v, dev([0, 10]), 0, 0.1, out=out)
    assert (out == 7).all()
    assert N.packed_attention(q[:0], k[:0], v[:0], dev([0, 0]), 5, 0.1).shape == (0, 4, 64)


def test_more_sequences_than_a_grid_dimension(gpu):
    r = np.random.default_rng(18)
    lens = [int(n) for n in r.integers(0, 3, 70001)]
    q, k, v = inputs(1, 1, 64, sum(lens), F16, 18)
    starts = starts_of(lens)
    out = N.packed_attention(q, k, v, dev(starts), 2, 0.125)
    s = (q[1:, 0].float() * k[:-1, 0].float()).sum(1) * 0.125  # a second token's two scores
    own = (q[:, 0].float() * k[:, 0].float()).sum(1) * 0.125
    want = v[:, 0].float().clone()
    second = torch.zeros(sum(lens), dtype=torch.bool, device="cuda")
    second[[a + 1 for a, n in zip(starts, lens) if n == 2]] = True
    p = torch.sigmoid(own[1:] - s)[:, None]  # the weight of the token itself
    want[1:] = torch.where(second[1:, None], p * v[1:, 0].float() + (1 - p) * v[:-1, 0].float(), want[1:])
    # f16: the result's rounding, the weights' rounding, and f32 scores
    tol = 2.0 ** -11 * 2.1 * v.float().abs().max() + 1e-4
    assert (out[:, 0].float() - want).abs().max() <= tol


def test_scales_below_zero_and_zero(gpu):
    q, k, v = inputs(4, 2, 128, 150, F16, 19)
    out = N.packed_attention(q, k, v, dev([0, 150]), 150, -0.2)
    check(out, -q, k, v, [0, 150], 0.2)
    out = N.packed_attention(q, k, v, dev([0, 150]), 150, 0.0)
    check(out, q * 0, k, v, [0, 150], 1.0)


@pytest.mark.parametrize("n", [5000, 131072])
def test_weights_below_f16s_smallest(gpu, n):
    """One key of weight 1 and n - 1 of 2^-25 each, which together are up to 4e-3 of the result."""
    k, v = one_large_and_many_tiny(n, 64, 20)
    q = torch.zeros((n, 1, 64), dtype=F16, device="cuda")
    q[:, :, 0] = 1.0
    out = N.packed_attention(q, k[:, None].cuda(), v[:, None].cuda(), dev([0, n]), n, 1.0)[:, 0].cpu().double()
    rows = torch.tensor([1, 700, n // 2, n - 33, n - 1])
    see = torch.arange(n)[None] <= rows[:, None]
    want, A, d = attend(q[:5, 0].cpu().double(), k.double(), v.double(), see, 1.0)
    err, tol = (out[rows] - want).abs(), tiny_bound(want, A, d, n, float(v.abs().max()))
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("hs", [64, 80, 128, 256])
def test_bf16_values_near_the_end_of_the_range(gpu, hs):
    """Sums of the numerators' products with v leave f32's range before they are divided by the numerators' sum."""
    q, k, v = (t.clone() for t in inputs(4, 2, hs, 330, BF16, 21))
    v[:200] *= 1e38 / 4  # normal: up to 1e38
    v[200:] = torch.where(v[200:] < 0, -torch.finfo(BF16).max, torch.finfo(BF16).max)
    for starts in ([0, 200, 330], [0, 330], [0, 1, 2, 5, 330]):
        out = N.packed_attention(q, k, v, dev(starts), 330, hs ** -0.5)
        check(out, q, k, v, starts, hs ** -0.5)
    q[:], k[:] = 0.0, 0.0  # every key alike
    v[:] = 2e38
    out = N.packed_attention(q, k, v, dev([0, 330]), 330, 1.0)
    check(out, q, k, v, [0, 330], 1.0)
    v[:] = torch.finfo(BF16).max
    out = N.packed_attention(q, k, v, dev([0, 330]), 330, 1.0)
    check(out, q, k, v, [0, 330], 1.0)


def test_bf16_large_values_behind_a_lagging_maximum(gpu):
    """Scores that grow to just below what moves the exponents' reference, 2^8, and values near 2^120."""
    n, hs = 300, 128
    q, k, v = (t.clone() for t in inputs(2, 1, hs, n, BF16, 22))
    q[:], k[:] = 0.0, 0.0
    q[:, :, 0] = 1.0
    k[:, :, 0] = torch.linspace(0, 5.5, n, device="cuda")[:, None]  # 2^7.9 at the end
    v *= 1.5e36
    v[5] = float("inf")  # some rows see this too, and are not finite
    out = N.packed_attention(q, k, v, dev([0, n]), n, 1.0)
    assert not torch.isfinite(out[5:]).any()
    check(out[:5], q[:5], k[:5], v[:5], [0, 5], 1.0)
    v[5] = 1e38
    out = N.packed_attention(q, k, v, dev([0, n]), n, 1.0)
    check(out, q, k, v, [0, n], 1.0)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv,hs", [(4, 2, 64), (5, 5, 80), (4, 1, 96), (6, 2, 112), (8, 2, 192), (3, 1, 256)])
def test_later_tokens_reach_nothing_at_any_size(gpu, heads, kv, hs, bad, dtype):
    """The careful pass where rows hold 8, 16 or 32 chunks and dims are repeated, with 1, 2 and 4 heads a workgroup."""
    q, k, v = (t.clone() for t in inputs(heads, kv, hs, 210, dtype, 23))
    k[57], v[57], v[161] = bad, bad, bad
    out = N.packed_attention(q, k, v, dev([0, 100, 210]), 110, hs ** -0.5)
    for a, b, first in ((0, 100, 57), (100, 210, 161)):
        check(out[a:first], q[a:first], k[a:first], v[a:first], [0, first - a], hs ** -0.5)
        assert not torch.isfinite(out[first:b]).all(-1).any()
