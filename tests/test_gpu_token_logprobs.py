"""GPU: log probabilities, entropy and top alternatives (tlh_token_logprobs) against the formula in 64 bits.

Bounds: x - max is one f32 rounding of at most 2^-24 times the largest |x - max| or |x|; exp's argument,
the exponential and the sums are off by at most 2^-19 relatively over a row, and log S by as much absolutely
plus its own rounding; so a log probability by 2^-23 (|x| + |lp|) + 2^-18. The entropy is log S - T / S:
T / S is a mean of x - max, off by 2^-18 of the mean of |x - max| and by 2^-18.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def reference(x, tokens, top):
    x = x.detach().cpu().double()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    logp = d - torch.log(S)
    mean = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1) / S[:, 0]
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -x.numpy()), axis=-1)[:, :top]
    ids = torch.from_numpy(order.copy())
    return (logp.gather(1, tokens.cpu().long()[:, None])[:, 0], torch.log(S)[:, 0] - mean, logp.gather(1, ids), ids,
            x.gather(1, tokens.cpu().long()[:, None])[:, 0], x.gather(1, ids), mean)


def close(got, want, tol):
    got = got.cpu().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    ok = same | ((got - want).abs() <= tol)
    assert ok.all(), (got[~ok][:5], want[~ok][:5])


def check(x, tokens, top, outs=None):
    lp, ent, tl, ti = outs or N.token_logprobs(x, tokens, top)
    wlp, went, wtl, wti, xt, xtop, mean = reference(x, tokens, top)
    assert torch.equal(ti.cpu().long(), wti)
    fin = lambda t: torch.where(torch.isinf(t), torch.zeros_like(t), t).abs()  # noqa: E731
    close(lp, wlp, 2.0 ** -23 * (fin(xt) + fin(wlp) + fin(x.cpu().double().amax(1))) + 2.0 ** -18)
    close(ent, went, 2.0 ** -18 * (1 + mean.abs()))
    close(tl, wtl, 2.0 ** -23 * (fin(xtop) + fin(wtl) + fin(x.cpu().double().amax(1))[:, None]) + 2.0 ** -18)


def logits(rows, vocab, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * std).to(dtype).cuda()


def tokens_of(rows, vocab, seed):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 5, 5), (3, 33, 32), (1, 4096, 20), (5, 4097, 8), (2, 16384, 32),
                                            (300, 1000, 3), (4, 32000, 20), (260, 32001, 5), (1, 128256, 32),
                                            (1, 300000, 20), (3, 1000000, 7), (7, 50257, 0), (4, 262144, 1)])
def test_against_64_bits(gpu, rows, vocab, top, dtype):
    """16-bit logits tie often: the lowest index wins."""
    x, t = logits(rows, vocab, dtype, 70 + rows), tokens_of(rows, vocab, 1)
    t[0], t[-1] = 0, vocab - 1
    check(x, t, top)


@pytest.mark.parametrize("allowed", [1, 3, 40, 5000])
@pytest.mark.parametrize("rows,vocab", [(2, 50000), (300, 20000)])
def test_masked_logits(gpu, rows, vocab, allowed):
    """A grammar's mask: -inf but for a few tokens, fewer than `top` among them."""
    x, r = logits(rows, vocab, torch.float32, 71), np.random.default_rng(allowed)
    keep = torch.zeros((rows, vocab), dtype=torch.bool)
    for i in range(rows):
        keep[i, torch.from_numpy(r.permutation(vocab)[:allowed])] = True
    x.masked_fill_(~keep.cuda(), float("-inf"))
    check(x, keep.int().argmax(1).int().cuda(), 20)
    check(x, tokens_of(rows, vocab, 2), 20)  # mostly masked tokens: -inf


def test_masked_by_the_lowest_number(gpu):
    x = logits(3, 9000, torch.float32, 72)
    x[:, 5:8000] = torch.finfo(torch.float32).min
    check(x, torch.tensor([0, 6, 8999], dtype=torch.int32, device="cuda"), 32)
    x = x.half().masked_fill(torch.rand((3, 9000), device="cuda") < 0.5, torch.finfo(torch.float16).min)
    check(x, torch.tensor([0, 6, 8999], dtype=torch.int32, device="cuda"), 32)


@pytest.mark.parametrize("value", [0.0, -3.5, 60000.0, -60000.0])
def test_equal_logits(gpu, value):
    """All alike: probability 1 / V, entropy log V, the lowest indices."""
    x = torch.full((2, 70000), value, device="cuda")
    check(x, torch.tensor([5, 69999], dtype=torch.int32, device="cuda"), 32)
    x[:, ::2] = -x[:, ::2]  # -0 equals 0
    check(x, torch.tensor([5, 69999], dtype=torch.int32, device="cuda"), 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_largest_logits_crowded_together(gpu, dtype):
    """Sorted logits, and the largest ones at the stride of one lane: more above a wave's threshold than it lists."""
    up = torch.linspace(-30, 30, 40000, device="cuda").to(dtype)[None].contiguous()
    t = torch.tensor([39000], dtype=torch.int32, device="cuda")
    check(up, t, 32)
    check(up.flip(1).contiguous(), t, 32)
    for rows in (1, 300):
        x = logits(rows, 20000, dtype, 73, 0.5)
        per = 8 if dtype == torch.float16 else 4
        for lane in range(0, 20):  # 20 lanes of the first wave hold nothing but large values
            for i in range(0, 20000, 256 * per):
                n = min(per, max(0, 20000 - i - lane * per))
                x[:, i + lane * per:i + lane * per + n] += 20 + torch.rand((rows, n), device="cuda").to(dtype) * 8
        check(x, tokens_of(rows, 20000, 3), 32)
        check(x, tokens_of(rows, 20000, 3), 19)


def test_great_and_small_spreads(gpu):
    for std in (1e-3, 100.0, 1e5):
        check(logits(4, 30000, torch.float32, 74, std), tokens_of(4, 30000, 4), 10)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (3, 5), (0, 1), (7, 8)])
def test_rows_at_any_stride_and_alignment(gpu, dtype, offset, pad):
    base = logits(1, 5 * (20001 + pad) + offset, dtype, 75)[0]
    x = base[offset:].as_strided((5, 20001), (20001 + pad, 1), base.storage_offset() + offset)
    check(x, tokens_of(5, 20001, 5), 12)


def test_neighbours_are_not_read_into_a_row(gpu):
    base = torch.full((6, 30011), float("nan"), device="cuda")
    x = base[:, 3:30004]
    x.copy_(logits(6, 30001, torch.float32, 76))
    check(x, tokens_of(6, 30001, 6), 9)


def test_what_is_not_defined_is_nan(gpu):
    x = logits(4, 9000, torch.float32, 77)
    x[0] = float("-inf")
    x[1, 77] = float("inf")
    x[2, 8000] = float("nan")
    t = torch.tensor([3, 4, 5, 9000], dtype=torch.int32, device="cuda")
    lp, ent, tl, ti = N.token_logprobs(x, t, 4)
    assert torch.isnan(lp).all() and torch.isnan(ent[:3]).all() and torch.isfinite(ent[3])
    assert ti[0].tolist() == [0, 1, 2, 3] and ti[1, 0] == 77 and ti[2, 0] == 8000
    assert torch.isfinite(tl[3]).all()
    lp = N.token_logprobs(x, torch.full((4,), -1, dtype=torch.int32, device="cuda"))[0]
    assert torch.isnan(lp).all()


def test_parts_left_out_and_smaller_batches(gpu):
    x, t = logits(9, 20000, torch.float32, 78), tokens_of(9, 20000, 7)
    node = N.TokenLogprobs(9, 20000, 6)
    f = lambda *s: torch.full(s, 7.0, device="cuda")  # noqa: E731
    ids = torch.zeros((4, 6), dtype=torch.int32, device="cuda")
    node.scratch.fill_(0xff)
    check(x[2:6], t[2:6], 6, node(x[2:6], t[2:6], f(4), f(4), f(4, 6), ids))
    lp, ent, _, _ = N.TokenLogprobs(9, 20000)(x, t, f(9), None)
    assert ent is None and torch.equal(lp, N.token_logprobs(x, t)[0])
    _, ent, _, _ = N.TokenLogprobs(9, 20000)(x, None, None, f(9))
    assert torch.equal(ent, N.token_logprobs(x, t)[1])


def test_more_rows_than_a_grid_dimension(gpu):
    x, t = logits(70001, 40, torch.float32, 79), tokens_of(70001, 40, 8)
    check(x, t, 3)


def test_rows_past_32_bits(gpu):
    """Row strides of 2^29 elements: the last row lies 2^32 bytes from the first."""
    base = torch.empty((2 * (1 << 29) + 5000,), device="cuda")
    x = base.as_strided((3, 5000), (1 << 29, 1))
    x.copy_(logits(3, 5000, torch.float32, 80))
    check(x, tokens_of(3, 5000, 9), 6)


def test_on_another_stream_and_captured(gpu):
    x, t = logits(3, 128256, torch.float32, 81), tokens_of(3, 128256, 10)
    want = N.token_logprobs(x, t, 5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = N.token_logprobs(x, t, 5, stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    node, outs = N.TokenLogprobs(3, 128256, 5), [torch.zeros_like(o) for o in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        node(x, t, *outs)
    for _ in range(4):
        x.copy_(torch.randn_like(x) * 3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, N.token_logprobs(x, t, 5)))


@pytest.mark.parametrize("rows,vocab,top", [(6, 128256, 5), (16, 21236, 8), (68, 19835, 32), (300, 8192, 32), (300, 8193, 32),
                                            (20, 4090, 20), (3, 8190, 7)])
@pytest.mark.parametrize("masked", [0.0, 0.999])
def test_ends_of_chunks(gpu, rows, vocab, top, masked):
    """Last chunks that hold a few vectors, masked ones among them, and vocabularies about the chunk lengths."""
    x = logits(rows, vocab, torch.float32, 82)
    off = torch.rand((rows, vocab), generator=torch.Generator().manual_seed(83)) < masked
    off[:, 0] = False
    x.masked_fill_(off.cuda(), float("-inf"))
    check(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), top)


@pytest.mark.parametrize("vocab", [500, 5000, 40000, 200000])
def test_numbers_too_far_apart_to_subtract(gpu, vocab):
    """Whole waves, and whole chunks, at one end of the range, the maximum at the other: their difference overflows."""
    x = torch.full((2, vocab), -3e38, dtype=torch.float32, device="cuda")
    x[0, vocab // 2] = x[0, vocab - 1] = 3e38
    x[1, 3] = x[1, 4] = x[1, vocab // 3] = 3e38
    t = torch.tensor([vocab - 1, 4], dtype=torch.int32, device="cuda")
    lp, ent, tl, ti = N.token_logprobs(x, t, 2)
    want = torch.log(torch.tensor([2.0, 3.0], dtype=torch.float64))  # two and three equal ones, the rest 0
    close(ent, want, torch.full((2,), 2.0 ** -18, dtype=torch.float64))
    close(lp, -want, torch.full((2,), 2.0 ** -18, dtype=torch.float64))
    close(tl, -want[:, None].expand(2, 2), torch.full((2, 2), 2.0 ** -18, dtype=torch.float64))
    assert ti.tolist() == [[vocab // 2, vocab - 1], [3, 4]]
