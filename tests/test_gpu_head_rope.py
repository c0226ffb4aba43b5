"""GPU: heads' norms, rotation and cache write (tlh_head_rope) against the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from step_refs import into_caches, rope_reference, rounded
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def build(tokens, heads, kv, hs, dtype, seed, norm=True, axes=1, rotated=None, mode=2, bs=16, far=100000, pair_axes=None):
    g, r = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    rows = torch.randn((tokens, (heads + 2 * kv) * hs), generator=g).to(dtype).cuda()
    q, k, v = rows.split([heads * hs, kv * hs, kv * hs], 1)
    pairs = (hs if rotated is None else rotated) // 2
    if pair_axes is None:
        pair_axes = [int(a) for a in r.integers(0, axes, pairs)]
        if pairs:
            pair_axes[-1] = axes - 1
    blocks = -(-tokens // bs) + 3
    c = dict(q=q.unflatten(1, (heads, hs)), k=k.unflatten(1, (kv, hs)), v=v.unflatten(1, (kv, hs)),
             positions=i32(r.integers(0, far, (axes, tokens))), freqs=N.rope_freqs(2 * pairs) if pairs else torch.empty(0, device="cuda"),
             pair_axes=pair_axes, mode=mode, eps=1e-5, factor=1.0,
             q_norm=torch.randn(hs, generator=g).cuda() if norm else None,
             k_norm=torch.randn(hs, generator=g).cuda() if norm else None,
             kc=torch.randn((blocks, kv, hs // 8, bs, 8), generator=g).half().cuda(),
             vc=torch.randn((blocks, kv, hs, bs), generator=g).half().cuda(),
             slots=torch.tensor(r.permutation(blocks * bs)[:tokens].astype(np.int64), device="cuda"))
    return c


def node_of(c):
    return N.HeadRope(c["q"].shape[1], c["k"].shape[1], c["q"].shape[2], c["freqs"], pair_axes=c["pair_axes"], mode=c["mode"],
                      eps=c["eps"], attn_factor=c["factor"])


def reference(c, dtype):
    out = [rope_reference(c[x], c[x + "_norm"], c["eps"], c["positions"].reshape(-1, len(c["q"])), c["pair_axes"],
                          c["freqs"], c["mode"], c["factor"], dtype) for x in "qk"]
    v = c["v"].cpu().double()
    return [*out, (v, rounded(v, dtype))]


def near(got, want):
    y, tol = want
    err = (got.cpu().double() - y).abs()
    assert (err <= tol).all(), float((err / tol).max())


def check(c, node=None, **kw):
    """Everything at once: the rotated heads, the plain outputs, the caches (elsewhere as they were)."""
    n, H, hs = c["q"].shape
    KV = c["k"].shape[1]
    new = lambda h: torch.full((n, h, hs), 7.0, dtype=torch.float16, device="cuda")  # noqa: E731
    qo, ko, vo, kc, vc = new(H), new(KV), new(KV), c["kc"].clone(), c["vc"].clone()
    (node or node_of(c))(c["q"], c["k"], c["v"], c["positions"], qo, q_norm=c["q_norm"], k_norm=c["k_norm"], k_out=ko,
                         v_out=vo, k_cache=kc, v_cache=vc, slots=c["slots"], **kw)
    torch.cuda.synchronize()
    for got, want in zip((qo, ko, vo), reference(c, torch.float16)):
        near(got, want)
    wk, wv = into_caches(c["kc"], c["vc"], ko, vo, c["slots"].tolist())
    assert torch.equal(kc.view(torch.int16), wk.view(torch.int16)) and torch.equal(vc.view(torch.int16), wv.view(torch.int16))
    return qo, ko, vo, kc, vc


CASES = [
    # tokens, heads, kv heads, head size, type, norm, axes, rotated, mode, block size
    (1, 32, 8, 128, torch.float32, True, 1, None, 2, 16), (1, 4, 1, 256, torch.bfloat16, True, 1, None, 2, 32),
    (7, 8, 2, 64, torch.float16, True, 1, None, 0, 8), (33, 8, 2, 80, torch.float32, False, 3, None, 2, 16),
    (130, 4, 4, 96, torch.bfloat16, True, 2, 48, 0, 8), (65, 6, 2, 112, torch.float32, True, 4, 56, 2, 32),
    (257, 28, 4, 128, torch.bfloat16, False, 3, None, 2, 16), (40, 2, 1, 192, torch.float32, True, 1, 64, 0, 16),
    (19, 5, 5, 128, torch.float16, False, 1, 2, 2, 16), (64, 8, 8, 128, torch.float32, True, 1, 0, 2, 16),
    (1031, 3, 1, 64, torch.float16, True, 2, None, 2, 32), (16, 64, 8, 256, torch.float32, True, 1, None, 2, 8),
    (3, 128, 1, 128, torch.float32, True, 1, None, 2, 16), (100, 1, 1, 80, torch.float32, True, 3, 78, 0, 8),
]


@pytest.mark.parametrize("tokens,heads,kv,hs,dtype,norm,axes,rotated,mode,bs", CASES)
def test_against_64_bits(gpu, tokens, heads, kv, hs, dtype, norm, axes, rotated, mode, bs):
    check(build(tokens, heads, kv, hs, dtype, 10 + tokens + hs, norm, axes, rotated, mode, bs))


@pytest.mark.parametrize("hs,rotated,mode", [(64, None, 2), (80, 78, 2), (128, 34, 2), (192, None, 0), (256, 250, 2)])
def test_a_tokens_heads_do_not_depend_on_the_others(gpu, hs, rotated, mode):
    """However many tokens come together, which lays heads and tokens out otherwise; a norm of one of the two."""
    whole = build(37, 9, 3, hs, torch.float32, 21, axes=2, rotated=rotated, mode=mode)
    whole["k_norm" if hs % 128 else "q_norm"] = None
    want = check(whole)
    for a, b in ((0, 1), (1, 3), (3, 8), (8, 20), (20, 37)):
        c = {**whole, **{x: whole[x][a:b] for x in ("q", "k", "v", "slots")}, "positions": whole["positions"][:, a:b].contiguous()}
        got = check(c)
        for x, y in zip(got[:3], want[:3]):
            assert torch.equal(x, y[a:b])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_bf16_out_without_a_cache(gpu, dtype):
    """For packed prompts in bf16; also q alone, and a norm of one of the two."""
    c = build(70, 8, 2, 128, dtype, 20)
    node = node_of(c)
    outs = [torch.full(c[x].shape, 7.0, dtype=torch.bfloat16, device="cuda") for x in "qkv"]
    node(c["q"], c["k"], c["v"], c["positions"], outs[0], c["q_norm"], c["k_norm"], outs[1], outs[2])
    for got, want in zip(outs, reference(c, torch.bfloat16)):
        near(got, want)
    alone = torch.empty_like(outs[0])
    node(c["q"], c["k"], c["v"], c["positions"], alone, c["q_norm"], c["k_norm"])
    assert torch.equal(alone, outs[0])
    c["q_norm"] = None
    node(c["q"], c["k"], c["v"], c["positions"], outs[0], None, c["k_norm"], outs[1])
    for got, want in zip(outs[:2], reference(c, torch.bfloat16)):
        near(got, want)


@pytest.mark.parametrize("far", [1 << 20, 1 << 30, (1 << 31) - 1])
def test_far_positions_keep_their_angle(gpu, far):
    c = build(50, 4, 2, 128, torch.float32, 21, far=far)
    check(c)
    c["positions"] = -c["positions"]
    check(c)


def test_sections_and_interleaved_axes(gpu):
    for interleaved in (False, True):
        axes = N.rope_sections((16, 24, 24), interleaved)
        assert [axes.count(a) for a in range(3)] == ([16, 24, 24] if not interleaved else [axes.count(0), 21, 21])
        check(build(45, 8, 2, 128, torch.float32, 22, axes=3, pair_axes=axes))
    assert N.rope_sections((3, 1, 2), True) == [0, 1, 2, 0, 0, 2]


def test_the_axes_are_those_of_one_when_positions_agree(gpu):
    """Text under three axes is text under one, bit for bit."""
    c = build(45, 8, 2, 128, torch.float32, 23)
    want = check(c)
    c["pair_axes"], c["positions"] = N.rope_sections((16, 24, 24)), c["positions"].repeat(3, 1)
    assert all(torch.equal(a, b) for a, b in zip(check(c), want))


def test_attention_factor_and_frequencies(gpu):
    c = build(45, 8, 2, 128, torch.float32, 24)
    c["factor"] = 1.3
    factors = torch.linspace(1, 8, 64)
    c["freqs"] = N.rope_freqs(128, 500000.0, 0.25, factors)
    want = (0.25 * 500000.0 ** (-2 * torch.arange(64, dtype=torch.float64) / 128) / factors.double()).float()
    assert torch.equal(c["freqs"].cpu(), want)
    check(c)


def test_agrees_with_the_nodes_it_joins(gpu):
    """RMS norm, ROPE and the cache write as nodes of their own, at positions where f32 angles are fine."""
    c = build(33, 8, 2, 128, torch.float32, 25, far=50)
    qo, ko, vo, kc, vc = check(c)
    for x, got in (("q", qo), ("k", ko)):
        y = N.mul(N.rms_norm(c[x].contiguous(), c["eps"]), c[x + "_norm"])
        y = N.rope(y, c["positions"][0], 128, mode=2)
        # f32 angles of up to 50 are off by 2^-19, on top of what either rounds
        assert ((y - got.float()).abs() <= 2.0 ** -11 * y.abs() + 2.0 ** -15 * y.abs().amax()).all()
    kc2, vc2 = c["kc"].clone(), c["vc"].clone()
    N.reshape_and_cache(ko.reshape(33, -1), vo.reshape(33, -1), kc2, vc2, c["slots"], 2, 16)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_slots_that_write_nothing(gpu):
    c = build(9, 8, 2, 128, torch.float32, 26)
    pool = c["kc"].shape[0] * 16
    c["slots"][:] = torch.tensor([-1, 3, pool, 1 << 62, -(1 << 62), pool - 1, 0, pool + 5, 17])
    check(c)


def test_consecutive_slots_and_broken_runs(gpu):
    """As sequences leave them: runs that start inside a page, end inside one, and jump."""
    for bs in (8, 16, 32):
        c = build(200, 4, 2, 64, torch.float32, 27, bs=bs)
        ids = np.random.default_rng(27).permutation(c["kc"].shape[0])
        place = np.concatenate([5 + np.arange(70), 100 + np.arange(1), 110 + np.arange(60), 80 + np.arange(9)])
        place = np.concatenate([place, np.setdiff1d(np.arange(len(ids) * bs), place)])[:200]
        c["slots"] = torch.tensor(ids[place // bs].astype(np.int64) * bs + place % bs, device="cuda")
        check(c)


def test_separate_tensors_and_strides(gpu):
    """q, k, v and the outputs at strides of their own; what lies between the outputs' heads stays."""
    c = build(21, 4, 2, 128, torch.float16, 28)
    want = check(c)
    wide = {}
    for x, extra in (("q", 1), ("k", 3), ("v", 2)):
        t = torch.randn((21, c[x].shape[1] + extra, 128), device="cuda").half()
        t[:, :c[x].shape[1]] = c[x]
        wide[x] = t[:, :c[x].shape[1]]
    out = torch.full((21, 12, 128), 7.0, dtype=torch.float16, device="cuda")
    kc, vc = c["kc"].clone(), c["vc"].clone()
    node_of(c)(wide["q"], wide["k"], wide["v"], c["positions"], out[:, 1:5], c["q_norm"], c["k_norm"], out[:, 6:8],
               out[:, 9:11], kc, vc, c["slots"])
    got = (out[:, 1:5], out[:, 6:8], out[:, 9:11], kc, vc)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (out[:, [0, 5, 8, 11]] == 7).all()


def test_values_that_are_not_finite_stay_in_their_head(gpu):
    for bad in (float("nan"), float("inf")):
        c = build(12, 4, 2, 128, torch.float32, 29)
        want = check(c)
        c["q"][3, 1, 5], c["k"][7, 0, 100], c["v"][2, 1, 9] = bad, bad, bad
        qo, ko, vo = (torch.empty(c[x].shape, dtype=torch.float16, device="cuda") for x in "qkv")
        node_of(c)(c["q"], c["k"], c["v"], c["positions"], qo, c["q_norm"], c["k_norm"], ko, vo)
        for got, w, at in ((qo, want[0], (3, 1)), (ko, want[1], (7, 0))):
            assert torch.isnan(got[at]).any()
            got[at] = w[at]
            assert torch.equal(got, w)
        assert not torch.isfinite(vo[2, 1, 9])
        vo[2, 1, 9] = want[2][2, 1, 9]
        assert torch.equal(vo, want[2])


def test_small_and_large_heads(gpu):
    """Heads of zeros (the eps decides), near f32's smallest and of 1e15."""
    c = build(6, 4, 2, 128, torch.float32, 30)
    c["q"][0], c["k"][1] = 0.0, 0.0
    c["q"][2] *= 1e-30
    c["k"][3] *= 1e15
    c["q"][4] *= 1e15
    check(c)


def test_a_pool_past_32_bits(gpu):
    kv, hs, bs = 8, 128, 16
    blocks = (1 << 32) // (kv * hs * bs * 2) + 40
    c = build(37, 8, kv, hs, torch.float32, 31)
    n = c["kc"].shape[0]
    kc = torch.empty((blocks, kv, hs // 8, bs, 8), dtype=torch.float16, device="cuda")
    vc = torch.empty((blocks, kv, hs, bs), dtype=torch.float16, device="cuda")
    kc[-n:], vc[-n:] = c["kc"], c["vc"]
    want = check(c)
    node_of(c)(c["q"], c["k"], c["v"], c["positions"], torch.empty_like(want[0]), c["q_norm"], c["k_norm"], k_cache=kc,
               v_cache=vc, slots=c["slots"] + (blocks - n) * bs)
    assert torch.equal(kc[-n:], want[3]) and torch.equal(vc[-n:], want[4])


def test_no_tokens(gpu):
    c = build(3, 4, 2, 128, torch.float32, 32)
    kc = c["kc"].clone()
    out = torch.full((3, 4, 128), 7.0, dtype=torch.float16, device="cuda")
    node_of(c)(c["q"][:0], c["k"][:0], c["v"][:0], c["positions"][:, :0].contiguous(), out[:0], c["q_norm"], c["k_norm"],
               k_cache=kc, v_cache=c["vc"], slots=c["slots"][:0])
    assert (out == 7).all() and torch.equal(kc, c["kc"])


def test_streams_and_graphs(gpu):
    c = build(90, 8, 2, 128, torch.float32, 33)
    node, want = node_of(c), check(c)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream, 0):
        got = check(c, node, stream=stream)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    out, kc, vc = torch.zeros_like(want[0]), c["kc"].clone(), c["vc"].clone()
    args = (c["q"], c["k"], c["v"], c["positions"], out, c["q_norm"], c["k_norm"], None, None, kc, vc, c["slots"])
    node(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        node(*args)
    for i in range(4):
        c["q"].copy_(torch.randn_like(c["q"])), c["k"].copy_(torch.randn_like(c["k"]))
        c["positions"].add_(17)
        out.zero_(), kc.copy_(c["kc"]), vc.copy_(c["vc"])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = check(c)
        assert torch.equal(out, want[0]) and torch.equal(kc, want[3]) and torch.equal(vc, want[4])


@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("hs,rotated", [(128, 64), (80, 34), (192, 0), (256, 250), (64, 2), (112, 104)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_dims_that_are_not_rotated_pass_through(gpu, bad, hs, rotated, mode):
    """One that is not finite stays in its place, also beside one that is."""
    c = build(21, 4, 2, hs, torch.float32, 34, norm=False, rotated=rotated, mode=mode)
    want = check(c)
    at = [(3, 1, rotated), (5, 0, rotated + 1), (7, 1, hs - 1), (9, 0, hs - 2)]
    c["q"], c["k"] = c["q"].clone(), c["k"].clone()
    for t, h, d in at:
        c["q"][t, h, d] = c["k"][t, h, d] = bad
    qo, ko = (torch.empty(c[x].shape, dtype=torch.float16, device="cuda") for x in "qk")
    kc, vc = c["kc"].clone(), c["vc"].clone()
    node_of(c)(c["q"], c["k"], c["v"], c["positions"], qo, k_out=ko, k_cache=kc, v_cache=vc, slots=c["slots"])
    wq, wk = want[0].clone(), want[1].clone()
    for t, h, d in at:
        wq[t, h, d] = wk[t, h, d] = bad
    for got, w in ((qo, wq), (ko, wk)):
        assert torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(w))
    wc, _ = into_caches(c["kc"], c["vc"], ko, c["v"].half(), c["slots"].tolist())
    assert torch.equal(kc.view(torch.int16), wc.view(torch.int16))
