"""What a serving step's operators refuse, on the CPU: nothing here reaches a launch."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from tensorlisp_amd import native as N

# addresses that no call may reach: every test below is refused before they are used
P, FAR, BIG = 0x10000, 1 << 44, 1 << 62


def status(fn, *args):
    st = fn(*args)
    return N.STATUS[st], N.lib().tlh_last_error().decode()


def fill(a, kw):
    for f, v in kw.items():
        setattr(a, f, v)
    return a


# --------------------------------------------------------- chunk attention
def chunk(**kw):
    a = N.TlhChunkArgs()
    for i, f in enumerate(("out", "q", "k_cache", "v_cache", "block_tables", "context_lens", "row_starts")):
        setattr(a, f, P + i * FAR)
    a.num_blocks, a.num_seqs, a.num_rows, a.max_rows = 100, 2, 10, 8
    a.num_heads, a.num_kv_heads, a.head_size, a.block_size = 8, 2, 128, 16
    a.out_stride = a.q_stride = 1024
    a.max_blocks_per_seq, a.max_context_len, a.scale = 8, 128, 0.1
    return fill(a, kw)


@pytest.mark.parametrize("kw,want", [
    (dict(head_size=100), "INVALID"), (dict(block_size=24), "INVALID"), (dict(num_heads=9), "INVALID"),
    (dict(num_kv_heads=0), "INVALID"), (dict(max_rows=-1), "INVALID"), (dict(num_seqs=-1), "INVALID"),
    (dict(num_seqs=65536), "INVALID"), (dict(num_rows=-1), "INVALID"), (dict(num_blocks=-1), "INVALID"),
    (dict(max_context_len=129), "INVALID"), (dict(max_context_len=-1), "INVALID"), (dict(window=-1), "INVALID"),
    (dict(max_context_len=(1 << 30) + 1, max_blocks_per_seq=1 << 27), "INVALID"), (dict(max_blocks_per_seq=-1), "INVALID"),
    (dict(num_rows=1 << 30), "INVALID"), (dict(q_stride=1016), "INVALID"), (dict(out_stride=1028), "INVALID"),
    (dict(q_stride=1 << 40), "INVALID"), (dict(out_stride=-1024), "INVALID"), (dict(k_cache=0), "INVALID"),
    (dict(block_tables=0), "INVALID"), (dict(row_starts=0), "INVALID"), (dict(context_lens=P + 1), "INVALID"),
    (dict(q=P + 8), "INVALID"), (dict(out=P + 4), "INVALID"), (dict(v_cache=P + 4), "INVALID"), (dict(out=0), "INVALID"),
    (dict(num_seqs=0), "OK"), (dict(num_rows=0), "OK"), (dict(max_rows=0, q=0), "OK"),
])
def test_chunk_attention_refusals(kw, want):
    assert status(N.lib().tlh_chunk_attention, C.byref(chunk(**kw)), P, BIG, None)[0] == want


@pytest.mark.parametrize("value", [-1, 2, 1 << 30])
def test_f16_weights_is_one_or_the_other(value):
    st, text = status(N.lib().tlh_chunk_attention, C.byref(chunk(f16_weights=value)), P, BIG, None)
    assert st == "INVALID" and "f16_weights" in text
    n = C.c_size_t()
    assert status(N.lib().tlh_chunk_attention_scratch_bytes, C.byref(chunk(f16_weights=value)), C.byref(n))[0] == "INVALID"
    assert chunk_size(f16_weights=1) == chunk_size(f16_weights=0)


def chunk_size(**kw):
    n = C.c_size_t()
    assert status(N.lib().tlh_chunk_attention_scratch_bytes, C.byref(chunk(**kw)), C.byref(n))[0] == "OK"
    return n.value


def test_chunk_attention_scratch_refusals():
    n = C.c_size_t()
    a = chunk(max_context_len=8192, max_blocks_per_seq=512)
    assert status(N.lib().tlh_chunk_attention_scratch_bytes, C.byref(a), None)[0] == "INVALID"
    assert status(N.lib().tlh_chunk_attention_scratch_bytes, None, C.byref(n))[0] == "INVALID"
    assert status(N.lib().tlh_chunk_attention_scratch_bytes, C.byref(chunk(head_size=1)), C.byref(n))[0] == "INVALID"
    need = chunk_size(max_context_len=8192, max_blocks_per_seq=512)
    if need:
        for scratch, nbytes in ((P, need - 1), (None, need), (P + 8, need)):
            st, text = status(N.lib().tlh_chunk_attention, C.byref(a), scratch, nbytes, None)
            assert st == "INVALID" and "scratch" in text


def test_chunk_attention_scratch_never_shrinks():
    """One buffer for the largest batch, rows and context serves every smaller call."""
    big = dict(max_blocks_per_seq=8192)
    for hs in (64, 128, 256):
        for seqs in (1, 3, 32, 200):
            for ctx in (1, 100, 4096, 100000):
                for most in (1, 16, 17, 700):
                    s = [chunk_size(num_seqs=seqs, num_rows=r, max_rows=most, max_context_len=ctx, head_size=hs, **big)
                         for r in (1, 8, 9, 64, 300, 2000, 50000)]
                    assert s == sorted(s), (seqs, ctx, most, s)
        for name, values in (("num_seqs", range(1, 80)), ("max_rows", range(1, 200, 3)),
                             ("max_context_len", range(0, 20000, 173))):
            for rows in (3, 300):
                s = [chunk_size(**{**dict(num_rows=rows, max_rows=300, max_context_len=9000), name: v}, head_size=hs, **big)
                     for v in values]
                assert s == sorted(s), name


def test_chunk_attention_scratch_never_shrinks_under_a_window():
    """A tile more or less that a block of few or of many rows sees: contexts around the window, counts around where one
    block becomes the other."""
    big = dict(max_blocks_per_seq=8192)
    for window in (1, 16, 64, 65, 100, 1024):
        for ctx in {1, 50, 90, window, *range(max(1, window - 3), window + 200, 7)}:
            for G in (1, 4, 8):
                s = [chunk_size(num_seqs=1, num_rows=r, max_rows=40, max_context_len=ctx, window=window, num_heads=8,
                                num_kv_heads=8 // G, **big) for r in range(1, 41)]
                assert s == sorted(s), (window, ctx, G, s)
                s = [chunk_size(num_seqs=2, num_rows=200, max_rows=m, max_context_len=ctx, window=window, num_heads=8,
                                num_kv_heads=8 // G, **big) for m in range(1, 101)]
                assert s == sorted(s), (window, ctx, G, s)
        s = [chunk_size(num_rows=300, max_rows=300, max_context_len=ctx, window=window, **big) for ctx in range(0, 3000, 13)]
        assert s == sorted(s), window


def test_chunk_attention_out_must_be_apart():
    """(Calls that pass are refused behind that, for want of scratch: more rows than any split leaves without.)"""
    row, n = 8 * 128 * 2, 10
    pool = 100 * 2 * 128 * 16 * 2
    big = dict(max_context_len=8192, max_blocks_per_seq=512)
    if not chunk_size(**big):
        pytest.skip("no scratch is needed, and calls that pass would launch")

    def refused(out, **kw):
        st, text = status(N.lib().tlh_chunk_attention, C.byref(chunk(out=out, **{**big, **kw})), None, 0, None)
        assert st == "INVALID" and ("overlaps" in text or "scratch" in text), text
        return "overlaps" in text

    at = P + FAR  # q's place
    for by in (0, 16, -16, (n - 1) * row, 1 - n * row + 15):
        assert refused(at + by), by
    assert not refused(at + n * row) and not refused(at - n * row)
    for base in (P + 2 * FAR, P + 3 * FAR):
        assert refused(base) and refused(base + pool - 16) and refused(base - n * row + 16)
        assert not refused(base + pool) and not refused(base - n * row)
    # columns of the same rows
    wide = dict(q_stride=4096, out_stride=4096)
    assert not refused(at + row, **wide) and not refused(at + 2 * row, **wide) and refused(at + row - 16, **wide)
    assert refused(at + 8192 - row + 16, **wide)


def test_chunk_attention_out_and_scratch_must_be_apart_from_what_is_read():
    """Workgroups read the tables, lengths and starts while others write out already, and partials while others write
    theirs. (Every call here is refused: those that are apart, for want of scratch.)"""
    big = dict(max_context_len=8192, max_blocks_per_seq=512)
    need, n = chunk_size(**big), 10 * 8 * 128 * 2
    size = dict(out=n, q=n, k_cache=100 * 2 * 128 * 32, v_cache=100 * 2 * 128 * 32, block_tables=2 * 512 * 4, context_lens=8,
                row_starts=12)
    at = {f: P + i * FAR for i, f in enumerate(size)}
    for x in ("block_tables", "context_lens", "row_starts"):
        for place in (at[x] - n + 16, at[x], at[x] + (size[x] - 1) // 16 * 16):
            st, text = status(N.lib().tlh_chunk_attention, C.byref(chunk(**{**big, "out": place})), None, 0, None)
            assert st == "INVALID" and "overlaps" in text, (x, text)
        for place in (at[x] - n, at[x] + (size[x] + 15) // 16 * 16):
            st, text = status(N.lib().tlh_chunk_attention, C.byref(chunk(**{**big, "out": place})), None, 0, None)
            assert st == "INVALID" and "overlaps" not in text, (x, text)
    for x in size:
        for place in ((at[x] - need + 16) // 16 * 16, at[x], at[x] + (size[x] - 1) // 16 * 16):
            st, text = status(N.lib().tlh_chunk_attention, C.byref(chunk(**big)), place, need, None)
            assert st == "INVALID" and "overlaps the scratch" in text, (x, text)


# --------------------------------------------------------------- head rope
ROPE = ("q", "k", "v", "positions", "freqs", "q_norm", "k_norm", "q_out", "k_out", "v_out", "k_cache", "v_cache", "slots")


def rope(**kw):
    a = N.TlhHeadRopeArgs()
    for i, f in enumerate(ROPE):
        setattr(a, f, P + i * FAR)
    a.q_stride = a.q_out_stride = 1024
    a.k_stride = a.v_stride = a.k_out_stride = a.v_out_stride = 256
    a.num_blocks, a.type, a.out_type, a.num_tokens = 100, N.F16, N.F16, 3
    a.num_heads, a.num_kv_heads, a.head_size, a.block_size, a.n_dims, a.mode, a.num_axes = 8, 2, 128, 16, 128, 2, 1
    a.eps, a.attn_factor = 1e-6, 1.0
    return fill(a, kw)


def axes(*values):
    return (C.c_uint8 * 128)(*values)


@pytest.mark.parametrize("kw,want", [
    (dict(type=N.Q8_0), "UNSUPPORTED"), (dict(out_type=N.F32), "UNSUPPORTED"), (dict(out_type=N.BF16), "UNSUPPORTED"),
    (dict(head_size=72), "INVALID"), (dict(num_heads=7), "INVALID"), (dict(num_kv_heads=0), "INVALID"),
    (dict(num_tokens=-1), "INVALID"), (dict(n_dims=130), "INVALID"), (dict(n_dims=63), "INVALID"), (dict(n_dims=-2), "INVALID"),
    (dict(mode=1), "INVALID"), (dict(num_axes=0), "INVALID"), (dict(num_axes=5), "INVALID"),
    (dict(pair_axis=axes(*([0] * 63), 1)), "INVALID"), (dict(num_axes=2, pair_axis=axes(0, 2)), "INVALID"),
    (dict(block_size=24), "INVALID"), (dict(num_blocks=-1), "INVALID"), (dict(num_blocks=BIG), "INVALID"),
    (dict(k_cache=0), "INVALID"), (dict(slots=0), "INVALID"), (dict(k_cache=0, v_cache=0), "INVALID"),
    (dict(q=0), "INVALID"), (dict(v=0), "INVALID"), (dict(q_out=0), "INVALID"), (dict(positions=0), "INVALID"),
    (dict(freqs=0), "INVALID"), (dict(q=P + 8), "INVALID"), (dict(k_out=P + 8), "INVALID"), (dict(v_cache=P + 2), "INVALID"),
    (dict(q_norm=P + 4), "INVALID"), (dict(slots=P + 4), "INVALID"), (dict(positions=P + 2), "INVALID"),
    (dict(q_stride=1016), "INVALID"), (dict(k_stride=260), "INVALID"), (dict(v_out_stride=128), "INVALID"),
    (dict(type=N.F32, k_stride=258), "INVALID"), (dict(q_stride=1 << 40), "INVALID"),
    (dict(num_tokens=0), "OK"), (dict(num_tokens=0, q=0, slots=P + 4), "OK"),
])
def test_head_rope_refusals(kw, want):
    assert status(N.lib().tlh_head_rope, C.byref(rope(**kw)), None)[0] == want


def test_head_rope_outputs_must_be_apart():
    """Every pair that may not overlap does here by 16 bytes, from either side. (Calls that pass would launch; that the
    ones beside each other do is tested where there is a GPU.)"""
    n, hs, es = 3, 128, 2
    size = dict(q=n * 8 * hs * es, k=n * 2 * hs * es, v=n * 2 * hs * es, positions=4 * n, freqs=256, q_norm=512, k_norm=512,
                q_out=n * 8 * hs * 2, k_out=n * 2 * hs * 2, v_out=n * 2 * hs * 2, k_cache=100 * 2 * hs * 32,
                v_cache=100 * 2 * hs * 32, slots=8 * n)
    at = {f: P + i * FAR for i, f in enumerate(ROPE)}
    for o in ("q_out", "k_out", "v_out", "k_cache", "v_cache"):
        for x in ROPE:
            if x == o:
                continue
            for place in (at[x] - size[o] + 16, at[x], at[x] + (size[x] - 1) // 16 * 16):
                st, text = status(N.lib().tlh_head_rope, C.byref(rope(**{o: place})), None)
                assert st == "INVALID" and "overlap" in text, (o, x, place - at[x], text)


# ------------------------------------------------------------ draft verify
VERIFY = ("target", "draft", "tokens", "draft_starts", "temperatures", "accept_at", "sample_at", "accepted", "out_tokens",
          "accept_probs")


def verify(**kw):
    a = N.TlhVerifyArgs()
    for i, f in enumerate(VERIFY):
        setattr(a, f, P + i * FAR)
    a.type, a.num_seqs, a.num_drafts, a.max_drafts, a.vocab = N.F32, 2, 7, 5, 1000
    a.target_stride = a.draft_stride = 1000
    return fill(a, kw)


@pytest.mark.parametrize("kw,want", [
    (dict(type=N.Q8_0), "UNSUPPORTED"), (dict(num_seqs=-1), "INVALID"), (dict(num_seqs=65536), "INVALID"),
    (dict(num_drafts=-1), "INVALID"), (dict(num_drafts=(1 << 23) + 1), "INVALID"), (dict(vocab=0), "INVALID"),
    (dict(vocab=1000001, target_stride=BIG, draft_stride=BIG), "INVALID"), (dict(max_drafts=-1), "INVALID"),
    (dict(max_drafts=1025), "INVALID"), (dict(target_stride=999), "INVALID"), (dict(draft_stride=999), "INVALID"),
    (dict(target_stride=1 << 40), "INVALID"), (dict(draft_stride=1 << 40), "INVALID"),
    (dict(target=0), "INVALID"), (dict(tokens=0), "INVALID"), (dict(draft_starts=0), "INVALID"),
    (dict(temperatures=0), "INVALID"), (dict(accept_at=0), "INVALID"), (dict(sample_at=0), "INVALID"),
    (dict(accepted=0), "INVALID"), (dict(out_tokens=0), "INVALID"), (dict(target=P + 2), "INVALID"),
    (dict(draft=P + FAR + 1), "INVALID"), (dict(type=N.F16, target=P + 1), "INVALID"), (dict(accept_probs=P + 2), "INVALID"),
    (dict(num_seqs=0), "OK"), (dict(num_seqs=0, target=0), "OK"),
])
def test_draft_verify_refusals(kw, want):
    assert status(N.lib().tlh_draft_verify, C.byref(verify(**kw)), P, BIG, None)[0] == want


def verify_size(**kw):
    n = C.c_size_t()
    assert status(N.lib().tlh_draft_verify_scratch_bytes, C.byref(verify(**kw)), C.byref(n))[0] == "OK"
    return n.value


def test_draft_verify_scratch():
    n, need = C.c_size_t(), verify_size()
    assert need > 0
    assert status(N.lib().tlh_draft_verify_scratch_bytes, C.byref(verify()), None)[0] == "INVALID"
    assert status(N.lib().tlh_draft_verify_scratch_bytes, None, C.byref(n))[0] == "INVALID"
    for scratch, nbytes in ((P, need - 1), (None, need), (P + 8, need)):
        st, text = status(N.lib().tlh_draft_verify, C.byref(verify()), scratch, nbytes, None)
        assert st == "INVALID" and "scratch" in text
    for vocab in (1, 5000, 32000, 128256, 1000000):
        wide = dict(vocab=vocab, target_stride=vocab, draft_stride=vocab)
        for draft in (0, P):
            for seqs in (1, 32, 500):
                s = [verify_size(num_drafts=r, num_seqs=seqs, draft=draft, **wide) for r in range(0, 700, 7)]
                assert s == sorted(s)
            s = [verify_size(num_drafts=10, num_seqs=r, draft=draft, **wide) for r in range(0, 700, 7)]
            assert s == sorted(s)


def test_draft_verify_outputs_must_be_apart():
    size = dict(target=9 * 4000, draft=7 * 4000, tokens=28, draft_starts=12, temperatures=8, accept_at=28, sample_at=8,
                accepted=8, out_tokens=48, accept_probs=28)
    at = {f: P + i * FAR for i, f in enumerate(VERIFY)}
    for o in ("accepted", "out_tokens", "accept_probs"):
        for x in VERIFY:
            if x == o:
                continue
            for place in (at[x] - size[o] + 4, at[x], at[x] + size[x] - 4):
                st, text = status(N.lib().tlh_draft_verify, C.byref(verify(**{o: place})), None, 0, None)
                assert st == "INVALID" and "overlap" in text, (o, x, place - at[x])
            for place in (at[x] - size[o], at[x] + size[x]):
                st, text = status(N.lib().tlh_draft_verify, C.byref(verify(**{o: place})), None, 0, None)
                assert st == "INVALID" and "scratch" in text, (o, x, place - at[x])


def test_draft_verify_scratch_must_be_apart():
    size = dict(target=9 * 4000, draft=7 * 4000, tokens=28, draft_starts=12, temperatures=8, accept_at=28, sample_at=8,
                accepted=8, out_tokens=48, accept_probs=28)
    need, at = verify_size(), {f: P + i * FAR for i, f in enumerate(VERIFY)}
    for x in VERIFY:
        for place in ((at[x] - need + 16) // 16 * 16, at[x], at[x] + (size[x] - 1) // 16 * 16):
            st, text = status(N.lib().tlh_draft_verify, C.byref(verify()), place, need, None)
            assert st == "INVALID" and "overlaps the scratch" in text, (x, text)


# ------------------------------------------------- the Python entry points
def f16(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_chunk_attention_names_the_tensor():
    kc, vc = f16(5, 2, 8, 16, 8), f16(5, 2, 64, 16)
    node = N.ChunkAttention(3, 10, 8, 8, 2, 64, 16, 4, 64, 0.1, device="cpu")

    def call(n, seqs, **kw):
        a = dict(out=f16(n, 8, 64), q=f16(n, 8, 64), k_cache=kc, v_cache=vc, block_tables=i32(seqs, 4),
                 context_lens=i32(seqs), row_starts=i32(seqs + 1))
        node(**{**a, **kw})

    for n, seqs in ((10, 3), (7, 3), (10, 1), (1, 1), (0, 3), (0, 0)):
        with pytest.raises(ValueError, match="on the GPU"):  # everything before that fits
            call(n, seqs)
    for n, seqs in ((11, 3), (10, 4)):
        with pytest.raises(ValueError, match="up to"):
            call(n, seqs)
    for name, bad in (("q", f16(6, 8, 64)), ("q", f16(7, 8, 64).float()), ("out", f16(7, 8, 128)), ("k_cache", kc.float()),
                      ("v_cache", vc[:4]), ("context_lens", i32(3)), ("row_starts", i32(2)), ("block_tables", i32(2, 3)),
                      ("q", f16(8, 7, 64).transpose(0, 1))):
        with pytest.raises(ValueError, match=name):
            call(7, 2, **{name: bad})
    with pytest.raises(N.TlhError, match="bad counts"):
        N.ChunkAttention(3, 10, 8, 8, 2, 64, 16, 4, 64, 0.1, window=-1, device="cpu")


def test_head_rope_names_the_tensor():
    node = N.HeadRope(8, 2, 64, torch.zeros(32), pair_axes=[0] * 16 + [1] * 16)
    good = dict(q=f16(3, 8, 64), k=f16(3, 2, 64), v=f16(3, 2, 64), positions=i32(2, 3), q_out=f16(3, 8, 64),
                q_norm=torch.zeros(64), k_norm=torch.zeros(64), k_out=f16(3, 2, 64), v_out=f16(3, 2, 64),
                k_cache=f16(5, 2, 8, 16, 8), v_cache=f16(5, 2, 64, 16), slots=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="on the GPU"):
        node(**good)
    for name, bad in (("q", f16(3, 7, 64)), ("k", f16(2, 2, 64)), ("v", f16(3, 2, 64).float()), ("positions", i32(3)),
                      ("positions", i32(1, 3)), ("q_out", f16(3, 8, 32)), ("q_out", f16(3, 16)[:, ::2]), ("q_norm", torch.zeros(32)),
                      ("k_norm", f16(64)), ("k_out", f16(3, 2, 64).bfloat16()), ("v_out", f16(4, 2, 64)),
                      ("k_cache", f16(5, 2, 8, 8, 8)), ("v_cache", f16(4, 2, 64, 16)), ("slots", i32(3)), ("slots", None),
                      ("k_cache", None), ("q", f16(8, 3, 64).transpose(0, 1))):
        with pytest.raises(ValueError, match=name):
            node(**{**good, name: bad})
    for bad in ([0] * 31, [0] * 31 + [4], [0] * 31 + [-1]):
        with pytest.raises(ValueError, match="pair_axes"):
            N.HeadRope(8, 2, 64, torch.zeros(32), pair_axes=bad)
    with pytest.raises(ValueError, match="freqs"):
        N.HeadRope(8, 2, 64, torch.zeros(32).double())
    with pytest.raises(ValueError, match="pair_axes"):
        N.HeadRope(8, 2, 64, torch.zeros(129))
    one = N.HeadRope(8, 2, 64, torch.zeros(32))
    for positions in (i32(3), i32(1, 3)):
        with pytest.raises(ValueError, match="on the GPU"):
            one(**{**good, "positions": positions})


def test_draft_verify_names_the_tensor():
    node = N.DraftVerify(2, 7, 5, 100, device="cpu")
    f = lambda *s: torch.zeros(s)  # noqa: E731

    def call(r=7, s=2, node=node, **kw):
        a = dict(target=f(r + s, 100), draft=f(r, 100), tokens=i32(r), draft_starts=i32(s + 1), temperatures=f(s),
                 accept_at=f(r), sample_at=f(s), accepted=i32(s), out_tokens=i32(s, 6), accept_probs=f(r))
        node(**{**a, **kw})

    for r, s in ((7, 2), (3, 2), (0, 1), (7, 1)):
        with pytest.raises(ValueError, match="on the GPU"):
            call(r, s)
    for r, s in ((8, 2), (7, 3)):
        with pytest.raises(ValueError, match="up to"):
            call(r, s)
    for name, bad in (("target", f(8, 100)), ("target", f(9, 99)), ("draft", f(7, 100).half()), ("draft", None),
                      ("draft", f(100, 7).t()), ("draft_starts", i32(2)), ("accept_at", f(6)), ("sample_at", i32(2)),
                      ("accepted", i32(3)), ("out_tokens", i32(2, 5)), ("accept_probs", f(6))):
        with pytest.raises(ValueError, match=name.replace("draft", "draft")):
            call(**{name: bad})
    with pytest.raises(ValueError, match="drafting model"):
        call(node=N.DraftVerify(2, 7, 5, 100, drafter=False, device="cpu"))
    with pytest.raises(N.TlhError, match="max_drafts"):
        N.DraftVerify(2, 7, 1025, 100, device="cpu")
    with pytest.raises(N.TlhError, match="type"):
        N.DraftVerify(2, 7, 5, 100, dtype=torch.float64, device="cpu")


@pytest.mark.parametrize("more", [1 << 31, (1 << 32) + 4, -(1 << 32) + 4])
def test_counts_past_32_bits_are_refused(more):
    names = ("num_seqs", "num_rows", "max_rows", "num_heads", "num_kv_heads", "head_size", "block_size",
             "max_blocks_per_seq", "max_context_len", "window")
    good = dict(zip(names, (1, 3, 3, 8, 2, 64, 16, 4, 64, 0)))
    N.ChunkAttention(**good, scale=0.1, device="cpu")
    for name in names:
        with pytest.raises(ValueError, match=f"{name} .* 32 bits"):
            N.ChunkAttention(**{**good, name: more}, scale=0.1, device="cpu")
    for name in ("num_heads", "num_kv_heads", "head_size", "mode"):
        args = dict(num_heads=8, num_kv_heads=2, head_size=64, mode=2)
        with pytest.raises(ValueError, match=f"{name} .* 32 bits"):
            N.HeadRope(**{**args, name: more}, freqs=torch.zeros(32))
    for name in ("num_seqs", "num_drafts", "max_drafts", "vocab"):
        args = dict(num_seqs=2, num_drafts=7, max_drafts=5, vocab=100)
        with pytest.raises(ValueError, match=f"{name} .* 32 bits"):
            N.DraftVerify(**{**args, name: more}, device="cpu")
