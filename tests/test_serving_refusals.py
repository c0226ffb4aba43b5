"""What the serving operators refuse, on the CPU: nothing here reaches a launch."""
from __future__ import annotations

import ctypes as C
import random

import pytest
import torch

from tensorlisp_amd import native as N

# an address that no call may reach: every test below is refused before it is used
P = 0x10000


def status(fn, *args):
    st = fn(*args)
    return N.STATUS[st], N.lib().tlh_last_error().decode()


def packed(**kw):
    a = N.TlhPackedArgs()
    for f in ("out", "q", "k", "v", "seq_starts"):
        setattr(a, f, P)
    a.out_stride = a.q_stride = 8 * 64
    a.k_stride = a.v_stride = 2 * 64
    a.type, a.num_seqs, a.num_tokens, a.max_seq_len = N.F16, 1, 10, 10
    a.num_heads, a.num_kv_heads, a.head_size, a.scale = 8, 2, 64, 0.125
    for f, v in kw.items():
        setattr(a, f, v)
    return a


@pytest.mark.parametrize("kw,want", [
    (dict(type=N.F32), "UNSUPPORTED"), (dict(type=N.Q8_0), "UNSUPPORTED"), (dict(head_size=72), "INVALID"),
    (dict(num_heads=7), "INVALID"), (dict(num_kv_heads=0), "INVALID"), (dict(num_seqs=-1), "INVALID"),
    (dict(num_tokens=-1), "INVALID"), (dict(max_seq_len=-1), "INVALID"), (dict(q_stride=511), "INVALID"),
    (dict(q_stride=508), "INVALID"), (dict(out_stride=516), "INVALID"), (dict(k_stride=120), "INVALID"),
    (dict(v_stride=-128), "INVALID"), (dict(q=0), "INVALID"), (dict(out=0), "INVALID"), (dict(seq_starts=0), "INVALID"),
    (dict(q=P + 8), "INVALID"), (dict(v=P + 2), "INVALID"), (dict(seq_starts=P + 2), "INVALID"),
    (dict(num_seqs=0), "OK"), (dict(num_tokens=0), "OK"), (dict(max_seq_len=0, q=0), "OK"),
])
def test_packed_attention_refusals(kw, want):
    assert status(N.lib().tlh_packed_attention, C.byref(packed(**kw)), None)[0] == want


def tree(**kw):
    a = N.TlhTreeArgs()
    for f in ("out", "q", "k_cache", "v_cache", "block_tables", "context_lens", "draft_starts", "draft_masks"):
        setattr(a, f, P)
    a.num_blocks, a.num_seqs, a.num_rows, a.max_drafts = 100, 2, 10, 8
    a.num_heads, a.num_kv_heads, a.head_size, a.block_size = 8, 2, 128, 16
    a.max_blocks_per_seq, a.max_context_len, a.scale = 8, 128, 0.1
    for f, v in kw.items():
        setattr(a, f, v)
    return a


BIG = 1 << 62


@pytest.mark.parametrize("kw,want", [
    (dict(head_size=100), "INVALID"), (dict(block_size=24), "INVALID"), (dict(num_heads=9), "INVALID"),
    (dict(max_drafts=65), "INVALID"), (dict(max_drafts=-1), "INVALID"), (dict(num_seqs=-1), "INVALID"),
    (dict(num_seqs=65536), "INVALID"), (dict(num_rows=-1), "INVALID"), (dict(num_blocks=-1), "INVALID"),
    (dict(max_context_len=129), "INVALID"), (dict(max_context_len=-1), "INVALID"), (dict(k_cache=0), "INVALID"),
    (dict(draft_masks=0), "INVALID"), (dict(draft_masks=P + 4), "INVALID"), (dict(q=P + 8), "INVALID"),
    (dict(v_cache=P + 4), "INVALID"), (dict(context_lens=P + 1), "INVALID"),
    (dict(num_seqs=0), "OK"), (dict(num_rows=0), "OK"), (dict(max_drafts=0), "OK"),
])
def test_tree_attention_refusals(kw, want):
    assert status(N.lib().tlh_tree_attention, C.byref(tree(**kw)), P, BIG, None)[0] == want


def test_tree_attention_scratch_refusals():
    n = C.c_size_t()
    a = tree(max_context_len=8192, max_blocks_per_seq=512)
    assert status(N.lib().tlh_tree_attention_scratch_bytes, C.byref(a), C.byref(n))[0] == "OK"
    assert status(N.lib().tlh_tree_attention_scratch_bytes, C.byref(a), None)[0] == "INVALID"
    assert status(N.lib().tlh_tree_attention_scratch_bytes, None, C.byref(n))[0] == "INVALID"
    if n.value:
        assert status(N.lib().tlh_tree_attention, C.byref(a), P, n.value - 1, None)[0] == "INVALID"
        assert status(N.lib().tlh_tree_attention, C.byref(a), None, n.value, None)[0] == "INVALID"
        assert status(N.lib().tlh_tree_attention, C.byref(a), P + 8, n.value, None)[0] == "INVALID"


def test_tree_attention_scratch_grows_with_the_batch():
    """One buffer for the largest batch, rows, drafts and context serves every smaller call."""
    def size(**kw):
        n = C.c_size_t()
        assert status(N.lib().tlh_tree_attention_scratch_bytes, C.byref(tree(**kw)), C.byref(n))[0] == "OK"
        return n.value
    for seqs in (1, 3, 32, 200):
        for ctx in (1, 100, 4096, 30000):
            s = [size(num_seqs=seqs, num_rows=r, max_drafts=8, max_context_len=ctx, max_blocks_per_seq=2000)
                 for r in (1, 8, 9, 64, 300, 2000)]
            assert s == sorted(s), (seqs, ctx, s)
    s = [size(num_seqs=n, num_rows=8 * n, max_context_len=5000, max_blocks_per_seq=2000) for n in range(1, 80)]
    assert s == sorted(s)
    s = [size(num_rows=64, max_drafts=64, max_context_len=c, max_blocks_per_seq=2000) for c in range(0, 20000, 173)]
    assert s == sorted(s)
    s = [size(num_rows=64, max_drafts=d, max_context_len=9000, max_blocks_per_seq=2000) for d in range(1, 65)]
    assert s == sorted(s)


def copy(pools=(P, P), block_bytes=4096, num_blocks=10, pairs=P, num_pairs=1):
    arr = (C.c_void_p * len(pools))(*pools) if pools else None
    return status(N.lib().tlh_copy_blocks, arr, len(pools) if pools is not None else 0, block_bytes, num_blocks, pairs,
                  num_pairs, None)[0]


def test_copy_blocks_refusals():
    assert copy(block_bytes=0) == copy(block_bytes=24) == copy(block_bytes=-16) == copy(block_bytes=1 << 30) == "INVALID"
    assert copy(num_blocks=-1) == copy(num_pairs=-1) == copy(pairs=None) == copy(pairs=P + 4) == "INVALID"
    assert copy(num_blocks=1 << 62) == copy(pools=(P, None)) == copy(pools=(P, P + 8)) == "INVALID"
    assert copy(num_pairs=0) == copy(pools=()) == "OK"


def compact(**kw):
    a = N.TlhCompactArgs()
    pools = kw.pop("pools", (P, P))
    arr = (C.c_void_p * 2)(*pools)
    a.k_caches = a.v_caches = arr
    for i, f in enumerate(("block_tables", "context_lens", "draft_starts", "keep", "new_lens")):
        setattr(a, f, P + 4096 * i)
    a.num_blocks, a.num_layers, a.num_seqs, a.max_drafts = 10, 2, 1, 8
    a.num_kv_heads, a.head_size, a.block_size, a.max_blocks_per_seq = 2, 128, 16, 4
    for f, v in kw.items():
        setattr(a, f, v)
    return status(N.lib().tlh_compact_cache, C.byref(a), None)[0]


@pytest.mark.parametrize("kw,want", [
    (dict(head_size=72), "INVALID"), (dict(block_size=64), "INVALID"), (dict(num_kv_heads=0), "INVALID"),
    (dict(max_drafts=65), "INVALID"), (dict(num_seqs=-1), "INVALID"), (dict(num_layers=-1), "INVALID"),
    (dict(num_blocks=-1), "INVALID"), (dict(max_blocks_per_seq=1 << 30), "INVALID"), (dict(keep=0), "INVALID"),
    (dict(new_lens=P + 4096), "INVALID"), (dict(new_lens=0), "INVALID"), (dict(keep=P + 4), "INVALID"),
    (dict(pools=(P, None)), "INVALID"), (dict(pools=(P, P + 4)), "INVALID"),
    (dict(num_seqs=0), "OK"), (dict(num_layers=0), "OK"),
])
def test_compact_cache_refusals(kw, want):
    assert compact(**kw) == want


def logprobs(scratch=P, nbytes=BIG, **kw):
    a = N.TlhLogprobsArgs()
    for f in ("logits", "tokens", "logprobs", "entropy", "top_logprobs", "top_ids"):
        setattr(a, f, P)
    a.type, a.rows, a.vocab, a.top, a.row_stride = N.F32, 3, 1000, 5, 1000
    for f, v in kw.items():
        setattr(a, f, v)
    return status(N.lib().tlh_token_logprobs, C.byref(a), scratch, nbytes, None)[0]


@pytest.mark.parametrize("kw,want", [
    (dict(type=N.Q8_0), "UNSUPPORTED"), (dict(rows=-1), "INVALID"), (dict(vocab=0), "INVALID"),
    (dict(vocab=1000001, row_stride=1000001), "INVALID"), (dict(top=33), "INVALID"), (dict(top=-1), "INVALID"),
    (dict(vocab=4, top=5), "INVALID"), (dict(row_stride=999), "INVALID"), (dict(logits=0), "INVALID"),
    (dict(logits=P + 2), "INVALID"), (dict(tokens=0), "INVALID"), (dict(logprobs=0), "INVALID"),
    (dict(top_ids=0), "INVALID"), (dict(top_logprobs=P + 2), "INVALID"), (dict(scratch=0), "INVALID"),
    (dict(scratch=P + 8), "INVALID"), (dict(nbytes=16), "INVALID"), (dict(rows=0), "OK"),
])
def test_token_logprobs_refusals(kw, want):
    assert logprobs(**kw) == want


def test_token_logprobs_scratch_grows_with_the_rows():
    def size(rows, vocab):
        a, n = N.TlhLogprobsArgs(), C.c_size_t()
        a.type, a.rows, a.vocab, a.top, a.row_stride = N.BF16, rows, vocab, 20, vocab
        assert status(N.lib().tlh_token_logprobs_scratch_bytes, C.byref(a), C.byref(n))[0] == "OK"
        return n.value
    for vocab in (20, 5000, 128256, 1000000):
        s = [size(r, vocab) for r in range(0, 600, 7)]
        assert s == sorted(s), vocab


# ------------------------------------------------- the Python entry points
def rows(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def test_python_checks_name_the_tensor():
    q, k = rows(4, 8, 64), rows(4, 2, 64)
    starts = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        N.packed_attention(q, k, k, starts, 4, 0.1)
    with pytest.raises(ValueError, match="f16 or all bf16"):
        N.packed_attention(q.float(), k, k, starts, 4, 0.1)
    with pytest.raises(ValueError, match="do not match"):
        N.packed_attention(q, k[:3], k[:3], starts, 4, 0.1)
    with pytest.raises(ValueError, match="heads must be contiguous"):
        N.packed_attention(rows(8, 4, 64).transpose(0, 1), k, k, starts, 4, 0.1)
    with pytest.raises(ValueError, match="seq_starts"):
        N.packed_attention(q, k, k, starts.long(), 4, 0.1)
    node = N.TreeAttention(1, 3, 3, 8, 2, 64, 16, 4, 64, 0.1, device="cpu")
    kc, vc = rows(5, 2, 8, 16, 8), rows(5, 2, 64, 16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    good = dict(out=rows(3, 8, 64), q=rows(3, 8, 64), k_cache=kc, v_cache=vc, block_tables=i32(1, 4),
                context_lens=i32(1), draft_starts=i32(2), draft_masks=torch.zeros(3, dtype=torch.int64))
    for name, bad in (("q", rows(2, 8, 64)), ("out", rows(3, 8, 128)), ("k_cache", kc.float()), ("v_cache", vc[:4]),
                      ("block_tables", i32(1, 3)), ("context_lens", i32(2)), ("draft_starts", i32(1)),
                      ("draft_masks", i32(3))):
        with pytest.raises(ValueError, match=name):
            node(**{**good, name: bad})
    with pytest.raises(ValueError, match="on the GPU"):
        node(**good)
    with pytest.raises(N.TlhError, match="max_drafts"):
        N.TreeAttention(1, 70, 70, 8, 2, 64, 16, 4, 64, 0.1, device="cpu")
    with pytest.raises(ValueError, match="v_cache"):
        N.KVPools([kc], [vc[:2]], 2, 64, 16)
    p = N.KVPools([kc], [vc], 2, 64, 16)
    with pytest.raises(ValueError, match="pairs"):
        p.copy_blocks(i32(2, 2))
    with pytest.raises(ValueError, match="keep"):
        p.compact(i32(1, 4), i32(1), i32(2), i32(1), i32(1), 3)
    lp = N.TokenLogprobs(2, 100, 3, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="logits"):
        lp(rows(3, 100, dtype=torch.float32), i32(3), None, None)
    with pytest.raises(ValueError, match="top_ids"):
        lp(rows(2, 100, dtype=torch.float32), i32(2), rows(2, dtype=torch.float32), None)
    with pytest.raises(N.TlhError, match="top"):
        N.TokenLogprobs(2, 10, 11, torch.float32, device="cpu")


def test_sizes_past_one_launch_are_refused():
    """Grids of more threads than a launch takes, told before it."""
    assert status(N.lib().tlh_packed_attention, C.byref(packed(num_tokens=2 ** 31 - 1, max_seq_len=2 ** 31 - 1)), None)[0] == "INVALID"
    assert status(N.lib().tlh_tree_attention, C.byref(tree(num_seqs=65535, num_heads=2048, num_kv_heads=1024)), P, BIG, None)[0] == "INVALID"
    assert compact(num_seqs=1 << 24) == "INVALID"
    assert logprobs(rows=(1 << 24) + 1) == "INVALID"


def test_compact_cache_lengths_must_not_overlap():
    base = 0x100000
    for at in (0, 4, 12, -4, -12):
        assert compact(num_seqs=4, context_lens=base, new_lens=base + at, draft_starts=base + 4096) == "INVALID", at
        assert compact(num_seqs=4, draft_starts=base, new_lens=base + at, context_lens=base + 4096) == "INVALID", at
    assert compact(num_seqs=4, draft_starts=base, new_lens=base + 16, context_lens=base + 4096) == "INVALID"


def test_tree_attention_refuses_contexts_past_its_integers():
    """A tile's lookahead past the last token is formed in 32 bits."""
    n = C.c_size_t()
    for ctx, want in ((1 << 30, "OK"), ((1 << 30) + 1, "INVALID"), ((1 << 31) - 1, "INVALID")):
        a = tree(max_context_len=ctx, max_blocks_per_seq=1 << 27)
        assert status(N.lib().tlh_tree_attention_scratch_bytes, C.byref(a), C.byref(n))[0] == want
    assert status(N.lib().tlh_tree_attention, C.byref(a), P, BIG, None)[0] == "INVALID"


def test_a_tree_node_takes_smaller_calls_and_refuses_larger_ones():
    kc, vc = rows(5, 2, 8, 16, 8), rows(5, 2, 64, 16)
    node = N.TreeAttention(3, 10, 8, 8, 2, 64, 16, 4, 64, 0.1, device="cpu")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731

    def call(n, seqs, **kw):
        a = dict(out=rows(n, 8, 64), q=rows(n, 8, 64), k_cache=kc, v_cache=vc, block_tables=i32(seqs, 4),
                 context_lens=i32(seqs), draft_starts=i32(seqs + 1), draft_masks=torch.zeros(n, dtype=torch.int64))
        node(**{**a, **kw})

    for n, seqs in ((10, 3), (7, 3), (10, 1), (1, 1), (0, 3), (0, 0)):
        with pytest.raises(ValueError, match="on the GPU"):  # everything before that fits
            call(n, seqs)
    for n, seqs in ((11, 3), (10, 4)):
        with pytest.raises(ValueError, match="up to"):
            call(n, seqs)
    for name, bad in (("q", rows(6, 8, 64)), ("draft_masks", torch.zeros(8, dtype=torch.int64)), ("context_lens", i32(3)),
                      ("draft_starts", i32(2)), ("block_tables", i32(2, 3))):
        with pytest.raises(ValueError, match=name):
            call(7, 2, **{name: bad})


@pytest.mark.parametrize("more", [1 << 31, (1 << 32) + 4, -(1 << 32) + 4])
def test_counts_past_32_bits_are_refused(more):
    """Cut to 32 bits most of these would be a count that fits."""
    q, k, starts = rows(4, 8, 64), rows(4, 2, 64), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="max_seq_len .* 32 bits"):
        N.packed_attention(q, k, k, starts, more, 0.1)
    names = ("num_seqs", "num_rows", "max_drafts", "num_heads", "num_kv_heads", "head_size", "block_size",
             "max_blocks_per_seq", "max_context_len")
    good = dict(zip(names, (1, 3, 3, 8, 2, 64, 16, 4, 64)))
    N.TreeAttention(**good, scale=0.1, device="cpu")
    for name in names:
        with pytest.raises(ValueError, match=f"{name} .* 32 bits"):
            N.TreeAttention(**{**good, name: more}, scale=0.1, device="cpu")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pools = N.KVPools([rows(5, 2, 8, 16, 8)], [rows(5, 2, 64, 16)], 2, 64, 16)
    with pytest.raises(ValueError, match="max_drafts .* 32 bits"):
        pools.compact(i32(1, 4), i32(1), i32(2), torch.zeros(1, dtype=torch.int64), i32(1), more)
    for at, name in enumerate(("rows", "vocab", "top")):
        args = [2, 100, 3]
        args[at] = more
        with pytest.raises(ValueError, match=f"{name} .* 32 bits"):
            N.TokenLogprobs(*args, torch.float32, device="cpu")


def test_packed_attention_out_must_be_apart():
    """Rows of out that share a byte with rows of q, k or v are told apart from those that lie between them. (Calls
    that pass are refused behind that, for more workgroups than a launch takes.)"""
    H, KV, n, base = 32768, 8192, 1 << 16, 1 << 44
    qrow, krow = 64 * H, 64 * KV  # elements

    def refused(o, q, k, v, so, sq, sk, sv):
        st, text = status(N.lib().tlh_packed_attention, C.byref(packed(
            out=base + 2 * o, q=base + 2 * q, k=base + 2 * k, v=base + 2 * v, out_stride=so, q_stride=sq, k_stride=sk,
            v_stride=sv, num_heads=H, num_kv_heads=KV, num_tokens=n, max_seq_len=n)), None)
        assert st == "INVALID" and ("overlaps" in text or "too large for one launch" in text), text
        return "overlaps" in text

    wide, far = 2 * qrow + 2 * krow, 1 << 40
    # columns of one buffer's rows: q, k, v, out in turn
    at = dict(q=0, k=qrow, v=qrow + krow, o=qrow + 2 * krow)
    steps = dict(so=wide, sq=wide, sk=wide, sv=wide)
    assert not refused(**at, **steps)
    for name in "qkv":  # any of them, from either side, and whole
        for by in (8, -8):
            assert refused(**{**at, "o": at[name] + by}, **steps)
        assert refused(**{**at, "o": at[name]}, **steps)
    assert refused(**{**at, "o": at["o"] + 8}, **steps)  # into the next row's q
    # tensors of their own, one behind the other
    own = dict(so=qrow, sq=qrow, sk=krow, sv=krow)
    ends = dict(q=0, o=n * qrow, k=2 * n * qrow, v=2 * n * qrow + n * krow)
    assert not refused(**ends, **own)
    for o in (n * qrow - 8, n * qrow + 8):
        assert refused(**{**ends, "o": o}, **own)
    # rows at another step than q's, against the bytes
    r = random.Random(5)
    seen = set()
    for _ in range(40):
        so, sq = qrow * r.choice([2, 3, 4]) + 8 * r.randrange(4), qrow * r.choice([2, 3, 4, 6]) + 8 * r.randrange(4)
        o, q = r.randrange(0, 4 * qrow, 8), r.randrange(0, 4 * qrow, 8)
        if r.random() < 0.5:  # between q's rows, as long as the steps are whole multiples
            so, sq, o, q = 4 * qrow, 2 * qrow, qrow * r.choice([1, 3]), 0
        want = False
        j = 0
        for i in range(n):
            while j < n and q + j * sq + qrow <= o + i * so:
                j += 1
            if j < n and q + j * sq < o + i * so + qrow:
                want = True
                break
        assert refused(o, q, far, far + n * krow, so, sq, krow, krow) == want
        seen.add(want)
    assert seen == {True, False}


def test_packed_attention_past_one_launch_is_told_as_such():
    a = packed(num_tokens=2 ** 31 - 1, max_seq_len=2 ** 31 - 1, out=1 << 50)
    assert status(N.lib().tlh_packed_attention, C.byref(a), None) == (
        "INVALID", "packed_attention: max_seq_len x num_heads too large for one launch")


def test_tree_attention_out_must_be_apart():
    """(Calls that pass are refused behind that, for want of scratch.)"""
    rows, pool, base = 10 * 8 * 128 * 2, 100 * 2 * 128 * 16 * 2, 1 << 40
    at = dict(q=base, k_cache=base + rows, v_cache=base + rows + pool)

    def refused(out, **kw):
        a = tree(**{**at, **kw}, out=out, max_context_len=8192, max_blocks_per_seq=512)
        st, text = status(N.lib().tlh_tree_attention, C.byref(a), None, 0, None)
        assert st == "INVALID" and ("overlaps" in text or "scratch" in text), text
        return "overlaps" in text

    assert not refused(base - rows) and not refused(base + rows + 2 * pool)
    for out in (base - rows + 16, base, base + rows - 16, base + rows, base + rows + pool - 16, base + rows + 2 * pool - 16):
        assert refused(out), out
    assert not refused(base + rows + 2 * pool, num_blocks=0) and not refused(base + rows + 16, num_blocks=0)
    assert refused(base + (1 << 50), num_blocks=1 << 62)


def test_compact_cache_lengths_must_be_apart_from_all_that_is_read():
    """(Calls that pass are refused behind that, for a layer without pools.)"""
    base = 0x100000

    def refused(new_lens, **kw):
        got = compact(num_seqs=4, new_lens=new_lens, pools=(P, None), **kw)
        assert got == "INVALID"
        return "overlap" in N.lib().tlh_last_error().decode()

    for name, size in (("keep", 32), ("block_tables", 64), ("context_lens", 16), ("draft_starts", 20)):
        for at in (-12, 0, 4, size - 4):
            assert refused(base + at, **{name: base}), (name, at)
        for at in (-16, size):
            assert not refused(base + at, **{name: base}), (name, at)


def test_a_split_contexts_scratch_is_asked_for_and_checked():
    n = C.c_size_t()
    a = tree(max_context_len=8192, max_blocks_per_seq=512)
    assert status(N.lib().tlh_tree_attention_scratch_bytes, C.byref(a), C.byref(n))[0] == "OK"
    assert n.value > 0
    a.out = 1 << 40
    for scratch, nbytes in ((P, n.value - 1), (None, n.value), (P + 8, n.value)):
        st, text = status(N.lib().tlh_tree_attention, C.byref(a), scratch, nbytes, None)
        assert st == "INVALID" and "scratch" in text
