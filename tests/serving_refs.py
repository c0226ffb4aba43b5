"""Plain 64-bit forms of the serving operators, and how far a 32-bit one may be from them.

Attention's bound for a result o = sum p v / sum p of one row, with A = sum p |v| / sum p:
 * the result's own rounding, eps / 2 of it;
 * the numerators' rounding to the type before the product with v, eps / 2 of A (below the type's
   normal range, f16's 2^-14, they are off by at most 2^-25 each, and the largest is at least 1:
   2^-25 times the number of keys times the largest |v|);
 * scores in f32: a dot product of D terms is off by at most D 2^-24 sum |q k|, times the scale; the
   exponent's argument by 2^-22 of the largest score, the exponential and the sums by 2^-20. exp
   turns an error d of a score into a relative error d of p, in the numerator and in the sum: 2 d A.
"""
from __future__ import annotations

import numpy as np
import torch


def attend(q, k, v, see, scale):
    """q (n, D), k and v (L, D) float64, see (n, L) -> (out, bound's A, rows' score error d)."""
    n, D = q.shape
    if k.shape[0] == 0:
        z = torch.zeros((n, v.shape[1]), dtype=torch.float64)
        return z, z, 0.0
    s = (q @ k.T) * scale
    s = torch.where(see, s, torch.full_like(s, -np.inf))
    m = s.amax(1, keepdim=True)
    p = torch.where(see, torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m)), torch.zeros_like(s))
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    # a key that a row does not see adds nothing, whatever it holds
    finite = torch.isfinite(v).all(1)
    o = p @ torch.where(finite[:, None], v, torch.zeros_like(v))
    for j in torch.nonzero(~finite)[:, 0].tolist():
        o = torch.where(see[:, j, None], o + p[:, j, None] * v[j], o)
    A = p @ torch.where(finite[:, None], v.abs(), torch.zeros_like(v))
    worst = lambda t: torch.where(see, t.abs(), torch.zeros_like(t)).amax(1, keepdim=True)  # noqa: E731
    d = D * 2.0 ** -24 * worst((q.abs() @ k.abs().T) * scale) + 2.0 ** -22 * worst(s) + 2.0 ** -20
    return o, A, d


def bound(out, A, d, keys, vmax, dtype):
    eps = torch.finfo(dtype).eps
    sub = 2.0 ** -25 * keys * vmax if dtype == torch.float16 else 0.0
    return (out.abs() + A) * eps / 2 * 1.01 + 2 * d * A + sub + torch.finfo(dtype).tiny * eps


def packed_reference(q, k, v, starts, scale, dtype):
    """-> (out, tolerance) float64 (tokens, heads, D) of the tokens that belong to a sequence."""
    T, H, D = q.shape
    G = H // k.shape[1]
    out, tol = torch.zeros((T, H, D), dtype=torch.float64), torch.zeros((T, H, D), dtype=torch.float64)
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    for a, b in zip(starts[:-1], starts[1:]):
        if b <= a:
            continue
        see = torch.ones((b - a, b - a)).tril().bool()
        for h in range(H):
            o, A, d = attend(q[a:b, h], k[a:b, h // G], v[a:b, h // G], see, scale)
            out[a:b, h] = o
            tol[a:b, h] = bound(o, A, d, b - a, float(v[a:b, h // G].abs().max()), dtype)
    return out, tol


def tree_reference(q, kc, vc, tables, lens, starts, masks, scale):
    """The paged form; pages outside the pools are not seen."""
    rows, H, D = q.shape
    NB, KV, _, bs, _ = kc.shape
    out, tol = torch.zeros((rows, H, D), dtype=torch.float64), torch.zeros((rows, H, D), dtype=torch.float64)
    q, kc, vc = (t.detach().cpu().double() for t in (q, kc, vc))
    for s, L in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n <= 0:
            continue
        pos = np.arange(L)
        page = np.asarray(tables)[s, pos // bs] if L else np.zeros(0, int)
        ok = (page >= 0) & (page < NB)
        pg = torch.from_numpy(np.where(ok, page, 0).astype(np.int64))
        off = torch.from_numpy(pos % bs)
        see = torch.from_numpy(np.tile(ok, (n, 1)))
        for i in range(n):
            for j in range(n):
                if L - n + j >= 0 and not (int(masks[a + i]) >> j) & 1:
                    see[i, L - n + j] = False
        for h in range(H):
            g = h // (H // KV)
            k, v = kc[pg, g, :, off].reshape(L, D), vc[pg, g, :, off].reshape(L, D)
            seen = see.any(0)[:, None]
            k, v = torch.where(seen, k, torch.zeros_like(k)), torch.where(seen, v, torch.zeros_like(v))
            o, A, d = attend(q[a:b, h], k, v, see, scale)
            out[a:b, h] = o
            tol[a:b, h] = bound(o, A, d, L, float(v[torch.isfinite(v)].abs().max()) if L else 0.0, torch.float16)
    return out, tol


def chain_masks(n):
    return [(1 << (i + 1)) - 1 for i in range(n)]


def random_tree(r, n):
    masks = []
    for i in range(n):
        p = int(r.integers(-1, i)) if i else -1
        masks.append((masks[p] if p >= 0 else 0) | (1 << i))
    return masks


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


def pools(g, blocks, kv, hs, bs):
    k = torch.randn((blocks, kv, hs // 8, bs, 8), generator=g).half()
    v = torch.randn((blocks, kv, hs, bs), generator=g).half()
    return k, v


def tables(r, lens, bs, spare=2, width=None):
    need = [max(1, -(-n // bs)) for n in lens]
    blocks = sum(need) + spare
    ids = r.permutation(blocks)
    t = np.zeros((len(lens), width or max(need)), np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = ids[at:at + n]
        at += n
    return t, blocks


def one_large_and_many_tiny(n, D, seed):
    """k and v (n, D) f16 and the weights' logarithm: with q = (1, 0, ..) and scale 1 every key but the first weighs 2^-25.09
    of it, which f16 rounds to 0, and carries the values: half of the dims 1 throughout, half normal."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.zeros((n, D), dtype=torch.float16), torch.randn((n, D), generator=g).half()
    k[0, 0] = 17.390625  # 25.0894 ln 2
    v[:, :D // 2] = 1.0
    v[0] = 0.0
    return k, v


def tiny_bound(out, A, d, keys, vmax):
    """f16, with numerators of at least 2^7 for the largest: those below 2^-14 are off by at most 2^-25, 2^-32 of it."""
    eps = torch.finfo(torch.float16).eps
    return (out.abs() + A) * eps / 2 * 1.01 + 2 * d * A + 2.0 ** -32 * keys * vmax + 2.0 ** -24
