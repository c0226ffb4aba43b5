"""Plain 64-bit forms of a serving step's operators (attention of new tokens over pages, heads' norms and rotation with
the cache write, verification of drafts), and how far a 32-bit one may be from them.

Attention's bound is serving_refs.bound. A rotated head y of f32 heads x, rounded to a 16-bit type:
 * the rounding, eps / 2 of y (below the type's normal range half its smallest number);
 * the norm: the sum of D squares is off by at most D 2^-24 of itself, the root by half of that; the division, the root
   and the products by 2^-24 each: (D / 2 + 6) 2^-24 of each of the pair's two products;
 * the angle: its fraction of a turn, at most 1/2, is rounded to f32 (2^-26 of a turn, 2 pi 2^-26 < 2^-23 of a radian),
   cos and sin are off by at most 2^-21, the two products and their sum by 3 2^-24: together below 2^-20 of |y_a| + |y_b|.
A probability in f32 is off by its rounding, 2^-24 of it.
"""
from __future__ import annotations

import numpy as np
import torch

from serving_refs import attend, bound


def new_token_starts(counts):
    return [0] + [int(n) for n in np.cumsum(counts)]


def chunk_reference(q, kc, vc, table, lens, starts, scale, window=0, max_rows=None, max_context=None):
    """-> (out, tolerance) float64 (rows, heads, D); rows of no sequence, or past max_rows, are NaN."""
    rows, H, D = q.shape
    NB, KV, _, bs, _ = kc.shape
    out = torch.full((rows, H, D), float("nan"), dtype=torch.float64)
    tol = torch.zeros((rows, H, D), dtype=torch.float64)
    q, kc, vc = (t.detach().cpu() for t in (q, kc, vc))
    for s, L in enumerate(lens):
        a, n = starts[s], starts[s + 1] - starts[s]
        n = n if max_rows is None else min(n, max_rows)
        L = max(0, L if max_context is None else min(L, max_context))
        if n <= 0:
            continue
        pos = np.arange(L)
        page = np.asarray(table)[s, pos // bs] if L else np.zeros(0, int)
        ok = (page >= 0) & (page < NB)
        pg, off = torch.from_numpy(np.where(ok, page, 0).astype(np.int64)), torch.from_numpy(pos % bs)
        at = torch.arange(L - n, L)[:, None]
        j = torch.arange(L)
        see = (j <= at) & torch.from_numpy(ok)
        if window:
            see = see & (j > at - window)
        seen = see.any(0)[:, None]
        for g in range(KV):
            if L:
                k, v = kc[pg, g, :, off].reshape(L, D).double(), vc[pg, g, :, off].reshape(L, D).double()
                k, v = torch.where(seen, k, torch.zeros_like(k)), torch.where(seen, v, torch.zeros_like(v))
                vmax = float(v[torch.isfinite(v)].abs().max())
            else:
                k, v, vmax = torch.zeros((0, D)).double(), torch.zeros((0, D)).double(), 0.0
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                o, A, d = attend(q[a:a + n, h].double(), k, v, see, scale)
                out[a:a + n, h] = o
                tol[a:a + n, h] = bound(o, A, d, L, vmax, torch.float16)
    return out, tol


def rope_reference(x, norm, eps, positions, pair_axes, freqs, mode, attn_factor, dtype):
    """One of q and k: x (tokens, heads, D), positions (axes, tokens) -> (y, tolerance) float64."""
    D, P = x.shape[-1], len(pair_axes)
    x = x.detach().cpu().double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.detach().cpu().double()
    pos = positions.detach().cpu().double()
    angle = torch.stack([pos[a] * float(f) for a, f in zip(pair_axes, freqs.detach().cpu().double())], -1)[:, None] if P else None
    y, size = x.clone(), x.abs()
    if P:
        a = list(range(0, 2 * P, 2)) if mode == 0 else list(range(P))
        b = list(range(1, 2 * P, 2)) if mode == 0 else list(range(P, 2 * P))
        c, s = torch.cos(angle) * attn_factor, torch.sin(angle) * attn_factor
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        both = (x[..., a].abs() + x[..., b].abs()) * abs(attn_factor)
        size[..., a], size[..., b] = both, both
    return y, rounded(y, dtype) + size * ((D / 2 + 6) * 2.0 ** -24 + 2.0 ** -20)


def rounded(y, dtype):
    """How far a rounding to dtype may move y."""
    info = torch.finfo(dtype)
    return y.abs() * info.eps / 2 * (1 + 2.0 ** -10) + info.tiny * info.eps / 2


def into_caches(kc, vc, k, v, slots):
    """The caches (copies) with each token's heads k, v (tokens, kv heads, D) at its slot."""
    NB, KV, C, bs, _ = kc.shape
    kc, vc = kc.clone(), vc.clone()
    for t, s in enumerate(slots):
        if 0 <= s < NB * bs:
            kc[s // bs, :, :, s % bs] = k[t].reshape(KV, C, 8)
            vc[s // bs, :, :, s % bs] = v[t]
    return kc, vc


def distribution(logits, temperature):
    """(V,) float64, or None where there is none."""
    x = np.asarray(logits, np.float64)
    if np.isnan(x).any() or (x == -np.inf).all() or (temperature > 0 and (x == np.inf).any()):
        return None
    if not temperature > 0:
        p = np.zeros(len(x))
        p[int(np.argmax(x))] = 1.0
        return p
    e = np.exp((x - x.max()) / temperature)
    return e / e.sum()


def verify_reference(target, draft, tokens, starts, temps, accept_at, sample_at, max_drafts):
    """-> (accepted, out_tokens, accept_probs); probabilities of drafts that nobody looks at are 7."""
    target, V = target.detach().cpu().double().numpy(), target.shape[1]
    draft = None if draft is None else draft.detach().cpu().double().numpy()
    probs, accepted, out = np.full(len(tokens), 7.0), [], []
    for s, t in enumerate(np.asarray(temps, np.float64)):
        b, n = starts[s], min(starts[s + 1] - starts[s], max_drafts)
        greedy, stop, undefined = not t > 0, None, False
        for i in range(n):
            x = int(tokens[b + i])
            p = distribution(target[b + s + i], t)
            if greedy or draft is None:  # greedy: the drafter does not matter
                q = np.zeros(V)
                if 0 <= x < V:
                    q[x] = 1.0
            else:
                q = distribution(draft[b + i], t)
            if p is None or q is None:
                probs[b + i] = np.nan
                ok = False
            else:
                px, qx = (p[x], q[x]) if 0 <= x < V else (0.0, 0.0)
                probs[b + i] = min(1.0, px / qx) if qx > 0 else float(px > 0)
                ok = px == 1.0 if greedy else float(accept_at[b + i]) * qx < px
            if not ok and stop is None:
                stop, undefined, where = i, p is None or q is None, (p, q)
        if stop is None:
            stop, where = n, (distribution(target[b + s + n], t), None)
            undefined = where[0] is None
        token = -1
        if not undefined:
            rest = where[0] if where[1] is None else np.maximum(where[0] - where[1], 0.0)
            rest = where[0] if rest.sum() == 0 else rest
            run = np.cumsum(rest)
            over = np.nonzero(run > float(sample_at[s]) * run[-1])[0]
            token = int(over[0]) if len(over) else int(np.nonzero(rest)[0][-1])
        accepted.append(stop)
        out.append([int(x) for x in tokens[b:b + stop]] + [token] + [-1] * (max_drafts - stop))
    return np.array(accepted), np.array(out).reshape(len(accepted), max_drafts + 1), probs
