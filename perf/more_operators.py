"""More operators of a serving step over a paged KV cache, and the calls they are measured on.

A server whose batch mixes pieces of prompts, single tokens and drafted tokens runs, between the
projections of a layer and behind the last one: the norms of the query and key heads, their rotation
by positions of one or several axes and the write of keys and values to the cache in one pass
(``native.HeadRope``), attention of each sequence's new tokens, one or thousands, over its pages
(``native.ChunkAttention``), and the verification of drafted tokens against the model's probabilities
(``native.DraftVerify``).

``listed`` names fixed cases, ``draw`` gives others of the same ranges, ``prepare`` builds what a
program has in hand, ``run`` is one pass (with ``own`` through the framework, else in plain torch),
``work`` the bytes and operations it cannot do without, ``exact`` the result in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one chat's next token over its pages, where latency counts
        dict(name="chunk 1 token over 1500", path="chunk", heads=32, kv_heads=8, head_size=128, block=16, decodes=1,
             chunks=0, shortest=1, longest=1, near=1500, far=1500, window=0),
        # a batch in flight: 31 sequences take a token each, one brings 600 tokens of its prompt
        dict(name="chunk 31 tokens + 600", path="chunk", heads=32, kv_heads=8, head_size=128, block=16, decodes=31,
             chunks=1, shortest=600, longest=600, near=512, far=8192, window=0),
        # a long document's next piece (the largest)
        dict(name="chunk 2048 over 16384", path="chunk", heads=32, kv_heads=8, head_size=128, block=16, decodes=0,
             chunks=1, shortest=2048, longest=2048, near=16384, far=16384, window=0),
        # prompts of odd lengths behind cached prefixes, a layer that looks back 1024 tokens, few wide heads
        dict(name="chunk 9x13..701 window", path="chunk", heads=4, kv_heads=1, head_size=256, block=32, decodes=0,
             chunks=9, shortest=13, longest=701, near=0, far=5000, window=1024),
        # one token's heads
        dict(name="heads 1 token", path="heads", dtype="f32", tokens=1, heads=32, kv_heads=8, head_size=128, block=16,
             norm=True, axes=1, interleaved=False, neox=True, rotated=128, furthest=4000),
        # the heads of an image's patches and its text: time, height, width
        dict(name="heads 2501 3 axes", path="heads", dtype="bf16", tokens=2501, heads=28, kv_heads=4, head_size=128,
             block=16, norm=False, axes=3, interleaved=False, neox=True, rotated=128, furthest=60000),
        # a large piece of a prompt, far into a long context
        dict(name="heads 8192 tokens", path="heads", dtype="f32", tokens=8192, heads=32, kv_heads=8, head_size=128,
             block=16, norm=True, axes=1, interleaved=False, neox=True, rotated=128, furthest=120000),
        # one chat, four tokens drafted by a smaller model
        dict(name="verify 1 x 4", path="verify", dtype="f32", seqs=1, drafts=4, ragged=False, vocab=128256,
             drafter=True, greedy=0.0, masked=0.0),
        # a batch, one to eight drafted tokens each, some of it greedy
        dict(name="verify 32 x 1..8", path="verify", dtype="f32", seqs=32, drafts=8, ragged=True, vocab=128256,
             drafter=True, greedy=0.25, masked=0.0),
        # tokens copied from the prompt (no drafting model), under a grammar's mask
        dict(name="verify 48 x 10 copied", path="verify", dtype="bf16", seqs=48, drafts=10, ragged=False, vocab=32003,
             drafter=False, greedy=0.0, masked=0.5),
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(32, 8), (32, 8), (32, 32), (16, 8), (28, 4), (8, 1), (12, 2), (64, 8), (8, 2), (4, 1)])


def draw(rng):
    path = rng.choices(["chunk", "heads", "verify"], [5, 4, 4])[0]
    head_size = rng.choice([64, 128, 128, 128, 80, 96, 112, 192, 256])
    block = rng.choice([8, 16, 16, 32])
    if path == "chunk":
        heads, kv_heads = _heads(rng)
        decodes, chunks = rng.choice([(1, 0), (0, 1), (1, 1)])
        decodes *= _log(rng, 1, 64)
        chunks *= _log(rng, 1, 16)
        longest, far = _log(rng, 2, 2048), _log(rng, 1, 16384)

        def cost():
            rows = decodes + chunks * longest
            return max(rows * (far + longest) * heads * head_size / (2048 * 17408 * 32 * 128),
                       (decodes + chunks) * (far + longest) * kv_heads * head_size / (32 * 8192 * 8 * 128))

        while cost() > 1:
            decodes, chunks = decodes * 3 // 4, chunks * 3 // 4 if chunks > 1 else chunks
            longest, far = max(2, longest * 7 // 8), max(1, far * 7 // 8)
            decodes = decodes if decodes + chunks else 1
        return dict(path=path, heads=heads, kv_heads=kv_heads, head_size=head_size, block=block, decodes=decodes,
                    chunks=chunks, shortest=max(1, int(longest * rng.uniform(0.02, 1.0))), longest=longest,
                    near=int(far * rng.uniform(0.0, 1.0)), far=far, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    if path == "heads":
        heads, kv_heads = _heads(rng)
        tokens = _log(rng, 1, 8192)
        while tokens * (heads + 2 * kv_heads) * head_size > 8192 * 48 * 128:
            tokens = tokens * 3 // 4
        return dict(path=path, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), tokens=tokens, heads=heads,
                    kv_heads=kv_heads, head_size=head_size, block=block, norm=rng.random() < 0.6,
                    axes=rng.choice([1, 1, 2, 3, 4]), interleaved=rng.random() < 0.4, neox=rng.random() < 0.7,
                    rotated=head_size if rng.random() < 0.7 else head_size // 2, furthest=_log(rng, 8192, 500000))
    seqs, drafts = _log(rng, 1, 64), _log(rng, 1, 16)
    vocab = _log(rng, 1000, 262144) if rng.random() < 0.6 else rng.choice([32000, 128256])
    while seqs * (2 * drafts + 1) * vocab > 32 * 10 * 128256:
        seqs, drafts = max(1, seqs * 3 // 4), max(1, drafts * 7 // 8)
    return dict(path=path, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), seqs=seqs, drafts=drafts,
                ragged=rng.random() < 0.5, vocab=vocab, drafter=rng.random() < 0.7,
                greedy=rng.choice([0.0, 0.0, 0.3, 1.0]), masked=rng.choice([0.0, 0.0, 0.5, 0.99]))


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _spread(lo, hi, n):
    """n numbers spread from the largest to the smallest."""
    return [int(v) for v in np.linspace(hi, lo, n)]


def _shuffled(r, values):
    return [values[i] for i in r.permutation(len(values))]


def _i32(values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def _starts(counts):
    return [0] + [int(t) for t in np.cumsum(counts)]


def _new_tokens(case):
    return [1] * case["decodes"] + _spread(case["shortest"], case["longest"], case["chunks"])


def _cached(case):
    return _spread(case["near"], case["far"], case["decodes"] + case["chunks"])


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _prepare_chunk(case, r, g):
    H, KV, D, bs = case["heads"], case["kv_heads"], case["head_size"], case["block"]
    new = _shuffled(r, _new_tokens(case))
    lens = [c + n for c, n in zip(_shuffled(r, _cached(case)), new)]  # the new tokens are in the cache
    need = [max(1, -(-n // bs)) for n in lens]
    blocks, width = sum(need) + 3, max(need)
    ids, table, at = r.permutation(blocks), np.zeros((len(lens), width), np.int32), _starts(need)
    for s, n in enumerate(need):  # pages drawn at random from the pool
        table[s, :n] = ids[at[s]:at[s] + n]
    kc = torch.randn((blocks, KV, D // 8, bs, 8), generator=g, device="cuda", dtype=torch.float16)
    vc = torch.randn((blocks, KV, D, bs), generator=g, device="cuda", dtype=torch.float16)
    starts = _starts(new)
    st = dict(q=_normal(g, starts[-1], H, D, dtype=torch.float16), kc=kc, vc=vc, tables=_i32(table), lens=lens, new=new,
              at=starts, context=_i32(lens), starts=_i32(starts), scale=D ** -0.5, block=bs, kv=KV,
              window=case["window"])
    if own:
        from tensorlisp_amd import native as N

        st["node"] = N.ChunkAttention(len(lens), starts[-1], max(new), H, KV, D, bs, width, max(lens), D ** -0.5,
                                      window=case["window"])
        st["out"] = torch.empty_like(st["q"])
    return st


def _pair_axes(case):
    """Which axis each rotated pair takes its position from: a quarter of the pairs the first, the others the rest
    in equal parts, one after another or in turn."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    if axes == 1:
        return [0] * pairs
    first = pairs // 4
    parts = [first] + [(pairs - first) * (i + 1) // (axes - 1) - (pairs - first) * i // (axes - 1)
                       for i in range(axes - 1)]
    if case["interleaved"]:
        return [p % axes if p < axes * parts[p % axes] else 0 for p in range(pairs)]
    return [a for a in range(axes) for _ in range(parts[a])]


def _prepare_heads(case, r, g):
    T, H, KV, D, bs = case["tokens"], case["heads"], case["kv_heads"], case["head_size"], case["block"]
    # q, k and v as the fused projection leaves them: views of one buffer's rows
    rows = _normal(g, T, (H + 2 * KV) * D, dtype=DTYPES[case["dtype"]])
    q, k, v = rows.split([H * D, KV * D, KV * D], dim=1)
    # text goes on from a place of the context, an image's patches repeat its rows and columns
    first = int(r.integers(0, max(1, case["furthest"] - T)))
    at = first + np.arange(T)
    side = max(1, int(T ** 0.5))
    grid = [at, first + np.arange(T) // side, first + np.arange(T) % side, at // 2]
    # consecutive tokens of a few sequences, each from some place of a page on, in pages drawn at random
    pages = -(-T // bs) + 4
    blocks = pages + 3
    ids, place = r.permutation(blocks), int(r.integers(0, bs)) + np.arange(T)
    slots = ids[place // bs].astype(np.int64) * bs + place % bs
    freqs = 10000.0 ** (-2.0 * np.arange(case["rotated"] // 2) / case["rotated"])
    st = dict(q=q.unflatten(1, (H, D)), k=k.unflatten(1, (KV, D)), v=v.unflatten(1, (KV, D)),
              positions=_i32(np.stack(grid[:case["axes"]])), slots=torch.tensor(slots, device="cuda"), block=bs,
              freqs=torch.tensor(freqs.astype(np.float32), device="cuda"), rotated=case["rotated"], neox=case["neox"],
              pair_axes=torch.tensor(_pair_axes(case), device="cuda"), eps=1e-6,
              q_norm=1 + 0.2 * _normal(g, D) if case["norm"] else None,
              k_norm=1 + 0.2 * _normal(g, D) if case["norm"] else None,
              kc=torch.randn((blocks, KV, D // 8, bs, 8), generator=g, device="cuda", dtype=torch.float16),
              vc=torch.randn((blocks, KV, D, bs), generator=g, device="cuda", dtype=torch.float16),
              q_out=torch.empty((T, H, D), device="cuda", dtype=torch.float16))
    if own:
        from tensorlisp_amd import native as N

        st["node"] = N.HeadRope(H, KV, D, st["freqs"], pair_axes=_pair_axes(case), mode=2 if case["neox"] else 0,
                                eps=st["eps"])
    return st


def _prepare_verify(case, r, g):
    S, V, dtype = case["seqs"], case["vocab"], DTYPES[case["dtype"]]
    drafts = _shuffled(r, _spread(1, case["drafts"], S) if case["ragged"] else [case["drafts"]] * S)
    starts, rows = _starts(drafts), sum(drafts)
    # a language model's logits: a broad normal, and a few likely tokens well above it
    x = _normal(g, rows + S, V) * 2.5
    likely = torch.arange(12, device="cuda") * (V // 12) + torch.randint(0, V // 12, (rows + S, 12), generator=g,
                                                                        device="cuda")
    x.scatter_(1, likely, 6 + 4 * _normal(g, rows + S, 12))
    # sequence s has its drafts' rows and one more
    row = torch.tensor([starts[s] + s + i for s in range(S) for i in range(drafts[s])], device="cuda")
    of = torch.tensor([s for s in range(S) for _ in range(drafts[s])], device="cuda")
    y = x[row] + 0.7 * _normal(g, rows, V)  # a smaller model's, near the target's
    if case["masked"] > 0:  # a grammar allows few tokens
        off = torch.rand((rows + S, V), generator=g, device="cuda") < case["masked"]
        off.scatter_(1, likely[:, :3], False)
        x.masked_fill_(off, -math.inf)
        y.masked_fill_(off[row], -math.inf)
    x, y = x.to(dtype), y.to(dtype)
    temps = 0.6 + 0.6 * torch.rand(S, generator=g, device="cuda")
    temps[torch.tensor(r.random(S) < case["greedy"], device="cuda")] = 0.0
    # the drafted tokens: drawn from the drafter's distribution, its likeliest where the sequence is greedy
    t = torch.where(temps > 0, temps, 1.0)[of, None]
    noise = -torch.log(-torch.log(torch.rand((rows, V), generator=g, device="cuda").clamp(1e-30, 1 - 1e-7)))
    tokens = (y.float() / t + noise * (temps[of, None] > 0)).argmax(1).to(torch.int32)
    st = dict(target=x, draft=y if case["drafter"] else None, tokens=tokens, drafts=drafts, starts=_i32(starts),
              temps=temps, accept_at=torch.rand(rows, generator=g, device="cuda"), row=row, of=of,
              sample_at=torch.rand(S, generator=g, device="cuda"))
    if own:
        from tensorlisp_amd import native as N

        st["node"] = N.DraftVerify(S, rows, max(drafts), V, dtype=dtype, drafter=case["drafter"])
        st["out"] = [torch.empty(S, device="cuda", dtype=torch.int32),
                     torch.empty((S, max(drafts) + 1), device="cuda", dtype=torch.int32),
                     torch.empty(rows, device="cuda")]
    return st


def prepare(case, seed):
    make = dict(chunk=_prepare_chunk, heads=_prepare_heads, verify=_prepare_verify)
    st = make[case["path"]](case, np.random.default_rng(int(seed)), _gen(seed))
    st["path"] = case["path"]
    return st


# ----------------------------------------------------------------- one pass
def run(st):
    return (_RUN_OWN if own else _RUN_PLAIN)[st["path"]](st)


def _own_chunk(st):
    return st["node"](st["out"], st["q"], st["kc"], st["vc"], st["tables"], st["context"], st["starts"])


def _own_heads(st):
    st["node"](st["q"], st["k"], st["v"], st["positions"], st["q_out"], q_norm=st["q_norm"], k_norm=st["k_norm"],
               k_cache=st["kc"], v_cache=st["vc"], slots=st["slots"])
    return [st["q_out"], st["kc"], st["vc"]]


def _own_verify(st):
    return st["node"](st["target"], st["draft"], st["tokens"], st["starts"], st["temps"], st["accept_at"],
                      st["sample_at"], *st["out"])


def _plain_chunk(st):
    """Sequence by sequence: softmax(scale q.k) over the keys that each row sees, times v."""
    q, bs, KV = st["q"], st["block"], st["kv"]
    _, H, D = q.shape
    out = torch.empty_like(q)
    for s, (L, n) in enumerate(zip(st["lens"], st["new"])):
        pages = st["tables"][s, :-(-L // bs)].long()
        k = st["kc"][pages].permute(1, 0, 3, 2, 4).reshape(KV, -1, D)[:, :L].float()
        v = st["vc"][pages].permute(1, 0, 3, 2).reshape(KV, -1, D)[:, :L].float().contiguous()
        rows = q[st["at"][s]:st["at"][s] + n].float().transpose(0, 1).reshape(KV, -1, D)  # a kv head's queries
        i, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")
        see = j <= i if not st["window"] else (j <= i) & (j > i - st["window"])
        x = torch.bmm(rows, k.transpose(1, 2).contiguous()).mul_(st["scale"]).reshape(H, n, L)
        x.masked_fill_(~see, -math.inf)
        x = x.sub_(x.amax(-1, keepdim=True)).exp_()  # every row sees itself
        o = torch.bmm(x.reshape(KV, -1, L), v).reshape(H, n, D) / x.sum(-1, keepdim=True)
        out[st["at"][s]:st["at"][s] + n] = o.transpose(0, 1).to(out.dtype)
    return out


def _plain_heads(st):
    R = st["rotated"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if st["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + st["eps"]) * st["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + st["eps"]) * st["k_norm"]
    # angles of far positions lose their fraction in 32 bits
    angle = st["positions"][st["pair_axes"]].double().T * st["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = (slice(0, R // 2), slice(R // 2, R)) if st["neox"] else (slice(0, R, 2), slice(1, R, 2))

    def rotate(x):
        y = x.clone()
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., a] * sin + x[..., b] * cos
        return y.to(torch.float16)

    page, off = st["slots"] // st["block"], st["slots"] % st["block"]
    st["q_out"].copy_(rotate(q))
    st["kc"][page, :, :, off] = rotate(k).unflatten(2, (-1, 8))
    st["vc"][page, :, :, off] = v.to(torch.float16)
    return [st["q_out"], st["kc"], st["vc"]]


def _plain_verify(st):
    """In 64 bits throughout: a sum over a vocabulary decides between neighbours that differ by less than 32 hold."""
    tokens, row, of, n = st["tokens"].long()[:, None], st["row"], st["of"], torch.tensor(st["drafts"], device="cuda")
    S, rows = len(n), len(row)
    last = st["starts"].long()[1:] + torch.arange(S, device="cuda")  # each sequence's row behind its drafts

    def distribution(logits, temps):
        x = logits.double()
        likeliest = torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
        x = x.sub_(x.amax(1, keepdim=True)).div_(torch.where(temps > 0, temps, 1.0)[:, None]).exp_()
        return torch.where(temps[:, None] > 0, x / x.sum(1, keepdim=True), likeliest)

    every = torch.empty(rows + S, device="cuda", dtype=torch.long)
    every[row], every[last] = of, torch.arange(S, device="cuda")
    p = distribution(st["target"], st["temps"][every])
    if st["draft"] is None:
        q = torch.zeros((rows, p.shape[1]), device="cuda", dtype=torch.float64).scatter_(1, tokens, 1.0)
    else:
        q = distribution(st["draft"], st["temps"][of])
    px, qx = p[row].gather(1, tokens)[:, 0], q.gather(1, tokens)[:, 0]
    good = st["accept_at"].double() * qx < px
    first = st["starts"].long()[:-1]
    bad = torch.cat([torch.zeros(1, device="cuda", dtype=torch.long), (~good).long().cumsum(0)])
    before = bad[:-1] - bad[first[of]]  # refused ones of the sequence before this one
    accepted = torch.zeros(S, device="cuda", dtype=torch.long).index_add_(0, of, (good & (before == 0)).long())
    # where one was refused, the target's distribution above the drafter's takes its place
    stop = accepted < n
    at = (first + accepted).clamp(max=rows - 1)
    left = p[first + torch.arange(S, device="cuda") + accepted]
    rest = torch.where(stop[:, None], (left - q[at]).clamp(min=0), left)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, left)
    cdf = rest.cumsum(1)
    drawn = (cdf <= (st["sample_at"].double() * cdf[:, -1])[:, None]).sum(1)
    width = max(st["drafts"]) + 1
    place = torch.arange(width, device="cuda")
    proposed = st["tokens"].long()[(first[:, None] + place).clamp(max=rows - 1)]
    out = torch.where(place < accepted[:, None], proposed, torch.where(place == accepted[:, None], drawn[:, None], -1))
    ratio = torch.where(qx > 0, (px / qx).clamp(max=1), (px > 0).double())
    return [accepted.to(torch.int32), out.to(torch.int32), ratio.float()]


_RUN_OWN = dict(chunk=_own_chunk, heads=_own_heads, verify=_own_verify)
_RUN_PLAIN = dict(chunk=_plain_chunk, heads=_plain_heads, verify=_plain_verify)


# ---------------------------------------------------------------- the least
def _seen(n, L, window):
    """(query, key) pairs of n new tokens at the end of L, and the keys that any of them sees."""
    if not window:
        return n * L - n * (n - 1) // 2, L
    return sum(min(window, L - n + i + 1) for i in range(n)), min(L, n + window - 1)


def work(case):
    if case["path"] == "verify":
        S = case["seqs"]
        rows = sum(_spread(1, case["drafts"], S)) if case["ragged"] else S * case["drafts"]
        n = (rows + S + (rows if case["drafter"] else 0)) * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 12 * rows + 16 * S, "flops": 5 * n}
    H, KV, D = case["heads"], case["kv_heads"], case["head_size"]
    if case["path"] == "heads":
        n = case["tokens"] * (H + 2 * KV) * D
        return {"bytes": n * ((4 if case["dtype"] == "f32" else 2) + 2) + case["tokens"] * (4 * case["axes"] + 8),
                "flops": 9 * n}
    seen = [_seen(n, c + n, case["window"]) for c, n in zip(_cached(case), _new_tokens(case))]
    rows = sum(_new_tokens(case))
    return {"bytes": sum(keys for _, keys in seen) * KV * D * 2 * 2 + rows * 2 * H * D * 2,
            "flops": 4 * H * D * sum(pairs for pairs, _ in seen)}


# ------------------------------------------------------------- in 64 bits
def _exact_chunk(case, st):
    """One head and 1024 rows at a time."""
    q, bs, w = st["q"], case["block"], case["window"]
    out = torch.empty(q.shape, device="cuda", dtype=torch.float64)
    for s, (L, n) in enumerate(zip(st["lens"], st["new"])):
        pos = torch.arange(L, device="cuda")
        page, off = st["tables"][s].long()[pos // bs], pos % bs
        for h in range(case["heads"]):
            g = h // (case["heads"] // case["kv_heads"])
            keys, values = st["kc"][page, g, :, off].reshape(L, -1).double(), st["vc"][page, g, :, off].double()
            for b in range(0, n, 1024):
                at = slice(st["at"][s] + b, st["at"][s] + min(n, b + 1024))
                where = torch.arange(L - n + b, L - n + min(n, b + 1024), device="cuda")[:, None]
                hidden = (pos > where) | (pos <= where - w if w else pos < 0)
                logit = torch.addmm(torch.zeros((), device="cuda", dtype=torch.float64), q[at, h].double(),
                                    keys.t().contiguous(), alpha=st["scale"]).masked_fill(hidden, -torch.inf)
                out[at, h] = torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)) @ values
    return out


def _exact_heads(case, st):
    kc, vc = st["kc"].double(), st["vc"].double()
    half = case["rotated"] // 2
    one, two = (range(half), range(half, 2 * half)) if case["neox"] else (range(0, 2 * half, 2), range(1, 2 * half, 2))
    where = torch.stack([st["positions"][a] for a in _pair_axes(case)], 1).double()
    turn = torch.polar(torch.ones_like(where), where * st["freqs"].double())[:, None]
    outs = []
    for x, weight in ((st["q"].double(), st["q_norm"]), (st["k"].double(), st["k_norm"])):
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["head_size"] + st["eps"]) * weight.double()
        z = torch.complex(x[..., list(one)], x[..., list(two)]) * turn
        x = x.clone()
        x[..., list(one)], x[..., list(two)] = z.real, z.imag
        outs.append(x)
    page, off = torch.div(st["slots"], case["block"], rounding_mode="floor"), st["slots"] % case["block"]
    kc[page, :, :, off] = outs[1].reshape(len(page), case["kv_heads"], -1, 8)
    vc[page, :, :, off] = st["v"].double()
    return [outs[0], kc, vc]


def _exact_verify(case, st):
    """The chance that each drafted token is accepted with."""
    out = []
    for i, (row, s, token) in enumerate(zip(st["row"].tolist(), st["of"].tolist(), st["tokens"].tolist())):
        t = float(st["temps"][s])
        x = st["target"][row].double()
        y = None if st["draft"] is None else st["draft"][i].double()
        if t == 0.0:
            p = 0.0 if (x[token] < x.max()) or (x[:token] == x[token]).any() else 1.0
            q = 1.0 if y is None else 0.0 if (y[token] < y.max()) or (y[:token] == y[token]).any() else 1.0
        else:
            p = float(torch.exp(x[token] / t - torch.logsumexp(x / t, 0)))
            q = 1.0 if y is None else float(torch.exp(y[token] / t - torch.logsumexp(y / t, 0)))
        out.append(min(1.0, p / q) if q > 0 else float(p > 0))
    return [None, None, torch.tensor(out, device="cuda", dtype=torch.float64)]


def exact(case, seed):
    return dict(chunk=_exact_chunk, heads=_exact_heads, verify=_exact_verify)[case["path"]](case, prepare(case, seed))
