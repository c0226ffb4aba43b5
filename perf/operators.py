"""The serving operators around a paged KV cache, and the calls they are measured on.

A server that drafts tokens and verifies them in trees runs, beside the decode
step: attention of whole prompts packed one after another (``native.packed_attention``),
attention of a tree of drafted tokens over the paged cache
(``native.TreeAttention``), the cache moves that fork a sequence and keep an
accepted branch (``native.KVPools``), and the log probabilities it accepts by
and answers with (``native.TokenLogprobs``).

``listed`` names fixed cases, ``draw`` gives others of the same ranges,
``prepare`` builds what a program has in hand, ``run`` is one pass (with ``own``
through the framework, else in plain torch), ``work`` the bytes and operations
it cannot do without, ``exact`` the result in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a short question to an 8B model: one prompt of odd length
        dict(name="prompt 1x77", path="packed", dtype="f16", heads=32, kv_heads=8, head_size=128, longest=77,
             shortest=77, seqs=1),
        # a batch of prompts of different lengths prefilled together
        dict(name="prompts 16x100..2000", path="packed", dtype="f16", heads=32, kv_heads=8, head_size=128,
             longest=2000, shortest=100, seqs=16),
        # a long document, one prompt, bf16 activations (the largest)
        dict(name="prompt bf16 1x8191", path="packed", dtype="bf16", heads=32, kv_heads=8, head_size=128,
             longest=8191, shortest=8191, seqs=1),
        # one chat being verified: a small tree over a short context, where latency counts
        dict(name="tree 1 seq x 7", path="tree", heads=32, kv_heads=8, head_size=128, block=16, seqs=1, drafts=7,
             ragged=False, shortest=600, longest=600),
        # a full batch with small trees of different sizes over contexts of 512..8192
        dict(name="trees 32 seqs x 1..8", path="tree", heads=32, kv_heads=8, head_size=128, block=16, seqs=32,
             drafts=8, ragged=True, shortest=512, longest=8192),
        # wide trees of 63 tokens, 16 sequences
        dict(name="trees 16 seqs x 63", path="tree", heads=32, kv_heads=8, head_size=128, block=16, seqs=16,
             drafts=63, ragged=False, shortest=512, longest=4096),
        # forking one sequence: its last page copied before the fork writes to it, in every layer
        dict(name="fork 1 page x 32 layers", path="copy", layers=32, kv_heads=8, head_size=128, block=16, pages=1),
        # a batch of prompts moved to other pages
        dict(name="copy 300 pages x 16 layers", path="copy", layers=16, kv_heads=8, head_size=128, block=16,
             pages=300),
        # the accepted branch of one tree
        dict(name="keep 1 seq x 32 layers", path="keep", layers=32, kv_heads=8, head_size=128, block=16, seqs=1,
             drafts=7),
        # a full batch's accepted branches
        dict(name="keep 32 seqs x 16 layers", path="keep", layers=16, kv_heads=8, head_size=128, block=16, seqs=32,
             drafts=63),
        # one sampled token's log probability and five alternatives, vocabulary of a Llama 3 model
        dict(name="logprobs 1x128256", path="logprobs", dtype="f32", rows=1, vocab=128256, top=5, masked=0.0),
        # a prompt scored token by token, twenty alternatives
        dict(name="logprobs 777x128256", path="logprobs", dtype="f32", rows=777, vocab=128256, top=20, masked=0.0),
    ]


# ------------------------------------------------------------------ drawing
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(32, 8), (32, 8), (32, 32), (16, 8), (28, 4), (8, 1), (12, 2), (64, 8), (8, 2), (4, 1)])


def draw(rng):
    path = rng.choices(["packed", "tree", "copy", "keep", "logprobs"], [5, 5, 1, 2, 3])[0]
    head_size = rng.choice([64, 128, 128, 128, 80, 96, 112, 192, 256])
    if path == "packed":
        heads, kv_heads = _heads(rng)
        longest, seqs = _log(rng, 1, 8191), _log(rng, 1, 64)
        while longest * longest * seqs * heads * head_size > 8191 * 8191 * 32 * 128:
            seqs = max(1, seqs // 2)
            longest = longest if seqs > 1 else longest * 3 // 4
        return dict(path=path, dtype=rng.choice(["f16", "bf16"]), heads=heads, kv_heads=kv_heads, head_size=head_size,
                    longest=longest, shortest=max(1, int(longest * rng.uniform(0.01, 1.0))), seqs=seqs)
    if path == "tree":
        heads, kv_heads = _heads(rng)
        longest, seqs, drafts = _log(rng, 1, 8192), _log(rng, 1, 32), _log(rng, 1, 64)
        while longest * seqs * drafts * heads * head_size > 16 * 4096 * 63 * 32 * 128 or \
                longest * seqs * kv_heads * head_size > 32 * 8192 * 8 * 128:
            seqs, longest = max(1, seqs * 3 // 4), max(64, longest * 3 // 4)
        return dict(path=path, heads=heads, kv_heads=kv_heads, head_size=head_size, block=rng.choice([8, 16, 16, 32]),
                    seqs=seqs, drafts=drafts, ragged=rng.random() < 0.6,
                    shortest=int(longest * rng.uniform(0.0, 1.0)), longest=longest)
    kv_heads, block = rng.choice([1, 2, 4, 8, 8, 32]), rng.choice([8, 16, 16, 32])
    if path in ("copy", "keep"):
        layers = rng.choice([1, 2, 16, 32, 61, 80])
        units = layers * kv_heads * head_size * block
        if path == "copy":
            pages = _log(rng, 1, 512)
            while pages * units > 300 * 16 * 8 * 128 * 16:
                pages = max(1, pages // 2) if pages > 1 else 1
                if pages == 1:
                    break
            return dict(path=path, layers=layers, kv_heads=kv_heads, head_size=head_size, block=block, pages=pages)
        seqs = _log(rng, 1, 32)
        while seqs > 1 and seqs * 160 * layers * kv_heads * head_size > 32 * 160 * 16 * 8 * 128:
            seqs = seqs // 2
        return dict(path=path, layers=layers, kv_heads=kv_heads, head_size=head_size, block=block, seqs=seqs,
                    drafts=_log(rng, 2, 64))
    rows, vocab = _log(rng, 1, 2048), _log(rng, 1000, 262144) if rng.random() < 0.6 else rng.choice([32000, 128256])
    while rows * vocab > 777 * 128256:
        rows = rows * 3 // 4
    return dict(path=path, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), rows=rows, vocab=vocab,
                top=rng.choice([0, 1, 5, 8, 20, 32]), masked=rng.choice([0.0, 0.0, 0.5, 0.999]))


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _spread(lo, hi, n):
    """n lengths spread from the shortest to the longest."""
    return [int(v) for v in np.linspace(hi, lo, n)]


def _lengths(case):
    return _spread(case["shortest"], case["longest"], case["seqs"])


def _drafts(case):
    return _spread(1, case["drafts"], case["seqs"]) if case.get("ragged", True) else [case["drafts"]] * case["seqs"]


def _shuffled(r, values):
    return [values[i] for i in r.permutation(len(values))]


def _i32(values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def _i64(values):
    return torch.tensor(np.asarray(values, np.int64), device="cuda")


def _tree(r, n):
    """A drafted tree, likeliest chain first: the parent of each token (-1: the last committed one)."""
    chain = int(r.integers(max(1, n // 4), n + 1)) if n > 1 else 1
    parents = list(range(-1, chain - 1))
    depth = list(range(chain))
    while len(parents) < n:  # branches no deeper than the chain
        p = int(r.integers(-1, len(parents)))
        d = depth[p] + 1 if p >= 0 else 0
        if d < chain:
            parents.append(p)
            depth.append(d)
    return parents


def _ancestors(parents):
    """Bit j of token i's mask: i sees drafted token j (its ancestors and itself)."""
    masks = []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | (1 << i))
    return masks


def _signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


def _pools(case, blocks, g, n):
    """The key and the value pools of n layers, as one buffer each."""
    kv, hs, bs = case["kv_heads"], case["head_size"], case["block"]
    kc = torch.randn((n, blocks, kv, hs // 8, bs, 8), generator=g, device="cuda", dtype=torch.float16)
    vc = torch.randn((n, blocks, kv, hs, bs), generator=g, device="cuda", dtype=torch.float16)
    return kc, vc


def _tables(r, lens, block, blocks=None):
    """Pages drawn at random from a pool, by default of three more than the sequences use."""
    need = [max(1, -(-n // block)) for n in lens]
    blocks = sum(need) + 3 if blocks is None else blocks
    ids, width = r.permutation(blocks), max(need)
    table = np.zeros((len(lens), width), np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, blocks


def _prepare_packed(case, r, g):
    H, KV, D, dt = case["heads"], case["kv_heads"], case["head_size"], DTYPES[case["dtype"]]
    lens = _shuffled(r, _lengths(case))
    starts = [0] + [int(t) for t in np.cumsum(lens)]
    # q, k and v as the fused projection leaves them: views of one buffer's rows
    rows = torch.randn((starts[-1], (H + 2 * KV) * D), generator=g, device="cuda", dtype=torch.float32).to(dt)
    q, k, v = rows.split([H * D, KV * D, KV * D], dim=1)
    st = dict(q=q.unflatten(1, (H, D)), k=k.unflatten(1, (KV, D)), v=v.unflatten(1, (KV, D)), lens=lens, at=starts,
              starts=_i32(starts), scale=D ** -0.5)
    st["out"] = torch.empty((starts[-1], H, D), device="cuda", dtype=dt)
    return st


def _prepare_tree(case, r, g):
    H, KV, D, bs = case["heads"], case["kv_heads"], case["head_size"], case["block"]
    S = case["seqs"]
    drafts = _shuffled(r, _drafts(case))
    lens = [n + d for n, d in zip(_shuffled(r, _lengths(case)), drafts)]  # the drafted tokens are in the cache
    table, blocks = _tables(r, lens, bs)
    kc, vc = _pools(case, blocks, g, 1)
    starts = [0] + [int(t) for t in np.cumsum(drafts)]
    masks = [m for n in drafts for m in _ancestors(_tree(r, n))]
    q = torch.randn((starts[-1], H, D), generator=g, device="cuda", dtype=torch.float16)
    st = dict(q=q, kc=kc[0], vc=vc[0], tables=_i32(table), lens=lens, drafts=drafts, at=starts, context=_i32(lens),
              starts=_i32(starts), masks=_i64([_signed(m) for m in masks]), scale=D ** -0.5, block=bs, kv=KV)
    if own:
        from tensorlisp_amd import native as N

        st["node"] = N.TreeAttention(S, starts[-1], max(drafts), H, KV, D, bs, table.shape[1], max(lens), D ** -0.5)
        st["out"] = torch.empty_like(q)
    return st


def _prepare_copy(case, r, g):
    blocks = 2 * case["pages"] + 5
    kc, vc = _pools(case, blocks, g, case["layers"])
    ids = r.permutation(blocks)
    n = case["pages"]
    src = ids[r.integers(0, n, n)] if n > 1 else ids[:1]  # a page forked more than once among them
    st = dict(kc=kc, vc=vc, pairs=_i64(np.stack([src, ids[n:2 * n]], 1)))
    if own:
        st["pools"] = _own_pools(case, kc, vc)
    return st


def _own_pools(case, kc, vc):
    from tensorlisp_amd import native as N

    return N.KVPools(list(kc), list(vc), case["kv_heads"], case["head_size"], case["block"])


def _prepare_keep(case, r, g):
    S, bs = case["seqs"], case["block"]
    drafts = _shuffled(r, _drafts(case))
    lens = [int(n) + d for n, d in zip(r.integers(0, 97, S), drafts)]
    table, blocks = _tables(r, lens, bs, S * (-(-(96 + case["drafts"]) // bs)) + 3)
    kc, vc = _pools(case, blocks, g, case["layers"])
    keep = []
    for n in drafts:  # the accepted branch: a random token and its ancestors
        keep.append(_ancestors(_tree(r, n))[int(r.integers(n // 2, n))])
    starts = [0] + [int(t) for t in np.cumsum(drafts)]
    st = dict(kc=kc, vc=vc, tables=_i32(table), lens=lens, drafts=drafts, context=_i32(lens), starts=_i32(starts),
              keep=_i64([_signed(m) for m in keep]), block=bs)
    if own:
        st["pools"], st["new_lens"] = _own_pools(case, kc, vc), torch.empty_like(st["context"])
    return st


def _prepare_logprobs(case, r, g):
    R, V = case["rows"], case["vocab"]
    # a language model's logits: a broad normal, and a few likely tokens well above it
    x = torch.randn((R, V), generator=g, device="cuda") * 2.5
    likely = torch.arange(12, device="cuda") * (V // 12) + torch.randint(0, V // 12, (R, 12), generator=g, device="cuda")
    x.scatter_(1, likely, 6 + 4 * torch.randn((R, 12), generator=g, device="cuda"))
    tokens = likely.gather(1, torch.randint(0, 12, (R, 1), generator=g, device="cuda"))
    if case["masked"] > 0:  # a grammar allows few tokens, the sampled one among them
        off = torch.rand((R, V), generator=g, device="cuda") < case["masked"]
        x.masked_fill_(off.scatter_(1, tokens, False), -math.inf)
    st = dict(logits=x.to(DTYPES[case["dtype"]]), tokens=tokens[:, 0].to(torch.int32), top=case["top"])
    if own:
        from tensorlisp_amd import native as N

        st["node"] = N.TokenLogprobs(R, V, case["top"], st["logits"].dtype)
        st["out"] = [torch.empty(R, device="cuda"), torch.empty(R, device="cuda"),
                     torch.empty((R, case["top"]), device="cuda"),
                     torch.empty((R, case["top"]), device="cuda", dtype=torch.int32)]
    return st


def prepare(case, seed):
    make = dict(packed=_prepare_packed, tree=_prepare_tree, copy=_prepare_copy, keep=_prepare_keep,
                logprobs=_prepare_logprobs)
    st = make[case["path"]](case, np.random.default_rng(int(seed)), _gen(seed))
    st["path"] = case["path"]
    return st


# ----------------------------------------------------------------- one pass
def run(st):
    return (_RUN_OWN if own else _RUN_PLAIN)[st["path"]](st)


def _own_packed(st):
    from tensorlisp_amd import native as N

    return N.packed_attention(st["q"], st["k"], st["v"], st["starts"], max(st["lens"]), st["scale"], out=st["out"])


def _own_tree(st):
    return st["node"](st["out"], st["q"], st["kc"], st["vc"], st["tables"], st["context"], st["starts"], st["masks"])


def _own_copy(st):
    st["pools"].copy_blocks(st["pairs"])
    return [st["kc"], st["vc"]]


def _own_keep(st):
    st["pools"].compact(st["tables"], st["context"], st["starts"], st["keep"], st["new_lens"], max(st["drafts"]))
    return [st["kc"], st["vc"], st["new_lens"]]


def _own_logprobs(st):
    return st["node"](st["logits"], st["tokens"], *st["out"])


def _attend(q, k, v, see, scale):
    """softmax(scale q.k) over the keys that each row sees, times v: q (H, n, D), k and v (KV, L, D), see (n, L)."""
    H, n, D = q.shape
    KV, L, _ = k.shape
    out = torch.empty((H, n, D), device=q.device)
    for h in range(KV):
        rows = slice(h * (H // KV), (h + 1) * (H // KV))
        s = torch.matmul(q[rows].float().reshape(-1, D), k[h].float().t().contiguous()).reshape(-1, n, L) * scale
        s = s.masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1.0, total)
        out[rows] = torch.matmul(p.reshape(-1, L), v[h].float()).reshape(-1, n, D)
    return out


def _plain_packed(st):
    out = st["out"]
    for s, n in enumerate(st["lens"]):
        rows = slice(st["at"][s], st["at"][s] + n)
        see = torch.ones((n, n), device="cuda", dtype=torch.bool).tril()
        o = _attend(st["q"][rows].transpose(0, 1), st["k"][rows].transpose(0, 1), st["v"][rows].transpose(0, 1), see,
                    st["scale"])
        out[rows] = o.transpose(0, 1).to(out.dtype)
    return out


def _plain_tree(st):
    q, bs = st["q"], st["block"]
    _, H, D = q.shape
    out = torch.empty_like(q)
    for s, (L, n) in enumerate(zip(st["lens"], st["drafts"])):
        pages = st["tables"][s, :-(-L // bs)].long()
        k = st["kc"][pages].permute(1, 0, 3, 2, 4).reshape(st["kv"], -1, D)[:, :L]
        v = st["vc"][pages].permute(1, 0, 3, 2).reshape(st["kv"], -1, D)[:, :L]
        rows = slice(st["at"][s], st["at"][s] + n)
        see = torch.ones((n, L), device="cuda", dtype=torch.bool)
        see[:, L - n:] = (st["masks"][rows, None] >> torch.arange(n, device="cuda")) & 1 == 1
        out[rows] = _attend(q[rows].transpose(0, 1), k, v, see, st["scale"]).transpose(0, 1).to(out.dtype)
    return out


def _plain_copy(st):
    src, dst = st["pairs"][:, 0], st["pairs"][:, 1]
    for pool in (st["kc"], st["vc"]):
        pool[:, dst] = pool[:, src]
    return [st["kc"], st["vc"]]


def _plain_keep(st):
    bs, new = st["block"], st["context"].clone()
    n_max, L_max = max(st["drafts"]), max(st["lens"])
    bit = torch.arange(n_max, device="cuda")
    n = (st["starts"][1:] - st["starts"][:-1]).long()
    first = st["context"].long() - n
    kept = ((st["keep"][:, None] >> bit) & 1 == 1) & (bit < n[:, None])
    to = first[:, None] + kept.cumsum(1) - 1  # the place of each kept token
    new.copy_(first + kept.sum(1))
    frm = (first[:, None] + bit).clamp(max=L_max)

    def slot(pos):  # (page, place in it) of each position
        pos = pos.clamp(min=0)
        page = torch.gather(st["tables"].long(), 1, (pos // bs).clamp(max=st["tables"].shape[1] - 1))
        return page[kept], (pos % bs)[kept]

    (sp, so), (dp, do) = slot(frm), slot(to)
    for k, v in zip(st["kc"], st["vc"]):
        k[dp, :, :, do] = k[sp, :, :, so]
        v[dp, :, :, do] = v[sp, :, :, so]
    return [st["kc"], st["vc"], new]


def _plain_logprobs(st):
    x = st["logits"].float()
    top = x.amax(1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    d = x - top
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse[:, 0] - torch.where(e > 0, e * d, 0.0).sum(1) / total[:, 0]
    lp = torch.gather(d, 1, st["tokens"].long()[:, None])[:, 0] - lse[:, 0]
    # ties to the lowest index: a stable sort of the values from the largest down
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :st["top"]]
    return [lp, entropy, torch.gather(d, 1, ids) - lse, ids.to(torch.int32)]


_RUN_OWN = dict(packed=_own_packed, tree=_own_tree, copy=_own_copy, keep=_own_keep, logprobs=_own_logprobs)
_RUN_PLAIN = dict(packed=_plain_packed, tree=_plain_tree, copy=_plain_copy, keep=_plain_keep,
                  logprobs=_plain_logprobs)


# ---------------------------------------------------------------- the least
def work(case):
    path = case["path"]
    if path == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (12 + 8 * case["top"]),
                "flops": 5 * n}
    KV, D = case["kv_heads"], case["head_size"]
    if path == "copy":
        page = KV * D * case["block"] * 2
        return {"bytes": 2 * 2 * case["layers"] * case["pages"] * page + 16 * case["pages"], "flops": 0}
    if path == "keep":
        # about a token in eight is kept and moves; each is read and written, keys and values
        moved = sum(max(1, n // 8) for n in _drafts(case))
        return {"bytes": 2 * 2 * case["layers"] * moved * KV * D * 2 + 20 * case["seqs"], "flops": 0}
    H = case["heads"]
    if path == "packed":
        tokens, pairs = sum(_lengths(case)), sum(n * (n + 1) // 2 for n in _lengths(case))
        return {"bytes": tokens * (2 * H + 2 * KV) * D * 2, "flops": 4 * H * D * pairs}
    rows, context = sum(_drafts(case)), sum(_lengths(case)) + sum(_drafts(case))
    return {"bytes": context * KV * D * 2 * 2 + rows * (2 * H * D * 2 + 8),
            "flops": 4 * H * D * (rows * context // case["seqs"])}


# ------------------------------------------------------------- in 64 bits
def _softmax_rows(q, keys, values, visible, scale):
    """One head in 64 bits: rows of q over the keys that `visible` allows; rows that see nothing are zero."""
    logit = torch.where(visible, (q.double() @ keys.double().T.contiguous()) * scale, -torch.inf)
    weight = torch.where(visible, torch.exp(logit - torch.logsumexp(logit, 1, keepdim=True)), 0.0)
    return weight @ values.double()


def exact(case, seed):
    if case["path"] in ("copy", "keep"):  # moves, not computed numbers
        return None
    st = prepare(case, seed)
    if case["path"] == "logprobs":
        lp, ent, tops = [], [], []
        for row, token in zip(st["logits"], st["tokens"].tolist()):
            x = row.double()
            logp = x - torch.logsumexp(x, 0)
            lp.append(logp[token])
            ent.append(-torch.where(torch.isinf(logp), 0.0, torch.exp(logp) * logp).sum())
            tops.append(torch.topk(logp, st["top"])[0])
        return [torch.stack(lp), torch.stack(ent), torch.stack(tops), None]
    q = st["q"]
    out = torch.empty(q.shape, device="cuda", dtype=torch.float64)
    group = case["heads"] // case["kv_heads"]
    for s, n in enumerate(st["lens"] if case["path"] == "packed" else st["drafts"]):
        a = st["at"][s]
        if case["path"] == "tree":
            L = st["lens"][s]
            pos = torch.arange(L, device="cuda")
            page, off = st["tables"][s].long()[pos // st["block"]], pos % st["block"]
            see = torch.ones((n, L), dtype=torch.bool)
            for i, m in enumerate(st["masks"][a:a + n].tolist()):
                for j in range(n):
                    see[i, L - n + j] = bool(m & (1 << j))
            see = see.cuda()
        for h in range(case["heads"]):
            g = h // group
            if case["path"] == "packed":
                for b in range(0, n, 2048):  # rows b.. see the keys up to themselves
                    e = min(n, b + 2048)
                    see = torch.arange(e, device="cuda") <= torch.arange(b, e, device="cuda")[:, None]
                    out[a + b:a + e, h] = _softmax_rows(q[a + b:a + e, h], st["k"][a:a + e, g], st["v"][a:a + e, g],
                                                        see, st["scale"])
            else:
                keys = st["kc"][page, g, :, off].reshape(L, -1)
                out[a:a + n, h] = _softmax_rows(q[a:a + n, h], keys, st["vc"][page, g, :, off], see, st["scale"])
    return out
