"""GPU: a serving step's operators together, as a server that mixes prompts in pieces with drafting sequences uses them.

The heads of a step's tokens (views of a fused projection) are normed, turned by three axes of positions and written to
the cache; the new tokens attend to it; the rows of the drafting sequences give logits, and their drafts are verified.
What was refused is overwritten by the next step's tokens.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from step_refs import chunk_reference, into_caches, new_token_starts, rope_reference, verify_reference
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu
H, KV, D, BS, VOCAB, MOST, BLOCKS, WIDTH = 8, 2, 128, 16, 3001, 5, 40, 10
AXES = N.rope_sections([16, 24, 24])


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


class Model:
    """One layer's weights, its cache and the three nodes, for up to 4 sequences and 200 tokens a step."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        self.kc = torch.full((BLOCKS, KV, D // 8, BS, 8), float("nan"), dtype=torch.float16, device="cuda")
        self.vc = torch.full((BLOCKS, KV, D, BS), float("nan"), dtype=torch.float16, device="cuda")
        self.q_norm, self.k_norm = (1 + 0.1 * self.normal(D) for _ in range(2))
        self.head = self.normal(H * D, VOCAB) * 0.2
        self.freqs = N.rope_freqs(D, 10000.0)
        self.rope = N.HeadRope(H, KV, D, self.freqs, pair_axes=AXES, mode=2)
        self.attention = N.ChunkAttention(4, 200, 150, H, KV, D, BS, WIDTH, WIDTH * BS, D ** -0.5)
        self.verify = N.DraftVerify(4, 20, MOST, VOCAB, torch.float32, drafter=True)
        self.table = i32(np.random.default_rng(seed).permutation(BLOCKS).reshape(4, WIDTH))

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def heads(self, rows):
        q, k, v = rows.split([H * D, KV * D, KV * D], 1)
        return q.unflatten(1, (H, D)), k.unflatten(1, (KV, D)), v.unflatten(1, (KV, D))

    def attend(self, rows, positions, slots, table, context, starts, q, out):
        self.rope(*self.heads(rows), positions, q, q_norm=self.q_norm, k_norm=self.k_norm, k_cache=self.kc, v_cache=self.vc,
                  slots=slots)
        return self.attention(out, q, self.kc, self.vc, table, context, starts)


def places(table, s, positions):
    return [int(table[s, p // BS]) * BS + p % BS for p in positions]


def test_pieces_decoding_and_drafts(gpu):
    m, r = Model(70), np.random.default_rng(70)
    table, lens = m.table.cpu().numpy(), [0, 0, 0, 0]
    for step in range(5):
        # sequence 3 gets its prompt in pieces; the others have a prompt first, then a token and its drafts
        drafts = [0, 0, 0] if step == 0 else [int(x) for x in r.integers(0, MOST + 1, 3)]
        new = [90, 1, 33] if step == 0 else [n + 1 for n in drafts]
        new.append([7, 0, 31, 1, 64][step])
        starts = new_token_starts(new)
        at = [lens[s] + i for s in range(4) for i in range(new[s])]
        slots = [p for s in range(4) for p in places(table, s, range(lens[s], lens[s] + new[s]))]
        positions = torch.tensor([at, [p // 3 for p in at], [2 * p for p in at]], dtype=torch.int32)
        rows, context = m.normal(starts[-1], (H + 2 * KV) * D), [a + b for a, b in zip(lens, new)]
        before = m.kc.clone(), m.vc.clone()
        q = torch.empty((starts[-1], H, D), dtype=torch.float16, device="cuda")
        out = m.attend(rows, positions.cuda(), torch.tensor(slots, dtype=torch.int64, device="cuda"), m.table, i32(context),
                       i32(starts), q, torch.empty_like(q))
        # the heads and the cache
        hq, hk, hv = m.heads(rows)
        for x, norm, got in ((hq, m.q_norm, q), (hk, m.k_norm, None)):
            want, tol = rope_reference(x, norm, 1e-6, positions, AXES, m.freqs, 2, 1.0, torch.float16)
            if got is None:
                pg, off = torch.tensor(slots) // BS, torch.tensor(slots) % BS
                got = m.kc.cpu()[pg, :, :, off].reshape(-1, KV, D)
                kc, vc = into_caches(before[0].cpu(), before[1].cpu(), got, hv.half().cpu(), slots)
                assert torch.equal(m.kc.cpu().view(torch.int16), kc.view(torch.int16))  # nothing else was written
                assert torch.equal(m.vc.cpu().view(torch.int16), vc.view(torch.int16))
            assert ((got.cpu().double() - want).abs() <= tol).all()
        # the attention
        want, tol = chunk_reference(q, m.kc, m.vc, table, context, starts, D ** -0.5)
        assert ((out.cpu().double() - want).abs() <= tol).all(), step
        lens[3] = context[3]
        if step == 0:
            lens[:3] = context[:3]
            continue
        # the drafts
        tokens = torch.randint(0, VOCAB, (sum(drafts),), generator=m.g, device="cuda", dtype=torch.int32)
        dstarts = new_token_starts(drafts)
        target = out[:starts[3]].flatten(1).float() @ m.head
        draft = m.normal(sum(drafts), VOCAB)
        for i, s in enumerate(s for s in range(3) for _ in range(drafts[s])):  # likely tokens, so that some are accepted
            tokens[i] = int(target[i + s].argmax())
            draft[i] += 0.7 * target[i + s]
        temps, u, v = [0.0 if step == 4 else 0.6, 0.9, 1.2], torch.rand(sum(drafts), generator=m.g, device="cuda"), torch.rand(
            3, generator=m.g, device="cuda")
        got = (torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty((3, MOST + 1), dtype=torch.int32, device="cuda"),
               torch.full((sum(drafts),), 7.0, device="cuda"))
        m.verify(target, draft, tokens, i32(dstarts), torch.tensor(temps, device="cuda"), u, v, *got)
        accepted, answer, probs = verify_reference(target, draft, tokens, dstarts, torch.tensor(temps).tolist(), u, v, MOST)
        assert got[0].tolist() == accepted.tolist() and got[1].tolist() == answer.tolist()
        assert (np.abs(got[2].cpu().double().numpy() - probs) <= 2.0 ** -24 * probs + 2.0 ** -60).all()
        # a chain of drafts is a tree of one branch
        rows3 = starts[3]
        masks = torch.tensor([(1 << (i + 1)) - 1 for s in range(3) for i in range(new[s])], device="cuda")
        tree = N.tree_attention(q[:rows3], m.kc, m.vc, m.table[:3], i32(context[:3]), i32(starts[:4]), masks, MOST + 1,
                                WIDTH * BS, D ** -0.5)
        assert ((tree.cpu().double() - want[:rows3]).abs() <= tol[:rows3]).all()
        for s in range(3):
            lens[s] += 1 + int(accepted[s])  # the next token is written with the next step


def test_a_captured_step(gpu):
    """Heads, attention, logits and verification in one graph, replayed over steps whose lengths follow from what was
    accepted, on the GPU; an eager run of the same steps gives the same."""
    S, n = 4, 4  # a token and 3 drafts a sequence
    rows = S * n
    runs = []
    for captured in (False, True):
        m = Model(71)
        m.kc.normal_(generator=m.g), m.vc.normal_(generator=m.g)
        lens = i32([30, 1, 100, 47])
        starts, dstarts = i32(range(0, rows + 1, n)), i32(range(0, S * 3 + 1, 3))
        x, draft = m.normal(rows, (H + 2 * KV) * D), m.normal(S * 3, VOCAB)
        tokens = torch.zeros(S * 3, dtype=torch.int32, device="cuda")
        u, v, temps = torch.zeros(S * 3, device="cuda"), torch.zeros(S, device="cuda"), torch.full((S,), 0.7, device="cuda")
        q, out = (torch.zeros((rows, H, D), dtype=torch.float16, device="cuda") for _ in range(2))
        accepted, answer = (torch.zeros(z, dtype=torch.int32, device="cuda") for z in (S, (S, MOST + 1)))
        probs = torch.zeros(S * 3, device="cuda")
        inner = (torch.arange(rows, device="cuda") % n != n - 1).nonzero()[:, 0]  # rows that a draft follows

        def step():
            at = (lens[:, None] + torch.arange(n, device="cuda", dtype=torch.int32)).long()
            slots = (m.table.gather(1, at // BS).long() * BS + at % BS).flatten()
            flat = at.flatten().int()
            positions = torch.stack([flat, flat // 2, flat * 3])
            m.attend(x, positions, slots, m.table, lens + n, starts, q, out)
            target = out.flatten(1).float() @ m.head
            tokens.copy_(target[inner].argmax(1))
            m.verify(target, draft + target[inner], tokens, dstarts, temps, u, v, accepted, answer, probs)
            lens.add_(accepted + 1)

        kept = [t.clone() for t in (m.kc, m.vc, lens)]
        step()  # (what the library sets up at first use comes before the capture)
        torch.cuda.synchronize()
        for a, b in zip((m.kc, m.vc, lens), kept):
            a.copy_(b)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        log, g = [], torch.Generator(device="cuda").manual_seed(72)
        for _ in range(6):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            u.copy_(torch.rand(u.shape, generator=g, device="cuda")), v.copy_(torch.rand(v.shape, generator=g, device="cuda"))
            torch.cuda.synchronize()
            graph.replay() if captured else step()
            torch.cuda.synchronize()
            log += [t.clone() for t in (q, out, accepted, answer, probs, lens)]
        runs.append(log)
    assert len({int(t.sum()) for t in runs[0][2::6]}) > 1  # not all accepted nor all refused
    assert all(torch.equal(a, b) for a, b in zip(*runs))
