"""GPU: verification of drafted tokens (tlh_draft_verify) against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from step_refs import new_token_starts, verify_reference
from tensorlisp_amd import native as N

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def i32(a):
    return torch.tensor(np.asarray(a, np.int32), device="cuda")


def build(drafts, vocab, dtype, seed, drafter=True, temps=None, near=0.7, masked=0.0):
    """Logits of a model and of a smaller one near it; drafted tokens mostly among the likely ones."""
    g, r = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    S, starts = len(drafts), new_token_starts(drafts)
    rows = starts[-1]
    x = torch.randn((rows + S, vocab), generator=g) * 2.5
    likely = torch.randint(0, vocab, (rows + S, min(6, vocab)), generator=g)
    x.scatter_(1, likely, 6 + 3 * torch.randn(likely.shape, generator=g))
    row = [starts[s] + s + i for s in range(S) for i in range(drafts[s])]
    y = x[row] + near * torch.randn((rows, vocab), generator=g)
    if masked:
        off = torch.rand(x.shape, generator=g) < masked
        off.scatter_(1, likely[:, :1], False)
        x = x.masked_fill(off, -INF)
        y = y.masked_fill(off[row], -INF)
    tokens = [int(r.choice(likely[i].numpy())) if r.random() < 0.8 else int(r.integers(0, vocab)) for i in row]
    temps = list(r.uniform(0.5, 1.4, S)) if temps is None else temps
    return dict(target=x.to(dtype).cuda(), draft=y.to(dtype).cuda() if drafter else None, tokens=tokens, starts=starts,
                temps=np.asarray(temps, np.float32), accept_at=r.random(rows, dtype=np.float32),
                sample_at=r.random(S, dtype=np.float32), most=max(max(drafts), 1) if drafts else 1)


def on_gpu(c):
    f = lambda a: torch.tensor(np.asarray(a, np.float32), device="cuda")  # noqa: E731
    return (c["target"], c["draft"], i32(c["tokens"]), i32(c["starts"]), f(c["temps"]), f(c["accept_at"]), f(c["sample_at"]))


def outputs(c):
    S = len(c["temps"])
    return (torch.full((S,), 77, dtype=torch.int32, device="cuda"),
            torch.full((S, c["most"] + 1), 77, dtype=torch.int32, device="cuda"),
            torch.full((len(c["tokens"]),), 7.0, device="cuda"))


def node_of(c):
    return N.DraftVerify(len(c["temps"]), len(c["tokens"]), c["most"], c["target"].shape[1], c["target"].dtype,
                         c["draft"] is not None)


def check(c, node=None, outs=None, **kw):
    outs = outputs(c) if outs is None else outs
    (node or node_of(c))(*on_gpu(c), *outs, **kw)
    torch.cuda.synchronize()
    accepted, out, probs = verify_reference(c["target"], c["draft"], c["tokens"], c["starts"], c["temps"], c["accept_at"],
                                            c["sample_at"], c["most"])
    assert outs[0].tolist() == accepted.tolist()
    assert outs[1].tolist() == out.tolist()
    got = outs[2].cpu().double().numpy()
    assert (np.isnan(got) == np.isnan(probs)).all()
    ok = ~np.isnan(probs)
    assert (np.abs(got[ok] - probs[ok]) <= 2.0 ** -24 * probs[ok] + 2.0 ** -140 + 1e-11 * probs[ok]).all()
    return outs


CASES = [
    # drafts, vocabulary, type, a drafting model
    ([4], 128256, torch.float32, True), ([1, 8, 3, 5, 2, 7, 4, 6], 32000, torch.float32, True),
    ([1, 8, 3, 5, 0, 7], 32003, torch.bfloat16, False), ([10] * 12, 5001, torch.float16, True), ([3, 2], 1, torch.float32, True),
    ([2, 2], 2, torch.float32, False), ([5], 63, torch.float16, True), ([40], 999, torch.float32, True),
    ([0, 0, 0], 4097, torch.float32, True), ([0], 128256, torch.bfloat16, False), ([1] * 100, 777, torch.bfloat16, True),
    ([2, 9], 262144, torch.float32, True), ([3], 1000000, torch.bfloat16, True), ([6, 1], 16385, torch.float32, False),
    ([100, 1, 70], 300, torch.float32, True),
]


@pytest.mark.parametrize("drafts,vocab,dtype,drafter", CASES)
def test_against_64_bits(gpu, drafts, vocab, dtype, drafter):
    for seed in range(3):
        check(build(drafts, vocab, dtype, 100 * seed + len(drafts) + vocab % 97, drafter))


@pytest.mark.parametrize("drafter", [True, False])
def test_all_accepted_and_none(gpu, drafter):
    """accept_at 0 accepts what has any probability; a drafted token the model gives none is always refused."""
    c = build([5, 3, 7], 5000, torch.float32, 11, drafter)
    c["accept_at"][:] = 0
    assert check(c)[0].tolist() == [5, 3, 7]
    for i, x in enumerate(c["tokens"]):
        c["target"][[0, 1, 2, 3, 4, 6, 7, 8, 10, 11, 12, 13, 14, 15, 16][i], x] = -INF
    assert check(c)[0].tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_greedy(gpu, dtype):
    """Temperatures that are not above 0: the likeliest token, the lowest index among equal ones; the drafter is not
    looked at."""
    c = build([4, 4, 4, 4, 4], 20000, dtype, 12, temps=[0.0, -1.0, NAN, 0.9, -0.0])
    t = c["target"]
    for s in (0, 1, 2, 4):
        for i in range(4 if s else 2):  # sequence 0 stops at its draft 2
            c["tokens"][4 * s + i] = int(t[5 * s + i].argmax())
    t[21, 50], t[21, 700], c["tokens"][17] = 100.0, 100.0, 50   # equal ones: the first
    t[22, 50], t[22, 700], c["tokens"][18] = 100.0, 100.0, 700  # not the second
    c["draft"][16:] = NAN
    got = check(c)
    assert got[0].tolist()[:3] == [2, 4, 4] and got[0].tolist()[4] == 2
    t[20, 9], c["tokens"][16] = INF, 9  # greedy takes an infinity
    check(c)


@pytest.mark.parametrize("masked", [0.5, 0.999])
def test_masked_vocabularies(gpu, masked):
    for dtype in (torch.float32, torch.float16):
        check(build([3, 5, 1], 32000, dtype, 13, masked=masked))
        check(build([3, 5, 1], 32000, dtype, 14, drafter=False, masked=masked))


@pytest.mark.parametrize("bad", [NAN, INF])
def test_rows_that_are_no_distribution(gpu, bad):
    """In the model's or the drafter's row, before, at and behind where a sequence stops; -inf throughout."""
    for fill in ("one", "all"):
        for where in ("target", "draft"):
            for row in range(4 if where == "target" else 3):
                c = build([3], 3001, torch.float32, 15)
                c["accept_at"][:] = 0.0
                if fill == "one":
                    c[where][row, 1234] = bad
                else:
                    c[where][row] = -INF
                got = check(c)
                assert got[0].item() == row and got[1][0, row].item() == -1


def test_equal_distributions_and_nothing_left(gpu):
    """Drafter and model agree: everything is accepted (u < 1). Where the model gives the token nothing and the rest is
    equal, there is nothing above the drafter and the token is drawn from the model's."""
    c = build([6, 6], 4000, torch.float32, 16, near=0.0)
    assert check(c)[0].tolist() == [6, 6]
    c = build([1], 4000, torch.float32, 17, near=0.0)
    c["target"][0, c["tokens"][0]] = -INF
    c["draft"][0, c["tokens"][0]] = -INF
    got = check(c)
    assert got[0].item() == 0 and got[2].item() == 0.0


def test_tokens_outside_the_vocabulary(gpu):
    for drafter in (True, False):
        for x in (-1, 4000, 2 ** 31 - 1, -2 ** 31):
            c = build([3, 2], 4000, torch.float32, 18, drafter)
            c["accept_at"][:] = 0.0
            c["tokens"][1] = x
            got = check(c)
            assert got[0].tolist() == [1, 2] and got[2][1].item() == 0.0


def test_random_numbers_at_the_ends(gpu):
    """0 takes the first token with a weight, the largest below 1 the last ones; NaN and 1 the last with a weight."""
    for u in (0.0, 1 - 2.0 ** -24, 1.0, NAN, -1.0):
        for drafter in (True, False):
            c = build([2, 2, 0], 3000, torch.float32, 19, drafter, masked=0.3)
            c["sample_at"][:] = u
            check(c)


def test_extreme_logits_and_temperatures(gpu):
    c = build([3, 3, 3, 3], 3000, torch.float32, 20, temps=[1e-30, 1e30, 1e-3, INF])
    check(c)
    c = build([3, 3], 3000, torch.float32, 21)
    c["target"] *= 1e30
    c["draft"] *= 1e30
    check(c)
    c["target"][0, 7], c["target"][0, 9] = 3e38, -3e38
    check(c)
    c = build([4], 50000, torch.float32, 22)
    c["target"][:] = 0.25  # all equal: running sums of 1 / 50000
    c["draft"][:] = -3.0
    check(c)


def test_more_drafts_than_looked_at(gpu):
    c = build([7, 2, 9], 3000, torch.float32, 23)
    c["most"] = 4
    c["accept_at"][:] = 0.0
    c["tokens"] = [int(x) for x in c["target"].argmax(1).cpu()[[0, 1, 2, 3, 4, 5, 6, 8, 9] + list(range(11, 20))]]
    got = check(c)
    assert got[0].tolist() == [4, 2, 4]
    c["most"] = 0
    check(c)


@pytest.mark.parametrize("starts", [[0, 0, 5], [2, 3, 5], [4, 4, 4], [-5, 3, 100], [5, 2, 4]])
def test_starts_that_leave_drafts_out(gpu, starts):
    """Gaps, empty sequences, starts outside the drafts (taken as the nearer end), an end before its start (empty)."""
    c = build([3, 2], 900, torch.float32, 24)
    clamped = [max(0, min(x, 5)) for x in starts]
    outs = outputs({**c, "most": 5})
    N.DraftVerify(2, 5, 5, 900)(*on_gpu({**c, "starts": starts}), *outs)
    for s in range(2):  # each sequence as one of its own
        a = clamped[s]
        n = max(0, clamped[s + 1] - a)
        probs = verify_reference(c["target"][a + s:a + s + n + 1], c["draft"][a:a + n], c["tokens"][a:a + n], [0, n],
                                 c["temps"][s:s + 1], c["accept_at"][a:a + n], c["sample_at"][s:s + 1], 5)
        assert outs[0][s].item() == probs[0][0] and outs[1][s].tolist() == probs[1][0].tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_at_any_stride_and_alignment(gpu, dtype):
    c = build([3, 4], 2999, dtype, 25)
    want = check(c)
    for pad, first in ((1, 1), (9, 3), (5, 7)):
        views = {}
        for x in ("target", "draft"):
            wide = torch.full((len(c[x]), 2999 + first + pad), NAN, dtype=dtype, device="cuda")
            wide[:, first:first + 2999] = c[x]
            views[x] = wide[:, first:first + 2999]
        got = check({**c, **views})
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_probabilities_are_not_asked_for(gpu):
    c = build([3, 4], 2999, torch.float32, 26)
    want, got = check(c), outputs(c)
    node_of(c)(*on_gpu(c), got[0], got[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_answer_is_distributed_as_the_model_alone(gpu):
    """20000 sequences of one draft over 40 tokens: the first token answered follows p, whatever the drafter says. Each
    count of 20000 p lies within 6 standard deviations of it (a chance of 40 * 2e-9 of failing)."""
    n, V = 20000, 40
    g = torch.Generator().manual_seed(27)
    p, q = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g) * 1.5
    target, draft = p.expand(2 * n, V).contiguous().cuda(), q.expand(n, V).contiguous().cuda()
    tokens = torch.multinomial(torch.softmax(q.double(), 0), n, True, generator=g).int().cuda()
    u, w = torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    accepted, out, _ = N.draft_verify(target, draft, tokens, i32(range(n + 1)), torch.ones(n, device="cuda"), u, w, 1)
    want = torch.softmax(p.double(), 0) * n
    got = torch.bincount(out[:, 0].cpu().long(), minlength=V).double()
    assert ((got - want).abs() <= 6 * torch.sqrt(want)).all()
    assert 0 < int(accepted.sum()) < n


def test_a_used_scratch_smaller_calls_streams_and_graphs(gpu):
    big = build([8] * 20, 32000, torch.float32, 28)
    node = node_of(big)
    want = check(big, node)
    node.scratch.fill_(0xff)
    assert all(torch.equal(a, b) for a, b in zip(check(big, node), want))
    for drafts in ([8, 3], [1], [0, 0, 5]):
        c = {**build(drafts, 32000, torch.float32, 29), "most": 8}
        check(c, node)
    c = {**build([5, 3, 8], 32000, torch.float32, 30), "most": 8}
    want = check(c, node)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream, 0):
        got = check(c, node, stream=stream)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    dev, outs = on_gpu(c), outputs(c)
    node(*dev, *outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        node(*dev, *outs)
    for i in range(4):
        dev[0].copy_(dev[0].roll(1, 0))
        dev[5].copy_(torch.rand(16, device="cuda")), dev[6].copy_(torch.rand(3, device="cuda"))
        for t in outs:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        other = outputs(c)
        node(*dev, *other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, other))


@pytest.mark.parametrize("vocab", [128256, 131064, 131065])
def test_one_node_for_few_and_many_sequences(gpu, vocab):
    """What is drawn from is summed in chunks whose length follows from the sequences of a call (16 of these
    vocabularies, and 131064 tokens, are the bounds); the node's scratch has room for each."""
    c = build([2] * 20, vocab, torch.bfloat16, 40)
    node = node_of(c)
    for n in (20, 17, 16, 15, 1):
        check({**c, "target": c["target"][:3 * n], "draft": c["draft"][:2 * n], "tokens": c["tokens"][:2 * n],
               "starts": c["starts"][:n + 1], "temps": c["temps"][:n], "accept_at": c["accept_at"][:2 * n],
               "sample_at": c["sample_at"][:n]}, node)


def test_one_call_form(gpu):
    c = build([5, 3, 8], 32000, torch.bfloat16, 31)
    want = check(c)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, s, s.cuda_stream, 0):
        got = N.draft_verify(*on_gpu(c), 8, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def each_alone(c, starts, most):
    """Every sequence as one of its own, its drafts from its start up to its end (none if that is before it); one that
    shares a draft with another is not verified."""
    R, S = len(c["tokens"]), len(starts) - 1
    lo = [max(0, min(x, R)) for x in starts]
    span = [(lo[s], min(max(lo[s], lo[s + 1]), lo[s] + most)) for s in range(S)]
    probs, accepted, out = np.full(R, 7.0), [], []
    for s, (a, b) in enumerate(span):
        if any(t != s and max(a, x) < min(b, y) for t, (x, y) in enumerate(span)):
            probs[a:b] = np.nan
            accepted.append(0), out.append([-1] * (most + 1))
            continue
        draft = None if c["draft"] is None else c["draft"][a:b]
        one = verify_reference(c["target"][a + s:b + s + 1], draft, c["tokens"][a:b], [0, b - a], c["temps"][s:s + 1],
                               c["accept_at"][a:b], c["sample_at"][s:s + 1], most)
        accepted.append(one[0][0]), out.append(one[1][0].tolist())
        probs[a:b] = one[2]
    return accepted, out, probs


def check_alone(c, starts, most, node):
    node.scratch.fill_(0xff)
    outs = outputs({**c, "most": most})
    node(*on_gpu({**c, "starts": starts}), *outs)
    torch.cuda.synchronize()
    accepted, out, probs = each_alone(c, starts, most)
    assert outs[0].tolist() == accepted
    assert outs[1].tolist() == out
    got, ok = outs[2].cpu().double().numpy(), ~np.isnan(probs)
    assert (np.isnan(got) == ~ok).all()
    assert (np.abs(got[ok] - probs[ok]) <= 2.0 ** -24 * probs[ok] + 1e-11 * probs[ok]).all()


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("starts", [[5, 2, 4], [4, 1, 3], [0, 5, 0], [5, 0, 5], [0, 3, 1, 2], [0, 3, 1, 4, 5], [3, 5, 0, 3, 3],
                                    [0, 0, 5, 5, 0], [2, 9, -4, 1], [0, 2, 5]])
def test_starts_that_decrease(gpu, starts, drafter):
    """Sequences in any order, of either kind beside each other, over a scratch that holds another call's rows or none."""
    S = len(starts) - 1
    for most in (5, 2):
        for seed, temps in enumerate(([0.0, 0.7, 0.0, 0.9], [0.7, 0.0, 1.1, 0.0], [0.4, 1.3, 0.8, 0.6])):
            c = build([3, 2] + [0] * (S - 2), 9001, torch.float32, 50 + seed, drafter, temps=temps[:S])
            node = N.DraftVerify(S, 5, most, 9001, drafter=drafter)
            check_alone(c, starts, most, node)
            if starts == sorted(starts):
                assert not np.isnan(each_alone(c, starts, most)[2]).any()


@pytest.mark.parametrize("at,to", [(0, 5), (70, 0), (699, 2), (1399, 1000), (1400, 3)])
def test_one_start_that_decreases_among_many(gpu, at, to):
    r = np.random.default_rng(60)
    c = build([int(x) for x in r.integers(0, 3, 1400)], 300, torch.float32, 61, temps=r.choice([0.0, 0.8, 1.2], 1400))
    node = N.DraftVerify(1400, len(c["tokens"]), 2, 300)
    starts = list(c["starts"])
    starts[at] = to
    check_alone(c, starts, 2, node)
    c["most"] = 2
    check(c, node)  # and the next call is as ever


def test_a_token_without_a_weight_is_never_drawn(gpu):
    """The random number falls between two tokens of different chunks, with masked ones between them: what was summed
    before a chunk comes out of a difference, which may be above it by a rounding."""
    S, V = 512, 3 * 4096
    g = torch.Generator().manual_seed(62)
    x = torch.full((S, V), -INF)
    w = torch.randn((S, 4), generator=g)
    x[:, 100:104] = w                                # the first chunk weighs half of all
    x[:, 4096 + 2000] = w[:, 0]                      # the second begins with masked tokens
    x[:, 2 * 4096 + 900:2 * 4096 + 903] = w[:, 1:]
    f = lambda v: torch.full((S,), v, device="cuda")  # noqa: E731
    none = torch.empty((0,), dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        accepted, out, _ = N.draft_verify(x.to(dtype).cuda(), None, none, i32([0] * (S + 1)), f(0.7), f(0.5)[:0], f(0.5), 0)
        assert (accepted == 0).all()
        drawn = out[:, 0].cpu().long()
        assert ((drawn >= 0) & (drawn < V)).all()
        assert (x.gather(1, drawn[:, None]) > -INF).all()
