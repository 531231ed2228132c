"""draft_verify on the GPU against its definition, one sequence and one token at a time."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
BIG = 3.4028234663852886e38


def _weights(p, q=None, without=None):
    """One row's weights as Python numbers (f64)."""
    w = p.double() - q.double() if q is not None else p.double().clone()
    w = torch.where(w > 0, w.clamp(max=BIG), torch.zeros_like(w))
    if without is not None:
        w[without] = 0
    return w


def _draw(w, pick):
    up = torch.cumsum(w, 0)
    share = pick * float(up[-1])
    for j in range(len(w)):
        if float(w[j]) > 0 and float(up[j]) > share:
            return j
    return int(torch.nonzero(w)[-1])


def reference(p, draft, cu, accept, pick, q, max_drafts):
    """tokens, counts of host tensors."""
    b, vocab = len(cu) - 1, p.shape[1]
    tokens, counts = torch.full((b, max_drafts + 1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int32)
    for s in range(b):
        rows = list(range(int(cu[s]), int(cu[s + 1])))
        for i, r in enumerate(rows):
            x, w = int(draft[r]), None
            if i + 1 < len(rows):
                fine = 0 <= x < vocab
                if fine and float(accept[r]) * (float(q[r, x]) if q is not None else 1.0) < float(p[r, x]):
                    tokens[s, i] = x
                    continue
                w = _weights(p[r], q[r] if q is not None else None, x if q is None and fine else None)
            if w is None or float(w.sum()) == 0:
                w = _weights(p[r])
            tokens[s, i] = _draw(w, float(pick[s])) if float(w.sum()) > 0 else 0
            counts[s] = i + 1
            break
    return tokens, counts


def _case(seqs, drafts, vocab, dtype, model, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    count = torch.randint(0, drafts + 1, (seqs,), generator=g)
    count[0] = drafts
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), (count + 1).cumsum(0)]).to(torch.int32)
    t = int(cu[-1])
    logits = spread * torch.randn(t, vocab, generator=g)
    p = torch.softmax(logits, 1).to(dtype)
    q = torch.softmax(logits + 0.3 * torch.randn(t, vocab, generator=g), 1).to(dtype)
    draft = torch.multinomial(q.float(), 1, generator=g)[:, 0]
    return dict(p=p, draft=draft, cu=cu, accept=torch.rand(t, generator=g), pick=torch.rand(seqs, generator=g), q=q if model else None), drafts


def _run(c, max_drafts, **more):
    import bigsmall_amd as bs
    return bs.draft_verify(**{k: v.cuda() if v is not None else None for k, v in c.items()}, max_drafts=max_drafts, **more)


def _same(got, want):
    assert torch.equal(got[1].cpu(), want[1]), (got[1], want[1])
    assert torch.equal(got[0].cpu(), want[0]), torch.nonzero(got[0].cpu() != want[0])


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,drafts,vocab", [(1, 0, 10), (1, 5, 1), (3, 1, 2), (5, 4, 255), (2, 3, 4097), (40, 6, 1000), (1, 70, 300), (3, 5, 50257)])
def test_against_the_definition(seqs, drafts, vocab, dtype, model):
    c, d = _case(seqs, drafts, vocab, dtype, model, seqs * 100 + drafts)
    _same(_run(c, d), reference(**c, max_drafts=d))


def test_many_sequences_and_a_large_vocabulary():
    c, d = _case(700, 2, 300, torch.float32, True, 5)
    _same(_run(c, d), reference(**c, max_drafts=d))
    for seqs, vocab, dtype in ((2, 200001, torch.float32), (1, 262145, torch.float32), (1, 700004, torch.bfloat16)):
        c, d = _case(seqs, 2, vocab, dtype, True, 6, spread=3.0)
        _same(_run(c, d), reference(**c, max_drafts=d))


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("vocab", [4, 256, 1023, 1024, 1025, 8192, 8193, 9216, 20000])
def test_borders_of_pieces(vocab, model):
    c, d = _case(5, 3, vocab, TYPES[vocab % 3], model, vocab, spread=0.3)
    _same(_run(c, d), reference(**c, max_drafts=d))
    for pick in (0.0, 1 - 2.0 ** -24):
        t = dict(c, pick=torch.full((5,), pick))
        _same(_run(t, d), reference(**t, max_drafts=d))


@pytest.mark.parametrize("seqs,vocab", [(3, 32767), (3, 32768), (4, 32769), (3, 33793), (5, 33794), (4, 33795), (255, 32801), (256, 32801), (300, 34000), (258, 1030)])
def test_one_launch_or_two(seqs, vocab):
    """Sizes on both sides of where one workgroup takes a sequence by itself; rows that start anywhere; alone as beside others."""
    import bigsmall_amd as bs
    dtype = TYPES[seqs % 3]
    c, d = _case(seqs, 1, vocab, dtype, True, seqs + vocab, spread=1.0)
    got = _run(c, d)
    _same(got, reference(**c, max_drafts=d))
    off = {k: torch.empty(c[k].numel() + 3, dtype=dtype, device="cuda")[i:].narrow(0, 0, c[k].numel()).view(c[k].shape) for k, i in (("p", 1), ("q", 3))}
    for k in off:
        off[k].copy_(c[k])
    rest = {k: v.cuda() for k, v in c.items() if k not in "pq"}
    _same(bs.draft_verify(p=off["p"], q=off["q"], max_drafts=d, **rest), [x.cpu() for x in got])
    lo, hi = int(c["cu"][1]), int(c["cu"][2])
    one = dict({k: v[lo:hi] for k, v in c.items() if k not in ("cu", "pick")}, cu=torch.tensor([0, hi - lo], dtype=torch.int32), pick=c["pick"][1:2])
    tokens, counts = _run(one, d)
    assert torch.equal(tokens[0], got[0][1]) and int(counts[0]) == int(got[1][1])


def test_picks_at_both_ends_and_between_equal_weights():
    """Dyadic weights: all sums are exact, so borders are hit exactly; a border belongs to the token after it."""
    vocab = 9000
    p = torch.zeros(12, vocab)
    p[:, 100:8292:1024] = 0.125                     # eight tokens
    pick = torch.tensor([i / 8 for i in range(8)] + [0.1249, 0.999999, 1.0, 0.5 - 2.0 ** -20])
    c = dict(p=p, draft=torch.zeros(12, dtype=torch.int64), cu=torch.arange(13, dtype=torch.int32), accept=torch.zeros(12), pick=pick, q=None)
    got = _run(c, 0)
    want = [100 + 1024 * i for i in range(8)] + [100, 100 + 7 * 1024, 100 + 7 * 1024, 100 + 3 * 1024]
    assert got[0][:, 0].tolist() == want and got[1].tolist() == [1] * 12
    _same(got, reference(**c, max_drafts=0))


def test_acceptance_is_strict_and_exact():
    p = torch.tensor([[0.5, 0.25, 0.25]] * 8)
    q = torch.tensor([[0.5, 0.5, 0.0], [0.5, 0.5, 0.0], [0.25, 0.5, 0.25], [1.0, 0.0, 0.0]] * 2)
    draft = torch.tensor([0, 0, 1, 0, 1, 0, 2, 0])
    accept = torch.tensor([1 - 2.0 ** -24, 0.0, 0.5, 0.0, 0.49999997, 0.0, 0.99999994, 0.0])
    c = dict(p=p, draft=draft, cu=torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32), accept=accept, pick=torch.tensor([0.0, 0.0, 0.9, 0.9]), q=q)
    tokens, counts = _run(c, 1)
    # u q < p: taken; 0.5 * 0.5 = 0.25 is not below 0.25; just below it is; p = q is always taken
    assert counts.tolist() == [2, 1, 2, 2]
    _same((tokens, counts), reference(**c, max_drafts=1))


def test_rows_that_leave_nothing_or_hold_no_numbers():
    from bigsmall_amd.device import StatusWord
    v = 5000
    p = torch.full((7, v), 1.0 / v)
    q = p.clone()
    p[1] = 0                                       # a refused draft, nothing in p
    p[2], q[2] = 0, 0.5                            # p - q nowhere positive
    p[2, 7] = 0.25
    p[3] = math.nan
    p[4, 11] = math.inf
    p[5] = -1.0
    p[6, :] = math.nan
    p[6, 4000] = 1e-30
    cu = torch.tensor([0, 1, 3, 4, 5, 6, 7], dtype=torch.int32)
    draft = torch.tensor([0, 3, 0, 0, 0, 0, 0])
    c = dict(p=p, draft=draft, cu=cu, accept=torch.full((7,), 0.5), pick=torch.full((6,), 0.75), q=q)
    status = StatusWord("cuda")
    tokens, counts = _run(c, 1, status=status)
    assert int(status.t) == 2                      # BS_DEV_ERR_COUNT: sequences without any probability
    _same((tokens, counts), reference(**c, max_drafts=1))
    assert tokens[:, 0].tolist() == [3750, 0, 0, 11, 0, 4000] and counts.tolist() == [1] * 6
    # p - q nowhere positive at a refused draft: from p
    c = dict(p=p[2:4], draft=torch.tensor([9, 0]), cu=torch.tensor([0, 2], dtype=torch.int32), accept=torch.tensor([0.9, 0.0]),
             pick=torch.tensor([0.3]), q=q[2:4])
    tokens, counts = _run(c, 1)
    assert tokens.tolist() == [[7, -1]] and counts.tolist() == [1]


def test_rows_and_drafts_that_do_not_exist():
    from bigsmall_amd.device import StatusWord
    c, d = _case(4, 3, 600, torch.float32, True, 9)
    full = _run(c, d)
    for cu, bad in ((torch.tensor([0, 4, 4, 9, 12]), True), (torch.tensor([0, 4, 4, 8, 12]), False), (torch.tensor([0, 4, 3, 9, 12]), True), (torch.tensor([0, 4, 7, 9, 1000]), True),
                    (torch.tensor([-3, 1, 2, 3, 4]), True), (torch.tensor([0, 5, 6, 7, 8]), True)):
        t = dict(c, cu=cu.to(torch.int32))
        t = {k: v if k in ("cu", "pick") or v is None else v.repeat(2, *[1] * (v.dim() - 1))[:12] for k, v in t.items()}
        status = StatusWord("cuda")
        tokens, counts = _run(t, d, status=status)
        assert bool(int(status.t)) == bad, cu
        n = cu[1:] - cu[:-1]
        for s in range(4):
            ok = 0 <= cu[s] <= cu[s + 1] <= 12 and n[s] <= d + 1
            if not ok or n[s] == 0:
                assert int(counts[s]) == 0 and tokens[s].tolist() == [-1] * (d + 1)
            else:
                lone = dict(t, cu=cu[s:s + 2].to(torch.int32), pick=t["pick"][s:s + 1])
                want = reference(**lone, max_drafts=d)
                assert torch.equal(tokens[s].cpu(), want[0][0])
    draft = c["draft"].clone()
    draft[0], draft[int(c["cu"][1])] = 600, -1
    t = dict(c, draft=draft)
    status = StatusWord("cuda")
    got = _run(t, d, status=status)
    assert int(status.t) == 4
    _same(got, reference(**t, max_drafts=d))
    for q in (None,):
        t = dict(t, q=q)
        _same(_run(t, d), reference(**t, max_drafts=d))
    assert full[0].shape == (4, d + 1)


def test_strides_graph_and_neighbours():
    import bigsmall_amd as bs
    c, d = _case(6, 4, 3000, torch.bfloat16, True, 3)
    want = reference(**c, max_drafts=d)
    wide = {k: torch.zeros(c[k].shape[0], 3007, dtype=torch.bfloat16, device="cuda") for k in "pq"}
    for k in "pq":
        wide[k][:, 5:3005] = c[k].cuda()
    rest = {k: v.cuda() for k, v in c.items() if k not in "pq"}
    _same(bs.draft_verify(p=wide["p"][:, 5:3005], q=wide["q"][:, 5:3005], max_drafts=d, **rest), want)
    _same(bs.draft_verify(p=c["p"].T.contiguous().cuda().T, q=wide["q"][:, 5:3005], max_drafts=d, **rest), want)
    tokens, counts = bs.draft_verify(c["p"].cuda(), q=c["q"].cuda(), **rest)               # room for all by default
    assert tokens.shape[1] == len(c["draft"]) - 6 + 1 and torch.equal(tokens[:, :d + 1].cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    # alone or beside others
    s = 2
    lo, hi = int(c["cu"][s]), int(c["cu"][s + 1])
    lone = dict({k: v[lo:hi] for k, v in c.items() if k not in ("cu", "pick")}, cu=torch.tensor([0, hi - lo], dtype=torch.int32), pick=c["pick"][s:s + 1])
    assert torch.equal(_run(lone, d)[0][0].cpu(), want[0][s])
    # captured: every replay as the eager call
    static = {k: v.cuda() for k, v in c.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bs.draft_verify(**static, max_drafts=d)
    for seed in (3, 4, 5):
        pick = torch.rand(6, generator=torch.Generator().manual_seed(seed))
        static["pick"].copy_(pick)
        graph.replay()
        _same(out, reference(**dict(c, pick=pick), max_drafts=d))
        _same(_run(dict(c, pick=pick), d), reference(**dict(c, pick=pick), max_drafts=d))
        torch.cuda.synchronize()


def test_tokens_follow_the_target():
    """Drafted from q and verified, tokens are distributed as p: 40,000 sequences, each frequency within five standard
    deviations."""
    import bigsmall_amd as bs
    n, v = 40000, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    p = torch.tensor([0.3, 0.2, 0.15, 0.12, 0.1, 0.08, 0.05, 0.0], device="cuda")
    q = torch.tensor([0.05, 0.3, 0.1, 0.05, 0.2, 0.1, 0.1, 0.1], device="cuda")
    draft = torch.multinomial(q, 2 * n, replacement=True, generator=g)
    tokens, _ = bs.draft_verify(p.expand(2 * n, v), draft, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                                torch.rand(2 * n, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"),
                                q=q.expand(2 * n, v), max_drafts=1)
    share = torch.bincount(tokens[:, 0], minlength=v).double().cpu() / n
    want = p.double().cpu()
    assert bool(((share - want).abs() <= 5 * (want * (1 - want) / n).sqrt() + 1e-12).all()), share
