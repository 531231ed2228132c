"""PagedLlama.generate with drafts and drawn tokens: what it refuses, what it takes of the cache, and that drafts are kept."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_paged_llama import model  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def loaded(model):  # noqa: F811
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        yield lambda pages, sequences, **more: PagedLlama(loader, config, pages=pages, sequences=sequences, **more)


def _same_again(tokens, lengths, n):
    """Drafts: the last token again."""
    b = tokens.shape[0]
    return tokens[torch.arange(b, device="cuda"), lengths.long() - 1][:, None].expand(b, n), None


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 2])
@pytest.mark.parametrize("draft", [None, _same_again])
def test_rows_without_any_probability_are_an_error(loaded, draft, at, value):
    """Logits of the prompt or of a later step that hold a NaN or an infinity: no token is made up from them."""
    m = loaded(pages=8, sequences=2)
    calls, plain = [], m._logits

    def logits(x):
        y = plain(x)
        if len(calls) == at:
            y[-1 if at == 0 else 0, 7] = value           # (a step's first row is its first sequence's first)
        calls.append(len(y))
        return y
    m._logits = logits
    prompts = [torch.arange(70) % 500, torch.arange(3)]
    with pytest.raises(RuntimeError, match="no probability"):
        m.generate(prompts, 10, temperature=0.7, draft=draft, generator=torch.Generator(device="cuda").manual_seed(1))
    assert len(calls) == at + 1 and m.cache.free_pages() == 8


class _Enough(Exception):
    pass


@pytest.mark.parametrize("drafts", [1025, 1 << 40])
def test_more_drafts_than_a_step_takes(loaded, drafts):
    """As many are asked for as one verification takes, and room is made for no more."""
    m = loaded(pages=24, sequences=1)
    asked = []

    def draft(tokens, lengths, n):
        asked.append((n, tokens.shape[1]))
        raise _Enough

    with pytest.raises(_Enough):
        m.generate([torch.arange(30)], 1200, draft=draft, drafts=drafts)
    assert asked[0][0] == 1024 and asked[0][1] <= 30 + 1200 + 63 + 1025
    asked.clear()
    with pytest.raises(_Enough):
        m.generate([torch.arange(30)], 8, draft=draft, drafts=drafts)
    assert asked[0][0] == 6           # of 8 tokens the prompt gave the first, and a step draws its last one itself


@pytest.mark.parametrize("lens,new,need", [((60, 3), 4, 0), ((60, 3), 5, 1), ((60, 124), 6, 3), ((128, 1, 63), 1, 2)])
def test_pages_that_the_sequences_do_not_need_stay_free(loaded, lens, new, need):
    """Other sequences of the cache go on while drafts are asked for; what is needed is enough, to the page."""
    prompts = [torch.arange(n) % 500 for n in lens]
    m = loaded(pages=max(1, need) + 2, sequences=len(lens) + 1)
    free = []

    def draft(tokens, lengths, n):
        free.append(m.cache.free_pages())
        if len(free) == 1:                           # a sequence of somebody else's
            m.forward({m.cache.add(): torch.arange(130)})
        return _same_again(tokens, lengths, n)

    out = m.generate(prompts, new, draft=draft)
    assert [len(o) for o in out] == [new] * len(lens)
    if new > 2:
        assert free[0] == 2 and m.cache.free_pages() == max(1, need)
    plain = m.generate(prompts, new)                 # (each of its tokens is the likeliest; so is each of those with drafts)
    assert [len(o) for o in plain] == [new] * len(lens)
    if need:
        short = loaded(pages=need, sequences=len(lens))
        taken = short.cache.step({short.cache.add(): 64}) if need > 1 else None
        if taken is not None:
            with pytest.raises(RuntimeError, match="free"):
                short.generate(prompts, new, draft=_same_again)
            assert short.cache.free_pages() == need - 1


# ---- drafts that are kept

def _rows_of_a_step(cached, left, n):
    """How many rows a step gives a sequence with `cached` tokens in the cache, one certain new one and drafts after it: none of
    these completes a page."""
    end = cached + min(1 + n, left)
    while end > cached + 1 and end // 64 * 64 > cached + 1:
        end -= 1
    return end - cached if left else 0


def _steps(lens, new, drafts):
    """Each step's n and rows of each sequence when every draft is taken."""
    made, steps = [1] * len(lens), []
    while min(made) < new:
        n = min(drafts, new - min(made) - 1)
        rows = [_rows_of_a_step(a + m - 1, new - m, n) for a, m in zip(lens, made)]
        steps.append((n, rows))
        made = [m + r for m, r in zip(made, rows)]
    return steps


class _Recorded:
    """draft_verify with its arguments and results kept, and the drafts' random numbers set to `accept`."""

    def __init__(self, monkeypatch, accept=None):
        from bigsmall_amd import paged_llama
        self.plain, self.accept, self.calls = paged_llama.draft_verify, accept, []
        monkeypatch.setattr(paged_llama, "draft_verify", self)

    def __call__(self, p, draft, cu, accept, pick, q=None, **more):
        if self.accept is not None:
            accept = torch.full_like(accept, self.accept)
        tokens, counts = self.plain(p, draft, cu, accept, pick, q=q, **more)
        self.calls.append({k: v.clone() if v is not None else None
                           for k, v in dict(p=p, draft=draft, cu=cu, q=q, tokens=tokens, counts=counts).items()})
        return tokens, counts


def _guess(lengths, n, vocab):
    """A guess that names its sequence and position, and probabilities that do: the guessed token has one that no other
    place has."""
    b = len(lengths)
    seq = torch.arange(b, device="cuda")[:, None]
    at = lengths.long()[:, None] + torch.arange(n, device="cuda")
    ids = (seq * 31 + at * 7 + 5) % vocab
    q = torch.zeros(b, n, vocab, device="cuda")
    return ids, q.scatter_(2, ids[:, :, None], (0.25 + (seq * 512 + at) * 2.0 ** -12)[:, :, None])


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("lens,new,drafts", [((60, 1, 127), 24, 4), ((63, 64), 90, 7), ((5,), 9, 16)])
def test_drafts_that_are_taken_are_kept(loaded, monkeypatch, lens, new, drafts, with_q):
    """Random numbers of 0 take every draft whose probability is not 0 (at this temperature none is): the text is then the drafts
    with the drawn tokens between them, in as few steps as pages allow, and each verification has its own row of everything."""
    m = loaded(pages=20, sequences=3)
    prompts = [torch.arange(n) % 500 for n in lens]
    record, asked = _Recorded(monkeypatch, accept=0.0), []

    def draft(tokens, lengths, n):
        ids, q = _guess(lengths, n, 500)
        asked.append((lengths.tolist(), n))
        return ids, q if with_q else None

    out = m.generate(prompts, new, draft=draft, drafts=drafts, temperature=20.0, generator=torch.Generator(device="cuda").manual_seed(7))
    steps = _steps(lens, new, drafts)
    assert [n for _, n in asked] == [n for n, _ in steps if n] and len(record.calls) == 1 + len(steps)
    made = [1] * len(lens)
    for i, (n, rows) in enumerate(steps):
        c = record.calls[1 + i]
        assert c["cu"].diff().tolist() == rows and c["counts"].tolist() == rows
        lengths = torch.tensor([a + k for a, k in zip(lens, made)], device="cuda")
        if n:
            assert asked[i] == (lengths.tolist(), n)
        ids, q = _guess(lengths, n, 500)
        for s, r in enumerate(rows):
            lo = int(c["cu"][s])
            text, given = out[s][made[s]:made[s] + r], ids[s, :max(r - 1, 0)]
            assert torch.equal(c["draft"][lo:lo + len(given)], given)
            if with_q and len(given):
                assert torch.equal(c["q"][lo:lo + len(given)], q[s, :len(given)])
            assert torch.equal(text[:len(given)], given) and torch.equal(c["tokens"][s, :r], text)
        made = [k + r for k, r in zip(made, rows)]
    # the rows of p are those of the model's own distribution after the same text
    for s, (prompt, o) in enumerate(zip(prompts, out)):
        ids = torch.cat([prompt, o.cpu()])
        step = m.cache.step({(seq := m.cache.add()): len(ids)})
        with torch.no_grad():
            want = m._logits(m._hidden(step, ids.cuda())).float()[lens[s] - 1:-1]
        m.cache.drop(seq)
        p = torch.cat([c["p"][int(c["cu"][s]):int(c["cu"][s + 1])] for c in record.calls])
        assert p.shape == want.shape
        got = p.log() * 20
        got, want = got - got.mean(1, keepdim=True), want - want.mean(1, keepdim=True)
        # K and V in 8 bits or bf16 by when they were seen: the bound of the logits' own test, twice; log of f32 adds 20 * 2^-20
        assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) < 2 * 0.06 + 1e-4


def test_drafts_that_are_refused_leave_a_token_a_step(loaded, monkeypatch):
    """Random numbers of nearly 1 against drafts that were certain: none is taken."""
    m = loaded(pages=20, sequences=3)
    record = _Recorded(monkeypatch, accept=1 - 2.0 ** -24)
    asked = []

    def draft(tokens, lengths, n):
        asked.append(n)
        return _guess(lengths, n, 500)[0], None

    out = m.generate([torch.arange(60), torch.arange(3)], 12, draft=draft, temperature=20.0, generator=torch.Generator(device="cuda").manual_seed(8))
    assert [len(o) for o in out] == [12, 12] and asked == [4] * 7 + [3, 2, 1] and len(record.calls) == 12
    assert all(c["counts"].tolist() == [1, 1] for c in record.calls)
    for s in range(2):
        assert out[s].tolist() == [int(c["tokens"][s, 0]) for c in record.calls]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_the_model_as_its_own_draft(loaded, temperature):
    """Drafts that the model itself makes, one by one, are nearly all taken: refused only where rounding moved a probability past
    the random number (or the likeliest token). Without any taken 22 calls would be made, with all of them 5 to 7 (pages cut some)."""
    m = loaded(pages=30, sequences=6)
    prompts = [torch.arange(n) % 500 for n in (60, 1, 127)]
    g = torch.Generator(device="cuda").manual_seed(9)
    asked = []

    def draft(tokens, lengths, n):
        asked.append(n)
        seqs = [m.cache.add() for _ in prompts]
        logits = m.forward({s: tokens[i, :k] for i, (s, k) in enumerate(zip(seqs, lengths.tolist()))})
        ids, probabilities = [], []
        for j in range(n):
            p = m._probabilities(logits, temperature)
            ids.append(torch.multinomial(p, 1, generator=g)[:, 0])
            probabilities.append(p)
            if j + 1 < n:
                logits = m.forward({s: ids[-1][i:i + 1] for i, s in enumerate(seqs)})
        for s in seqs:
            m.cache.drop(s)
        return torch.stack(ids, 1), torch.stack(probabilities, 1)

    out = m.generate(prompts, 24, draft=draft, temperature=temperature, generator=g)
    assert [len(o) for o in out] == [24] * 3
    assert len(asked) <= 11, asked
