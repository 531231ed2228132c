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
