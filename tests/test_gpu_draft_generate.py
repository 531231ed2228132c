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
