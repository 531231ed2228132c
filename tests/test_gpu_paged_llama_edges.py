"""PagedLlama where a call is refused: the cache is as it was before."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged_llama import model  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def _books(m):
    b = m.cache._books
    return b.free[:], b.free_tails[:], {s: [e[0], e[1][:], e[2], e[3]] for s, e in b.seqs.items()}


def test_forward_that_is_refused_leaves_the_cache_as_it_was(model):  # noqa: F811
    """One sequence past the rotation's positions, refused by the first layer, and a layer that fails half-way: the other
    sequence of the step goes on as if nothing had been."""
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    path, config, _ = model
    ids = torch.arange(130) % config.vocab_size
    with bigsmall_amd.StreamingLoader(str(path), device="cuda") as loader:
        m = PagedLlama(loader, config, pages=24, sequences=3)
        alone = m.cache.add()
        m.forward({alone: ids[:70]})
        want = m.forward({alone: ids[70:]})
        m.cache.drop(alone)
        seq, other = m.cache.add(), m.cache.add()
        m.forward({seq: ids[:70]})
        was = _books(m)
        with pytest.raises(ValueError, match="positions"):
            m.forward({other: torch.zeros(600, dtype=torch.int64), seq: ids[:60]})
        assert _books(m) == was
        attend, calls = m.cache.attend, []

        def failing(layer, step, q):
            calls.append(layer)
            if layer == 1:
                raise MemoryError
            return attend(layer, step, q)
        m.cache.attend = failing
        for n in (1, 57, 58, 60):                    # the tail goes on, is filled, a page is completed
            with pytest.raises(MemoryError):
                m.forward({seq: ids[:n], other: ids})
        assert calls == [0, 1] * 4 and _books(m) == was
        m.cache.attend = attend
        assert torch.equal(m.forward({seq: ids[70:]}), want)


def test_steps_are_taken_back_once():
    import bigsmall_amd
    cache = bigsmall_amd.PagedKVCache(1, 1, 64, pages=4, sequences=2)
    a = cache.add()
    x = torch.randn(200, 1, 64, device="cuda").bfloat16()
    cache.append(0, cache.step({a: 100}), None, x[:100], x[:100])
    kept = cache.read(0, a)
    step = cache.step({a: 100})
    cache.append(0, step, None, x[100:], x[100:])
    cache.undo(step)
    assert cache.length(a) == 100 and cache.free_pages() == 3 and all(torch.equal(p, q) for p, q in zip(cache.read(0, a), kept))
    with pytest.raises(RuntimeError, match="already"):
        cache.undo(step)
    step = cache.step({a: 1})
    cache.step({a: 1})
    with pytest.raises(RuntimeError, match="gone on"):
        cache.undo(step)
