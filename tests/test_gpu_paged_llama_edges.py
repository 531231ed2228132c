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


def test_resume_without_room_or_entry_takes_nothing():
    import bigsmall_amd
    from bigsmall_amd.paged_llama import PagedLlama
    m = PagedLlama.__new__(PagedLlama)
    m.device = torch.device("cuda")
    m.cache = bigsmall_amd.PagedKVCache(2, 1, 64, pages=4, sequences=2)
    x = torch.randn(200, 1, 64, device="cuda").bfloat16()
    seq, store = m.cache.add(), bigsmall_amd.CompressedKVCache(device="cuda")
    step = m.cache.step({seq: 200})
    for i in range(2):
        m.cache.append(i, step, None, x, x)
    kept = m.cache.read(1, seq)
    m.park(seq, store)
    assert m.cache.free_pages() == 4
    other = m.cache.add()
    m.cache.step({other: 130})                        # two of four pages: three are needed
    was = _books(m)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="pages"):
            m.resume(seq, store)
        with pytest.raises(KeyError):
            m.resume(seq + 100, store)                # never parked
        assert _books(m) == was
    m.cache.drop(other)
    back = m.resume(seq, store)
    for got, want in zip(m.cache.read(1, back), kept):
        assert got.shape == want.shape
