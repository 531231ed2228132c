"""Status words that lie on another device than the call are refused before anything is launched: their address is not one
that the call's GPU may write to."""
from __future__ import annotations

import pytest
import torch

from bigsmall_amd.device import StatusWord
from bigsmall_amd.draft import draft_verify
from bigsmall_amd.kv_tables import KVTables
from bigsmall_amd.paged_kv import KVPool, kv_append, kv_attend, kv_read
from test_paged_kv_cpu import _batch, _parts, on_gpu  # noqa: F401 (a fixture)


class _Elsewhere:
    """A status word's tensor on a GPU that the call does not run on."""
    device = "cuda:3"

    def get_device(self):
        return 3

    def data_ptr(self):
        raise AssertionError("its address was taken")


ELSEWHERE = StatusWord(view=_Elsewhere())


def test_words_of_no_call_and_of_the_calls_device():
    from bigsmall_amd.device import status_ptr
    assert status_ptr(None, 0) is None
    word = StatusWord(view=torch.zeros(1, dtype=torch.int32))
    assert status_ptr(word, -1) == word.t.data_ptr()
    for index in (0, 5):            # on the host, where StatusWord() without a device puts it
        with pytest.raises(ValueError, match="status word is on"):
            status_ptr(StatusWord(), index)


def test_cache_calls_refuse_words_of_another_device(on_gpu):  # noqa: F811
    pool, batch = KVPool(*_parts()), _batch()
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kv_append(pool, batch, x, x, x, status=ELSEWHERE), lambda: kv_attend(pool, batch, x, status=ELSEWHERE),
                 lambda: kv_read(pool, pages, 1, pages, status=ELSEWHERE)):
        with pytest.raises(ValueError, match="status word is on cuda:3"):
            call()


def test_verification_refuses_words_of_another_device():
    with pytest.raises(ValueError, match="status word is on cuda:3"):
        draft_verify(torch.zeros(5, 10), torch.zeros(5, dtype=torch.int64), torch.tensor([0, 2, 5], dtype=torch.int32), torch.zeros(5),
                     torch.zeros(2), status=ELSEWHERE)


def test_tables_refuse_words_of_another_device(monkeypatch):
    t = KVTables.__new__(KVTables)
    t.places, t.longest, t.device, t.index, t._made = 3, 128, torch.device("cpu"), -1, "a step"
    monkeypatch.setattr(KVTables, "_call", lambda self, name, *args: pytest.fail(f"{name} was called"))
    a = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="status word is on cuda:3"):
        t.step(a, a, rows=2, status=ELSEWHERE)
    with pytest.raises(ValueError, match="status word is on cuda:3"):
        t.drop(a, status=ELSEWHERE)
    assert t._made == "a step"               # a refused call leaves the step before as it was
