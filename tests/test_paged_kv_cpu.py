"""The paged KV cache's host side: argument checks, the C entry points' refusals, and which pages and
tails belong to which sequence."""
from __future__ import annotations

import ctypes

import pytest
import torch

from bigsmall_amd import _native
from bigsmall_amd.paged_kv import HEAD_DIMS, PAGE, KVBatch, KVPool, PagedKVCache, Rope, _Books, kv_append, kv_attend, kv_read


def _aligned(*shape, dtype):
    size = torch.empty(0, dtype=dtype).element_size()
    n = 1
    for s in shape:
        n *= s
    raw = torch.zeros(n * size + 64, dtype=torch.uint8)
    at = -raw.data_ptr() % 64
    return raw[at:at + n * size].view(dtype).view(shape)


def _parts(pages=4, tails=2, heads=2, dim=64, kind=torch.int8):
    return [_aligned(pages, heads, PAGE, dim, dtype=kind), _aligned(pages, heads, dim, PAGE, dtype=kind),
            _aligned(pages, heads, dtype=torch.float32), _aligned(pages, heads, dtype=torch.float32),
            _aligned(tails, heads, PAGE, dim, dtype=torch.bfloat16), _aligned(tails, heads, dim, PAGE, dtype=torch.bfloat16)]


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def _batch(**change):
    args = dict(start=_i32(0, 5), cu=_i32(0, 1, 2), table=torch.zeros(2, 3, dtype=torch.int32),
                tails=torch.zeros(2, 2, dtype=torch.int32), max_new=1, max_len=6)
    args.update(change)
    return KVBatch(**args)


def test_pool_refuses_what_does_not_fit():
    KVPool(*_parts())
    for d in HEAD_DIMS:
        KVPool(*_parts(dim=d, kind=torch.float8_e4m3fn))
    for change in (dict(dim=72), dict(kind=torch.uint8), dict(kind=torch.bfloat16), dict(pages=0), dict(tails=0), dict(heads=0)):
        with pytest.raises(ValueError):
            KVPool(*_parts(**change))
    for i in range(6):
        for bad in (lambda t: t.to(torch.float64), lambda t: t[:0], lambda t: t[:1], lambda t: t.repeat_interleave(2, -1)[..., ::2]):
            parts = _parts()
            parts[i] = bad(parts[i])
            if i in (0, 4) and parts[i].dtype == _parts()[i].dtype and parts[i].is_contiguous() and len(parts[i]) == 1:
                continue        # fewer pages (tails) of k alone disagrees with v's: checked by the next one
            with pytest.raises(ValueError):
                KVPool(*parts)
    parts = _parts()
    raw = torch.zeros(parts[0].numel() + 1, dtype=torch.int8)
    at = 1 if raw.data_ptr() % 16 == 0 else 0
    parts[0] = raw[at:at + parts[0].numel()].view(parts[0].shape)
    if parts[0].data_ptr() % 16:
        with pytest.raises(ValueError, match="aligned"):
            KVPool(*parts)


def test_batch_refuses_what_does_not_fit():
    _batch()
    for change in (dict(start=_i32(0, 5).long()), dict(start=_i32(0)), dict(cu=_i32(0, 1)), dict(cu=torch.zeros(3)),
                   dict(table=torch.zeros(2, 3)), dict(table=torch.zeros(3, 3, dtype=torch.int32)),
                   dict(table=torch.zeros(3, 2, dtype=torch.int32).t()), dict(tails=_i32(0, 0)), dict(max_new=-1), dict(max_len=1 << 30)):
        with pytest.raises(ValueError):
            _batch(**change)
    wide = torch.zeros(2, 10, dtype=torch.int32)[:, 2:5]
    assert _batch(table=wide).c.table_stride == 10


def test_rope():
    r = Rope.from_theta(32, 50, 10000.0, device="cpu")
    assert r.rot == 32 and r.cos.shape == (50, 16) and float(r.cos[0, 0]) == 1.0
    assert abs(float(r.sin[3, 1]) - torch.sin(torch.tensor(3 * 10000.0 ** (-2 / 32))).item()) < 1e-6
    for cos, sin in ((torch.zeros(5, 6), torch.zeros(5, 6)), (torch.zeros(5, 8), torch.zeros(5, 4)),
                     (torch.zeros(5, 8, dtype=torch.float64), torch.zeros(5, 8)), (torch.zeros(8), torch.zeros(8))):
        with pytest.raises(ValueError):
            Rope(cos, sin)


def test_operators_run_on_a_gpu_only():
    pool, batch = KVPool(*_parts()), _batch()
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: kv_append(pool, batch, x, x, x), lambda: kv_attend(pool, batch, x),
                 lambda: kv_read(pool, _i32(0, 1), 65, _i32(0))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.fixture
def on_gpu(monkeypatch):
    """The checks that come after the device's, on host tensors; nothing may be launched."""
    from bigsmall_amd import paged_kv
    monkeypatch.setattr(paged_kv, "_gpu", lambda pool: None)

    class Nothing:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(paged_kv._native, "lib", lambda: Nothing())


def test_calls_refuse_what_does_not_fit(on_gpu):
    pool, batch = KVPool(*_parts()), _batch()

    def rows(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype)

    k, q = rows(2, 2, 64), rows(2, 4, 64)
    rope = Rope.from_theta(64, 10, device="cpu")
    for args in ((q, k, rows(2, 2, 64, dtype=torch.float16)), (q, rows(2, 2, 80), k), (q, rows(2, 1, 64), k), (q, k, rows(3, 2, 64)),
                 (rows(3, 4, 64), k, k), (rows(2, 3, 64), k, k), (rows(2, 0, 64), k, k), (rows(2, 64), k, k), (None, None, k),
                 (q, k, k, Rope.from_theta(72, 10, device="cpu")), (q, k, k, Rope.from_theta(64, 5, device="cpu"))):
        with pytest.raises(ValueError):
            kv_append(pool, batch, *args)
    with pytest.raises(ValueError, match="out"):
        kv_append(pool, batch, q, k, k, rope, out=rows(2, 8, 64)[:, ::2])
    for q_bad in (rows(2, 3, 64), rows(2, 4, 96), rows(2, 4, 64, dtype=torch.float32), rows(8, 64)):
        with pytest.raises(ValueError):
            kv_attend(pool, batch, q_bad)
    for options in (dict(window=-1), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(slopes=torch.zeros(3)),
                    dict(slopes=torch.zeros(4, dtype=torch.float64)), dict(prefix=_i32(0)), dict(first=_i32(0, 0, 0)),
                    dict(first=torch.zeros(2, dtype=torch.int64)), dict(slopes=torch.zeros(8)[::2])):
        with pytest.raises(ValueError):
            kv_attend(pool, batch, q, **options)
    for args in ((_i32(0), 128, _i32(0)), (_i32(0), -1, _i32(0)), (_i32(0).long(), 64, _i32(0)), (_i32(0)[None], 64, _i32(0)),
                 (_i32(0), 5, _i32()), (_i32(0, 0, 0)[::2], 64, _i32(0))):
        with pytest.raises(ValueError):
            kv_read(pool, *args)


def test_c_entries_refuse_bad_arguments():
    """Every refusal comes before any launch, so these run without a GPU."""
    L = _native.lib()
    keep = KVPool(*_parts()), _batch()                # (they own the memory)
    ok_pool, ok_batch = (x.c for x in keep)
    ok_batch.n_rows = 2
    P, ARG = ctypes.byref, _native.BS_ERR_ARG
    x = _aligned(2, 8, 64, dtype=torch.bfloat16)

    def pool(**change):
        c = _native.BsKvPool.from_buffer_copy(ok_pool)
        for n, v in change.items():
            setattr(c, n, v)
        return c

    def batch(**change):
        c = _native.BsKvBatch.from_buffer_copy(ok_batch)
        for n, v in change.items():
            setattr(c, n, v)
        return c

    def rows(**change):
        c = _native.BsKvRows(x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr(), 512, 64, 512, 64,
                             512, 64, 4, 64, 0, 10)
        for n, v in change.items():
            setattr(c, n, v)
        return c

    def query(**change):
        c = _native.BsKvQuery(x.data_ptr(), x.data_ptr(), 0, 0, 0, 0, 512, 64, 4, 0, 0.125, 0.0)
        for n, v in change.items():
            setattr(c, n, v)
        return c

    bad_pools = [pool(k=0), pool(v_scale=0), pool(k_tail=ok_pool.k_tail + 2), pool(head_dim=72), pool(kind=2), pool(n_kv_heads=0)]
    bad_batches = [batch(start=0), batch(table=0), batch(table_cols=1 << 25), batch(table_stride=1), batch(n_rows=1 << 31)]
    assert L.bs_kv_append(None, P(ok_batch), P(rows()), None, None) == ARG
    assert L.bs_kv_attend(P(ok_pool), P(ok_batch), None, None, 0, None, None) == ARG
    for p, b in [(p, ok_batch) for p in bad_pools] + [(ok_pool, b) for b in bad_batches]:
        assert L.bs_kv_append(P(p), P(b), P(rows()), None, None) == ARG
        assert L.bs_kv_attend(P(p), P(b), P(query()), None, 0, None, None) == ARG
        assert L.bs_kv_attend_work_bytes(P(p), P(b), 4) == 0
    for r in (rows(rot=12), rows(rot=72), rows(cos=0), rows(sin=x.data_ptr() + 4), rows(k=0), rows(v=x.data_ptr() + 2), rows(k_token=7),
              rows(v_head=4), rows(q_out=0), rows(q_head=1), rows(n_q_heads=3), rows(n_q_heads=0)):
        assert L.bs_kv_append(P(ok_pool), P(ok_batch), P(r), None, None) == ARG
    for a in (query(q=0), query(out=x.data_ptr() + 8), query(q_token=4), query(n_q_heads=5), query(softcap=-1.0), query(softcap=float("nan"))):
        assert L.bs_kv_attend(P(ok_pool), P(ok_batch), P(a), None, 0, None, None) == ARG
    long = batch(max_len=100000)
    need = L.bs_kv_attend_work_bytes(P(ok_pool), P(long), 4)
    assert need > 0
    assert L.bs_kv_attend(P(ok_pool), P(long), P(query()), None, 0, None, None) == _native.BS_ERR_CAP
    assert L.bs_kv_attend(P(ok_pool), P(long), P(query()), x.data_ptr(), need - 1, None, None) == _native.BS_ERR_CAP
    for n, cols, out in ((65, 0, x.data_ptr()), (64, 1, x.data_ptr() + 2), (64, 1, 0), ((1 << 30) + 1, 1 << 24, x.data_ptr())):
        assert L.bs_kv_read(P(ok_pool), x.data_ptr(), cols, x.data_ptr(), n, out, out, None, None) == ARG
    # nothing to do
    empty = batch(n_rows=0)
    assert L.bs_kv_append(P(ok_pool), P(empty), P(rows()), None, None) == _native.BS_OK
    assert L.bs_kv_attend(P(ok_pool), P(empty), P(query()), None, 0, None, None) == _native.BS_OK
    assert L.bs_kv_read(P(ok_pool), None, 0, None, 0, None, None, None, None) == _native.BS_OK


def _step(books, new):
    flat, (b, m), max_new, max_len = books.step(new)
    start, cu, tails, table = flat[:b], flat[b:2 * b + 1], flat[2 * b + 1:4 * b + 1], flat[4 * b + 1:]
    assert len(table) == b * m
    return start, cu, [tails[2 * i:2 * i + 2] for i in range(b)], [table[i * m:(i + 1) * m] for i in range(b)], max_new, max_len


def test_books():
    books = _Books(10, 3)
    a = books.add()
    start, cu, tails, table, max_new, max_len = _step(books, {a: 130})
    assert (start, cu, table, max_new, max_len) == ([0], [0, 130], [[0, 1, 0]], 130, 130)
    assert tails[0][0] != tails[0][1]                  # a page was completed
    now = tails[0][1]
    b = books.add()
    start, cu, tails, table, _, max_len = _step(books, {b: 1, a: 1})
    assert start == [0, 130] and cu == [0, 1, 2] and max_len == 131
    assert tails[0][0] == tails[0][1] and tails[1] == [now, now] and len({tails[0][0], now}) == 2
    _, _, tails, table, _, _ = _step(books, {a: 61})
    assert books.length(a) == 192 and table == [[0, 1, 2]] and tails[0][0] != tails[0][1]
    with pytest.raises(RuntimeError, match="pages"):
        books.step({b: 64 * 8})
    assert books.length(b) == 1 and len(books.free) == 7
    books.step({b: 64 * 7})
    assert not books.free and books.where(b)[0] == 449
    books.drop(a)
    assert len(books.free) == 3 and books.where(b)[1] == [3, 4, 5, 6, 7, 8, 9]
    for bad in (lambda: books.step({a: 1}), lambda: books.length(a), lambda: books.drop(a)):
        with pytest.raises(KeyError):
            bad()
    for bad in ({}, {b: 0}, {b: -1}, {b: 1 << 30}):
        with pytest.raises(ValueError):
            books.step(bad)
    books.add(), books.add()
    with pytest.raises(RuntimeError):
        books.add()
    used = {t for s in books.seqs.values() for t in s[2:]}
    assert len(used) == 6


def test_cache_constructor():
    for args in ((0, 1, 64, 1, 1), (1, 1, 65, 1, 1), (1, 1, 64, 0, 1), (1, 1, 64, 1, 0)):
        with pytest.raises(ValueError):
            PagedKVCache(*args)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, 1, 1, kind=torch.bfloat16)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            PagedKVCache(1, 1, 64, 1, 1)
