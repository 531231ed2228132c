"""A paged KV cache in 8 bits, and attention over it (no reference counterpart;
the reference's KV cache, bigsmall/kv_cache_manager.py:22-91, stores entries
for later and does not attend).

Storage of a layer (KVPool): pages of 64 tokens in int8 or e4m3 with one scale
per page and kv head, for K and for V; K pages [pages, kv heads, 64, dim], V
pages [pages, kv heads, dim, 64]. The tokens of a sequence's unfinished page
are kept in bf16 in a tail of the same shape and quantised once, when the page
is full: what the cache holds depends neither on how the tokens were cut into
chunks nor on later tokens.

A step (KVBatch) is one call for every sequence in it: where each sequence's
new rows lie, how many tokens it has cached, its pages and its tails.

    kv_append(pool, batch, q, k, v, rope)  rotate q and k, write k and v; returns q
    kv_attend(pool, batch, q, ...)         attention of the new rows over the cache
    kv_read(pool, pages, n, tail)          a sequence's K and V as bf16 [heads, n, dim]

PagedKVCache keeps the pools of all layers and does the bookkeeping: sequences,
pages, tails, steps.

Inference only: inputs that require a gradient are refused while gradients are
recorded. All calls run on the current torch stream of the pool's device and do not
synchronise. Work areas come from torch's allocator for each call. Tensors of
another stream need the usual wait and record_stream by the caller.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import _native

PAGE = 64
HEAD_DIMS = (64, 80, 96, 128, 256)
_KINDS = {torch.int8: 0, torch.float8_e4m3fn: 1}


def _tensor(name: str, t, dtype, device=None, shape=None):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache is on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


class KVPool:
    """One layer's storage: the six tensors (contiguous, on one GPU), checked once. What kv_append writes is what
    kv_attend takes; where something else fills them: v_scale positive (2^-49 to 2^54), the tails' V finite."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "device", "index", "dtype", "n_pages", "n_tails",
                 "n_kv_heads", "head_dim", "c", "ref")

    def __init__(self, k, v, k_scale, v_scale, k_tail, v_tail):
        if not isinstance(k, torch.Tensor) or k.dtype not in _KINDS or k.dim() != 4 or k.shape[2] != PAGE:
            raise ValueError("KVPool: k must be an int8 or float8_e4m3fn tensor [pages, kv heads, 64, head dim]")
        n, h, _, d = k.shape
        if d not in HEAD_DIMS or h < 1:
            raise ValueError(f"KVPool: head dim {d} is not one of {HEAD_DIMS}" if h else "KVPool: no kv heads")
        _tensor("v", v, k.dtype, k.device, (n, h, d, PAGE))
        _tensor("k_scale", k_scale, torch.float32, k.device, (n, h))
        _tensor("v_scale", v_scale, torch.float32, k.device, (n, h))
        if not isinstance(k_tail, torch.Tensor) or k_tail.dim() != 4:
            raise ValueError("KVPool: k_tail must be a tensor [tails, kv heads, 64, head dim]")
        m = k_tail.shape[0]
        _tensor("k_tail", k_tail, torch.bfloat16, k.device, (m, h, PAGE, d))
        _tensor("v_tail", v_tail, torch.bfloat16, k.device, (m, h, d, PAGE))
        if n < 1 or m < 1:
            raise ValueError("KVPool: at least one page and one tail")
        for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale), ("k_tail", k_tail), ("v_tail", v_tail)):
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"KVPool: {name} must be contiguous and 16-byte aligned")
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self.device, self.index, self.dtype = k.device, k.get_device(), k.dtype       # index: -1 on the host
        self.n_pages, self.n_tails, self.n_kv_heads, self.head_dim = n, m, h, d
        self.c = _native.BsKvPool(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k_tail.data_ptr(),
                                  v_tail.data_ptr(), n, m, h, d, _KINDS[k.dtype])
        self.ref = ctypes.byref(self.c)


class KVBatch:
    """One step over a batch of sequences, device int32 tensors:

    start [B]      tokens in the cache before the step
    cu [B + 1]     first new row of each sequence in the packed rows, from 0, ascending
    table [B, M]   page numbers; page p of a sequence holds its tokens 64 p .. 64 p + 63
    tails [B, 2]   the tail before the step and after it; where the step completes a page they
                   must differ (a step run again then reads what it read before)
    max_new, max_len: the largest number of new tokens and of tokens after the step of a
    sequence. They choose launch shapes; a wrong value costs time, not results (kv_append asks for
    a rope of max_len positions). Rows of q, k
    and v that no sequence covers are not read, and their outputs are not defined.
    total: the rows of all sequences, where the host knows them: calls with another number of
    rows are then refused. None: rows that reach past the given ones drop their sequence, which
    only a status word tells.
    """

    __slots__ = ("start", "cu", "table", "tails", "index", "n_seqs", "max_new", "max_len", "total", "before", "c", "_head", "_rest")

    def __init__(self, start, cu, table, tails, max_new: int, max_len: int, total: Optional[int] = None):
        _tensor("start", start, torch.int32)
        if start.dim() != 1:
            raise ValueError("KVBatch: start must be [sequences]")
        b = start.shape[0]
        _tensor("cu", cu, torch.int32, start.device, (b + 1,))
        _tensor("table", table, torch.int32, start.device)
        _tensor("tails", tails, torch.int32, start.device, (b, 2))
        if table.dim() != 2 or table.shape[0] != b or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("KVBatch: table must be [sequences, pages], rows contiguous")
        stride = table.stride(0) if b > 1 else max(table.stride(0), table.shape[1])
        if not (start.is_contiguous() and cu.is_contiguous() and tails.is_contiguous()) or stride < table.shape[1]:
            raise ValueError("KVBatch: start, cu and tails must be contiguous, table's rows apart")
        if b > 65535 or not 0 <= max_new < 1 << 30 or not 0 <= max_len < 1 << 30:
            raise ValueError("KVBatch: at most 65535 sequences, max_new and max_len below 2^30")
        self.start, self.cu, self.table, self.tails = start, cu, table, tails
        self.n_seqs, self.max_new, self.max_len, self.total = b, int(max_new), int(max_len), total
        self.before = None           # of a PagedKVCache's step: how to take it back
        self.c = _native.BsKvBatch(start.data_ptr(), cu.data_ptr(), table.data_ptr(), tails.data_ptr(), b, stride,
                                   table.shape[1], 0, int(max_new), int(max_len))
        self.index = start.get_device()
        at = _native.BsKvBatch.n_rows.offset
        self._head, self._rest = bytes(self.c)[:at], bytes(self.c)[at + 4:]

    def with_rows(self, n: int) -> bytes:
        """The C structure of a call with n rows: a value of its own, since layers and threads share the batch."""
        return self._head + n.to_bytes(4, "little") + self._rest


class Rope:
    """Rotation angles by position: cos and sin f32 [positions, turned channels / 2] on the GPU.
    The first 2 * cos.shape[1] channels turn, in pairs (i, i + half), or (2i, 2i + 1) if interleaved."""

    __slots__ = ("cos", "sin", "interleaved", "rot", "positions", "index", "cos_ptr", "sin_ptr")

    def __init__(self, cos, sin, interleaved: bool = False):
        _tensor("cos", cos, torch.float32)
        if cos.dim() != 2 or cos.shape[1] % 4:
            raise ValueError("Rope: cos must be [positions, turned channels / 2], the turned channels a multiple of 8")
        _tensor("sin", sin, torch.float32, cos.device, cos.shape)
        self.cos, self.sin = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                              for t in (cos, sin))
        self.interleaved, self.rot, self.positions = bool(interleaved), 2 * cos.shape[1], cos.shape[0]
        self.index, self.cos_ptr, self.sin_ptr = cos.get_device(), self.cos.data_ptr(), self.sin.data_ptr()

    @classmethod
    def from_theta(cls, rot: int, positions: int, theta: float = 10000.0, interleaved: bool = False, device="cuda") -> "Rope":
        """Angles position * theta^(-2i / rot), computed in 64 bits."""
        freq = float(theta) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cpu") / rot)
        angle = torch.arange(positions, dtype=torch.float64, device="cpu")[:, None] * freq
        return cls(angle.cos().float().to(device), angle.sin().float().to(device), interleaved)


def _rows(name: str, t, n: Optional[int], heads: Optional[int], pool: KVPool):
    """t as bf16 rows [tokens, heads, dim] that the kernels can read, with its tokens, heads, address
    and strides: in place if its rows start at multiples of 16 bytes and its last dimension is
    contiguous, else a contiguous copy."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be a bfloat16 tensor [tokens, heads, head dim]")
    shape = t.shape
    if len(shape) != 3 or shape[2] != pool.head_dim or (n is not None and shape[0] != n) or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} has shape {tuple(shape)}, expected [{n if n is not None else 'tokens'}, "
                         f"{heads if heads is not None else 'heads'}, {pool.head_dim}]")
    if t.get_device() != pool.index:
        raise ValueError(f"{name} is on {t.device}, the cache is on {pool.device}")
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    if s2 != 1 or (s0 | s1) & 7 or p & 15:
        # the stride of a dimension of one is any number: torch calls such a tensor contiguous
        s0, s1 = 0 if shape[0] == 1 else s0, 0 if shape[1] == 1 else s1
        if s2 != 1 or (s0 | s1) & 7 or p & 15:
            t = t.clone(memory_format=torch.contiguous_format)
            s0, s1, p = shape[1] * shape[2], shape[2], t.data_ptr()
    return t, shape[0], shape[1], p, s0, s1


def _check_heads(h: int, pool: KVPool) -> None:
    if h < 1 or h % pool.n_kv_heads:
        raise ValueError(f"q has {h} heads, not a multiple of the cache's {pool.n_kv_heads} kv heads")


def _gpu(pool: KVPool) -> None:
    if pool.index < 0:
        raise RuntimeError("the paged KV cache's operators run on an AMD GPU (MI355X); the pool is on " + str(pool.device))


def _refuse_grad() -> None:
    raise RuntimeError("the paged KV cache has no backward pass: call it under torch.no_grad(), or detach q, k and v")


def _refuse_total(batch: KVBatch, n: int) -> None:
    raise ValueError(f"{n} rows, the step has {batch.total}")


def _check_batch(pool: KVPool, batch: KVBatch) -> None:
    _gpu(pool)
    if batch.index != pool.index:
        raise ValueError(f"the batch is on {batch.start.device}, the cache is on {pool.device}")


# The current stream's handle of a device, without the Stream object that torch.cuda.current_stream makes (2 us of a
# call that takes 10).
_stream = torch._C._cuda_getCurrentRawStream
_recording = torch.is_grad_enabled

# bs_kv_rows and bs_kv_query of include/bigsmall_kv.h, packed: a ctypes structure of as many fields takes 1 us more to fill
_ROWS = struct.Struct("=6Q6q4I")
_QUERY = struct.Struct("=6Q2q2I2f")
assert _ROWS.size == ctypes.sizeof(_native.BsKvRows) and _QUERY.size == ctypes.sizeof(_native.BsKvQuery)


def _call(name: str, pool: KVPool, *args) -> None:
    """A C entry point on the pool's device and its current stream."""
    index = pool.index
    if index == torch.cuda.current_device():
        rc = getattr(_native.lib(), name)(pool.ref, *args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(_native.lib(), name)(pool.ref, *args, _stream(index))
    if rc:
        _native.check(rc, name)


def kv_append(pool: KVPool, batch: KVBatch, q, k, v, rope: Optional[Rope] = None, out=None, status=None):
    """Rotate q [T, q heads, dim] and k [T, kv heads, dim] (bf16) by their tokens' positions and write k
    and v into the cache. Returns the rotated q (into `out`, a contiguous bf16 tensor of q's shape, q
    itself among them), or None if q is None. rope None: nothing turns and q comes back as it is.

    A token whose rotated k, or whose v, is not finite in a head makes NaN of exactly the rows that see
    it there (once its page is full: of the rows that see any token of the page). status: a
    device.StatusWord that gets BS_DEV_ERR_BOUNDS where the batch names pages, tails or positions that
    do not exist; such parts are not written."""
    _check_batch(pool, batch)
    k, t, _, kp, k0, k1 = _rows("k", k, None, pool.n_kv_heads, pool)
    if t != batch.total and batch.total is not None:
        _refuse_total(batch, t)
    v, _, _, vp, v0, v1 = _rows("v", v, t, pool.n_kv_heads, pool)
    rot = cos = sin = inter = n_pos = heads = qp = op = q0 = q1 = 0
    if rope is not None:
        rot, inter, n_pos, cos, sin = rope.rot, rope.interleaved, rope.positions, rope.cos_ptr, rope.sin_ptr
        if rot > pool.head_dim:
            raise ValueError(f"rope turns {rot} channels, the head dim is {pool.head_dim}")
        if n_pos < batch.max_len:
            raise ValueError(f"rope has {n_pos} positions, the batch reaches {batch.max_len}")
        if rope.index != pool.index:
            raise ValueError(f"rope is on {rope.cos.device}, the cache is on {pool.device}")
    result = q
    if q is not None:
        q, _, heads, qp, q0, q1 = _rows("q", q, t, None, pool)
        _check_heads(heads, pool)
        if rot or out is not None:
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                op = out.data_ptr()
            else:
                copy, _, _, op, _, _ = _rows("out", out, t, heads, pool)
                if copy is not out or not out.is_contiguous():
                    raise ValueError("out must be contiguous and 16-byte aligned")
            result = out
        else:
            qp = 0
    if _recording() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)):
        _refuse_grad()
    if t:
        _call("bs_kv_append", pool, batch.with_rows(t), _ROWS.pack(qp, kp, vp, op, cos, sin, q0, q1, k0, k1, v0, v1, heads, rot, inter, n_pos),
              status.ptr if status else None)
    return result


def kv_attend(pool: KVPool, batch: KVBatch, q, scale: Optional[float] = None, softcap: float = 0.0, slopes=None,
              window: int = 0, prefix=None, first=None, return_lse: bool = False, status=None):
    """Attention of the step's rows q [T, q heads, dim] (bf16, rotated) over their sequences' caches, the
    step's own tokens included: append first. Returns bf16 [T, q heads, dim], with return_lse also the
    f32 [T, q heads] natural logarithm of the sum of exp(score).

    score = scale * q.k (scale: head_dim ** -0.5 by default), then softcap * tanh(score / softcap) if
    softcap is not 0, then minus slopes[head] * |position - key| if slopes (f32 [q heads]) are given.
    The row at position p sees key j if (j <= p, or j < prefix of its sequence) and j >= first of its
    row and j > p - window; prefix: int32 [B], first: int32 [T], window 0: none. A row that sees
    nothing gives 0 and -inf."""
    _check_batch(pool, batch)
    q, t, heads, qp, q0, q1 = _rows("q", q, None, None, pool)
    if t != batch.total and batch.total is not None:
        _refuse_total(batch, t)
    _check_heads(heads, pool)
    if not 0 <= window < 1 << 31 or not 0.0 <= softcap < float("inf"):
        raise ValueError("window and softcap must not be negative or infinite")
    if _recording() and (q.requires_grad or (slopes is not None and slopes.requires_grad)):
        _refuse_grad()
    sp = pp = fp = 0
    if slopes is not None:
        sp = _vector("slopes", slopes, heads, torch.float32, pool)
    if prefix is not None:
        pp = _vector("prefix", prefix, batch.n_seqs, torch.int32, pool)
    if first is not None:
        fp = _vector("first", first, t, torch.int32, pool)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((t, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if t:
        step = batch.with_rows(t)
        n = _native.lib().bs_kv_attend_work_bytes(pool.ref, step, heads)
        work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        if softcap:               # (what f32 can hold; the library takes what lies outside for these)
            softcap = min(max(softcap, 2.0 ** -60), 2.0 ** 60)
        query = _QUERY.pack(qp, out.data_ptr(), lse.data_ptr() if return_lse else 0, sp, pp, fp, q0, q1, heads, window,
                            pool.head_dim ** -0.5 if scale is None else scale, softcap)
        _call("bs_kv_attend", pool, step, query, work.data_ptr() if n else 0, n, status.ptr if status else None)
    return (out, lse) if return_lse else out


def _vector(name: str, x, n: int, dtype, pool: KVPool) -> int:
    if not _tensor(name, x, dtype, pool.device, (n,)).is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return x.data_ptr()


def kv_read(pool: KVPool, pages, n: int, tail, status=None):
    """One sequence's first n tokens as bf16 K and V [kv heads, n, dim] (the layout that
    CompressedKVCache.set_blocks takes). pages: its page numbers, a contiguous int32 row of a batch's
    table; tail: an int32 tensor whose first element is its tail's number, read if n is no multiple of 64."""
    _gpu(pool)
    _tensor("pages", pages, torch.int32, pool.device)
    _tensor("tail", tail, torch.int32, pool.device)
    shape = pages.shape
    if len(shape) != 1 or not pages.is_contiguous() or tail.numel() < 1:
        raise ValueError("kv_read: pages must be a contiguous row, tail must hold a number")
    if not 0 <= n < 1 << 30 or n // PAGE > shape[0]:
        raise ValueError(f"kv_read: {n} tokens need {n // PAGE} full pages, {shape[0]} given")
    k = torch.empty((pool.n_kv_heads, n, pool.head_dim), dtype=torch.bfloat16, device=pool.device)
    v = torch.empty_like(k)
    _call("bs_kv_read", pool, pages.data_ptr(), shape[0], tail.data_ptr(), n, k.data_ptr(), v.data_ptr(), status.ptr if status else None)
    return k, v


class PagedKVCache:
    """The pools of all layers and their sequences.

        cache = PagedKVCache(layers, kv_heads, head_dim, pages=4096, sequences=64)
        a = cache.add()                                  # a sequence
        step = cache.step({a: 37})                       # 37 new tokens of a: pages are taken, lengths advance
        for layer in range(layers):
            q = cache.append(layer, step, q, k, v, rope)
            y = cache.attend(layer, step, q)
        k, v = cache.read(layer, a)                      # bf16 [kv heads, tokens, dim]
        cache.drop(a)

    A page number names the same page in every layer's pool. kind: torch.int8 or torch.float8_e4m3fn.
    Where a step's calls raise, `undo(step)` takes it back.
    Memory: each page 64 * head_dim * kv_heads * 2 bytes a layer, each sequence two tails of four
    times that in all (a tail is bf16 and has a second one to move to when its page is completed)."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, sequences: int, kind=torch.int8, device="cuda"):
        from .device import require_gpu
        if kind not in _KINDS:
            raise ValueError("PagedKVCache: kind must be torch.int8 or torch.float8_e4m3fn")
        if min(layers, kv_heads, pages, sequences) < 1 or head_dim not in HEAD_DIMS:
            raise ValueError(f"PagedKVCache: counts must be positive and the head dim one of {HEAD_DIMS}")
        self.device = require_gpu(device)
        self.kind = kind

        def room(*shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=self.device)

        self.pools = [KVPool(room(pages, kv_heads, PAGE, head_dim, dtype=torch.uint8).view(kind),
                             room(pages, kv_heads, head_dim, PAGE, dtype=torch.uint8).view(kind),
                             room(pages, kv_heads, dtype=torch.float32), room(pages, kv_heads, dtype=torch.float32),
                             room(2 * sequences, kv_heads, PAGE, head_dim, dtype=torch.bfloat16),
                             room(2 * sequences, kv_heads, head_dim, PAGE, dtype=torch.bfloat16)) for _ in range(layers)]
        self._books = _Books(pages, sequences)

    # ---- sequences
    def add(self) -> int:
        """A new, empty sequence."""
        return self._books.add()

    def drop(self, seq: int) -> None:
        """Forget a sequence; its pages may be taken by steps made from now on."""
        self._books.drop(seq)

    def length(self, seq: int) -> int:
        return self._books.length(seq)

    def free_pages(self) -> int:
        return len(self._books.free)

    def step(self, new: dict) -> KVBatch:
        """A step that appends new[seq] tokens to each sequence, rows packed in the dict's order. Takes the
        pages it needs (RuntimeError, and nothing taken, if there are too few). Appending must follow for
        every layer before the sequences' next step; where it does not, `undo` takes the step back."""
        before = self._books.note(new)
        arrays, shape, max_new, max_len = self._books.step(new)
        try:
            step = self._upload(arrays, shape, max_new, max_len)
        except BaseException:
            self._books.undo(before)
            raise
        step.before = before
        return step

    def undo(self, step: KVBatch) -> None:
        """Take back a step whose appends were refused or came to an end half-way: its sequences have their
        lengths, pages and tails of before it, and what they held then is untouched. Once, and before their
        next step (RuntimeError otherwise)."""
        if step.before is None:
            raise RuntimeError("not a step of this cache, or taken back already")
        self._books.undo(step.before)
        step.before = None

    def _upload(self, arrays, shape, max_new, max_len) -> KVBatch:
        flat = torch.tensor(arrays, dtype=torch.int32, device="cpu").pin_memory().to(self.device, non_blocking=True)
        b, m = shape
        start, cu, tails, table = flat.split([b, b + 1, 2 * b, b * m])
        return KVBatch(start, cu, table.view(b, m), tails.view(b, 2), max_new, max_len, arrays[2 * b])

    # ---- one layer
    def append(self, layer: int, step: KVBatch, q, k, v, rope: Optional[Rope] = None, **options):
        return kv_append(self.pools[layer], step, q, k, v, rope, **options)

    def attend(self, layer: int, step: KVBatch, q, **options):
        return kv_attend(self.pools[layer], step, q, **options)

    def read(self, layer: int, seq: int, status=None):
        """K and V of a sequence's appended tokens, bf16 [kv heads, tokens, dim]."""
        n, pages, tail = self._books.where(seq)
        row = torch.tensor(pages + [tail], dtype=torch.int32, device="cpu").to(self.device)
        return kv_read(self.pools[layer], row[:-1], n, row[-1:], status)


class _Books:
    """Which pages and tails belong to which sequence (host side of PagedKVCache)."""

    def __init__(self, pages: int, sequences: int):
        self.free = list(range(pages - 1, -1, -1))
        self.free_tails = list(range(2 * sequences - 2, -1, -2))
        self.seqs: dict = {}        # sequence -> [length, pages, its tail now, the other one]
        self.next = 0

    def _get(self, seq):
        if seq not in self.seqs:
            raise KeyError(f"no sequence {seq!r} in the cache")
        return self.seqs[seq]

    def add(self) -> int:
        if not self.free_tails:
            raise RuntimeError("PagedKVCache: as many sequences as it was made for are in use")
        tail = self.free_tails.pop()
        seq, self.next = self.next, self.next + 1
        self.seqs[seq] = [0, [], tail, tail + 1]
        return seq

    def drop(self, seq) -> None:
        _, pages, a, b = self._get(seq)
        del self.seqs[seq]
        self.free += reversed(pages)
        self.free_tails.append(min(a, b))

    def length(self, seq) -> int:
        return self._get(seq)[0]

    def where(self, seq):
        n, pages, tail, _ = self._get(seq)
        return n, list(pages), tail

    def note(self, new: dict) -> list:
        """What `undo` needs to take back the step that comes next: sequence, entry, length before and after it."""
        return [(seq, self._get(seq), self._get(seq)[0], self._get(seq)[0] + int(n)) for seq, n in new.items()]

    def undo(self, before: list) -> None:
        for seq, e, _, after in before:
            if self.seqs.get(seq) is not e or e[0] != after:
                raise RuntimeError(f"sequence {seq} has gone on or been dropped since the step")
        for _, e, length, after in reversed(before):
            # a completed page's step went on in the other tail, and an unfinished one's wrote past `length` only
            pages = e[1]
            while len(pages) > length // PAGE:
                self.free.append(pages.pop())
            if after // PAGE > length // PAGE:
                e[2], e[3] = e[3], e[2]
            e[0] = length

    def step(self, new: dict):
        """(start, cu, tails, table) as one flat list, (sequences, table width), max_new, max_len."""
        rows, need = [], 0
        for seq, n in new.items():
            n = int(n)
            e = self._get(seq)
            if n < 1:
                raise ValueError(f"sequence {seq}: {n} new tokens; a step appends at least one")
            if e[0] + n >= 1 << 30:
                raise ValueError(f"sequence {seq}: too long")
            rows.append((e, n))
            need += (e[0] + n) // PAGE - len(e[1])
        if not rows:
            raise ValueError("a step needs at least one sequence")
        if need > len(self.free):
            raise RuntimeError(f"PagedKVCache: the step needs {need} pages, {len(self.free)} are free")
        start, cu, tails, tables = [], [0], [], []
        for e, n in rows:
            length, pages, tail, other = e
            end = length + n
            pages += [self.free.pop() for _ in range(end // PAGE - len(pages))]
            moves = end // PAGE > length // PAGE
            after = other if moves else tail
            start.append(length)
            cu.append(cu[-1] + n)
            tails += [tail, after]
            tables.append(pages)
            e[0] = end
            if moves:
                e[2], e[3] = other, tail
        m = max(1, max((start[i] + rows[i][1] + PAGE - 1) // PAGE for i in range(len(rows))))
        flat = start + cu + tails
        for pages in tables:
            flat += pages + [0] * (m - len(pages))
        return flat, (len(rows), m), max(n for _, n in rows), max(e[0] for e, _ in rows)


__all__ = ["PAGE", "HEAD_DIMS", "KVPool", "KVBatch", "Rope", "kv_append", "kv_attend", "kv_read", "PagedKVCache"]
