"""The paged KV cache's books on the GPU (no reference counterpart).

PagedKVCache keeps on the host which pages belong to which sequence. KVTables keeps it
on the GPU: a step's tables are built there from the lengths, a step may bring drafted
tokens that are taken back later, and nothing waits for the host.

    tables = cache.tables(sequences=64, longest=8192)     # of a PagedKVCache; all its free pages
    step, rows = tables.step(seqs, new, sure, rows=320)   # int32 tensors; step: a KVBatch for append and attend
    tables.keep(step, kept)                               # of each sequence's new tokens the first `kept`
    tables.drop(seqs)                                     # places emptied, pages free
    tables.close()                                        # pages back to the cache's own books

Runs on the current torch stream of the books' device and does not synchronise; the
books are one sequence of calls, so calls on several streams need the usual waits.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from . import _native
from .device import status_ptr
from .paged_kv import PAGE, KVBatch, _tensor

MOST_PLACES = 65536

# bs_kv_tables of include/bigsmall_kv.h
_TABLES = struct.Struct("=8Q3I4x")
assert _TABLES.size == ctypes.sizeof(_native.BsKvTables)

_stream = torch._C._cuda_getCurrentRawStream


class StepRows(NamedTuple):
    """Of each row of a step: its sequence's number in the step (int32), its position (int32), and its slot (int64):
    place * longest + position, where it lies in an array [places, longest]. -1 for rows that no sequence covers."""
    owner: torch.Tensor
    position: torch.Tensor
    slot: torch.Tensor


class KVTables:
    """Books over the page numbers `pages` (int32, each once) for as many places as `tails` has numbers (int32: the
    first of a place's two tails, tails[i] and tails[i] + 1), each of at most `longest` tokens (rounded up to whole pages).

    A place holds one sequence; all are empty at first. State, device int32 tensors: length [places], which [places]
    (0 or 1: the tail it is in), table [places, longest / 64], free [pages] and n_free [1] (the first n_free of `free`
    are free; they are taken from the end)."""

    __slots__ = ("length", "which", "table", "free", "n_free", "tails", "places", "longest", "device", "index", "c", "ref", "_made",
                 "_give_back")

    def __init__(self, pages, tails, longest: int):
        _tensor("pages", pages, torch.int32)
        _tensor("tails", tails, torch.int32, pages.device)
        if pages.dim() != 1 or tails.dim() != 1 or not len(pages) or not 0 < len(tails) <= MOST_PLACES:
            raise ValueError(f"KVTables: pages and tails must be vectors, of at least one page and 1 to {MOST_PLACES} places")
        cols = -(-int(longest) // PAGE)
        if not 0 < cols < 1 << 23:
            raise ValueError(f"KVTables: longest is {longest}")
        if pages.get_device() < 0:
            raise RuntimeError("the paged KV cache's operators run on an AMD GPU (MI355X); the pages are on " + str(pages.device))
        self.device, self.index = pages.device, pages.get_device()
        self.places, self.longest = len(tails), cols * PAGE

        def zeros(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=self.device)

        self.length, self.which, self.table = zeros(self.places), zeros(self.places), zeros(self.places, cols)
        self.free, self.tails = pages.clone(), tails.clone()
        self.n_free = zeros(1).fill_(len(pages))
        self.c = _native.BsKvBooks(*(t.data_ptr() for t in (self.length, self.which, self.table, self.free, self.n_free, self.tails)),
                                   self.places, cols, len(pages))
        self.ref = ctypes.byref(self.c)
        self._made, self._give_back = None, None

    def _vector(self, name, x, n=None):
        if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32:
            raise ValueError(f"{name} must be an int32 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
        shape = x.shape
        if len(shape) != 1 or (n is not None and shape[0] != n):
            raise ValueError(f"{name} has shape {tuple(shape)}, expected [{n if n is not None else 'sequences'}]")
        if x.get_device() != self.index:
            raise ValueError(f"{name} is on {x.device}, the tables are on {self.device}")
        return x if x.is_contiguous() else x.contiguous()

    def _call(self, name, *args):
        index = self.index
        if index == torch.cuda.current_device():
            rc = getattr(_native.lib(), name)(self.ref, *args, _stream(index))
        else:
            with torch.cuda.device(index):
                rc = getattr(_native.lib(), name)(self.ref, *args, _stream(index))
        if rc:
            _native.check(rc, name)

    def step(self, seqs, new, sure=None, *, rows: int, max_new: int | None = None, max_len: int | None = None, status=None):
        """The tables of a step that brings new[b] tokens to the sequence in place seqs[b] (int32 tensors; each place
        once). Returns a KVBatch whose sequences are seqs, in that order, packed into `rows` rows (more than are
        needed may be given: the rest belong to no sequence), and their StepRows.

        sure (int32): how many of the new tokens are certain; None: all. The others may be taken back by `keep`, so a
        sequence gets no more of them than complete no page (which is quantised once): its number of new tokens is the
        difference of the KVBatch's cu. max_new, max_len: as KVBatch takes them (rows and longest by default).

        The books stay as they are until `keep`, which reads seqs and sure again; another step made before it replaces this one. All or nothing: where
        pages, rows or a place's length do not suffice (status, a device.StatusWord, gets BS_DEV_ERR_COUNT), or places do
        not exist or are named twice or numbers are negative (BS_DEV_ERR_BOUNDS), no sequence has a new token."""
        seqs = self._vector("seqs", seqs)
        b = seqs.shape[0]
        if not 0 < b <= min(self.places, 65535):
            raise ValueError(f"a step of {b} sequences; the tables have {self.places} places" + ("" if self.places else " (closed)"))
        new = self._vector("new", new, b)
        if sure is not None:
            sure = self._vector("sure", sure, b)
        max_new, max_len = rows if max_new is None else int(max_new), self.longest if max_len is None else int(max_len)
        if not (0 <= rows < 1 << 30 and 0 <= max_new < 1 << 30 and 0 <= max_len < 1 << 30):
            raise ValueError(f"rows {rows}, max_new {max_new} and max_len {max_len} must be 0 or more, below 2^30")
        cols = self.longest // PAGE
        small = 4 * b + 1 + b * cols
        # one allocation: slot first, which wants 8 bytes, then the tables, then owner and position
        flat = torch.empty(4 * rows + small, dtype=torch.int32, device=self.device)
        slot, start, cu, tails, table, owner, position = flat.split_with_sizes((2 * rows, b, b + 1, 2 * b, b * cols, rows, rows))
        at = flat.data_ptr()
        start_at = at + 8 * rows
        cu_at = start_at + 4 * b
        tails_at = cu_at + 4 * (b + 1)
        table_at = tails_at + 8 * b
        owner_at = at + 8 * rows + 4 * small
        batch = KVBatch.__new__(KVBatch)
        batch._set(start, cu, table.view(b, cols), tails.view(b, 2), b, cols, cols, max_new, max_len, rows, self.index, start_at, cu_at,
                   table_at, tails_at)
        c = _TABLES.pack(seqs.data_ptr(), start_at, cu_at, tails_at, table_at, owner_at, owner_at + 4 * rows, at, b, rows, max_new)
        self._call("bs_kv_books_step", c, new.data_ptr(), sure.data_ptr() if sure is not None else 0, status_ptr(status, self.index))
        self._made = (batch, c, seqs, sure)
        return batch, StepRows(owner, position, slot.view(torch.int64))

    def keep(self, step: KVBatch, kept=None) -> None:
        """Enter the step that was made last into the books, once: of each sequence's new tokens the first kept[b]
        (int32; None: all of them) stay, held to what is certain and to what there is. RuntimeError for another step."""
        if self._made is None or self._made[0] is not step:
            raise RuntimeError("not the step that these tables made last, or it is kept already")
        _, c, _, sure = self._made
        if kept is not None:
            kept = self._vector("kept", kept, step.n_seqs)
        self._call("bs_kv_books_keep", c, sure.data_ptr() if sure is not None else 0,
                   kept.data_ptr() if kept is not None else 0)
        self._made = None

    def drop(self, seqs, status=None) -> None:
        """Empty the places seqs (int32); their pages are free for steps made from now on. All or nothing: no place is
        emptied where one does not exist or is named twice (BS_DEV_ERR_BOUNDS)."""
        seqs = self._vector("seqs", seqs)
        if seqs.shape[0] > self.places:
            raise ValueError(f"{seqs.shape[0]} places; the tables have {self.places}")
        word = status_ptr(status, self.index)
        self._made = None
        self._call("bs_kv_books_drop", seqs.data_ptr(), seqs.shape[0], word)

    def lent_by(self, give_back) -> None:
        """give_back() is called by close()."""
        self._give_back = give_back

    def close(self) -> None:
        """Give pages and tails back to the cache that lent them. Sequences in the tables end with it, and steps are refused."""
        give, self._give_back = self._give_back, None
        self._made, self.places = None, 0
        if give is not None:
            give()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


__all__ = ["MOST_PLACES", "KVTables", "StepRows"]
