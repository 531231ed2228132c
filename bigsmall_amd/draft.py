"""Verification of drafted tokens (no reference counterpart).

A cheap guess proposes the next few tokens of each sequence; the model computes its
distributions after all of them in one step, and `draft_verify` keeps as many drafts as
agree with them, so that the tokens come out distributed as if the model had drawn each.

Runs on the current torch stream of p's device and does not synchronise; the work area
comes from torch's allocator for each call.
"""
from __future__ import annotations

import struct

import torch

from . import _native
from .device import status_ptr

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_DRAFTS = 1024
_BATCH = struct.Struct("=8Q2q5I4x")

_stream = torch._C._cuda_getCurrentRawStream


def _vector(name, x, n, dtype, index):
    """x as a contiguous vector of n numbers on device `index` (n None: any number)."""
    if not isinstance(x, torch.Tensor) or x.dtype is not dtype:
        raise ValueError(f"{name} must be a {dtype} tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    shape = x.shape
    if len(shape) != 1 or (n is not None and shape[0] != n):
        raise ValueError(f"{name} has shape {tuple(shape)}, expected [{n if n is not None else 'sequences + 1'}]")
    if x.get_device() != index:
        raise ValueError(f"{name} is on {x.device}, p is not")
    return x if x.is_contiguous() else x.contiguous()


def _rows(name, x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES:
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    shape = x.shape
    if len(shape) != 2 or not 1 <= shape[1] <= 1 << 30 or shape[0] > 1 << 30:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected [rows, vocabulary]")
    return x if x.stride(1) == 1 or shape[1] == 1 else x.contiguous()


def draft_verify(p, draft, cu, accept, pick, q=None, max_drafts=None, status=None):
    """Which drafted tokens stay, and the token after them. Returns tokens int64 [B, max_drafts + 1] (the drafts
    taken, the token drawn, then -1) and counts int32 [B] (how many tokens those are).

    p [T, vocab]     the target's probabilities after each row's token (f32, bf16 or f16). The draw does not depend on a row's sum,
                     taking a draft does: tokens follow p only if its rows, and q's, add up to 1
    draft [T] int64  the token proposed to follow each row
    cu [B + 1] int32 sequence b has the rows cu[b] .. cu[b + 1] - 1, one more than drafts; its last row's draft,
                     accept and q are not read. A sequence without rows gets no token and count 0
    accept [T], pick [B] f32   random numbers in [0, 1)
    q [T, vocab]     the probabilities that the drafts were drawn from, of p's type; None: they were not drawn
    max_drafts       the most that a sequence has, up to 1,024 (by default T - B, held to 0 and 1,024: enough where every sequence
                     has a row; say it where some have none)

    Draft x is taken while accept * q[x] < p[x] (without q: accept < p[x]). Then one token is drawn: where a draft was
    refused from max(p - q, 0) of its row (without q: from p without the draft), after the last one from p. It is the first
    at which the sum of the weights up to it exceeds pick times their whole sum, in 64 bits. Weights that are no
    numbers count as 0; if nothing is left it is drawn from p.

    status: a device.StatusWord that gets BS_DEV_ERR_BOUNDS where rows do not exist or are more than max_drafts + 1 (the
    sequence gets no token) or a draft is no token (it is refused), and BS_DEV_ERR_COUNT where p's row has no
    probability at all (the token is 0)."""
    p = _rows("p", p)
    index, (t, vocab) = p.get_device(), p.shape
    qp = q_stride = 0
    if q is not None:
        q = _rows("q", q)
        if q.dtype is not p.dtype or q.shape != p.shape or q.get_device() != index:
            raise ValueError(f"q is {q.dtype} {tuple(q.shape)} on {q.device}, p {p.dtype} {tuple(p.shape)} on {p.device}")
        qp, q_stride = q.data_ptr(), q.stride(0)
    draft = _vector("draft", draft, t, torch.int64, index)
    accept = _vector("accept", accept, t, torch.float32, index)
    cu = _vector("cu", cu, None, torch.int32, index)
    b = cu.shape[0] - 1
    if not 0 <= b <= 1 << 20:
        raise ValueError(f"cu has {b + 1} numbers, expected 1 to {(1 << 20) + 1}")
    pick = _vector("pick", pick, b, torch.float32, index)
    if max_drafts is None:
        max_drafts = min(max(0, t - b), MOST_DRAFTS)
    if not 0 <= max_drafts <= MOST_DRAFTS:
        raise ValueError(f"max_drafts must be 0 to {MOST_DRAFTS}, got {max_drafts}")
    word = status_ptr(status, index)
    if index < 0:
        raise RuntimeError(f"draft_verify runs on an AMD GPU (MI355X); p is on {p.device}")
    device = p.device
    tokens = torch.empty((b, max_drafts + 1), dtype=torch.int64, device=device)
    counts = torch.empty(b, dtype=torch.int32, device=device)
    if b:
        L = _native.lib()
        n = L.bs_draft_verify_work_bytes(b, vocab)
        work = torch.empty(n, dtype=torch.uint8, device=device) if n else None
        batch = _BATCH.pack(p.data_ptr(), qp, draft.data_ptr(), accept.data_ptr(), cu.data_ptr(),
                            pick.data_ptr(), tokens.data_ptr(), counts.data_ptr(), p.stride(0), q_stride,
                            _TYPES[p.dtype], t, vocab, b, max_drafts)
        args = batch, work.data_ptr() if n else 0, n, word
        if index == torch.cuda.current_device():
            rc = L.bs_draft_verify(*args, _stream(index))
        else:
            with torch.cuda.device(index):
                rc = L.bs_draft_verify(*args, _stream(index))
        if rc:
            _native.check(rc, "bs_draft_verify")
    return tokens, counts


__all__ = ["MOST_DRAFTS", "draft_verify"]
