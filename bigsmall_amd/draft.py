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

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_DRAFTS = 1024
_BATCH = struct.Struct("=8Q2q5I4x")

_stream = torch._C._cuda_getCurrentRawStream


def _vector(name, x, n, dtype, device):
    if not isinstance(x, torch.Tensor) or x.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if x.dim() != 1 or (n is not None and x.shape[0] != n):
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected [{n if n is not None else 'sequences + 1'}]")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, p on {device}")
    return x if x.is_contiguous() else x.contiguous()


def _rows(name, x, shape, dtype, device):
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{name} must be a {dtype or 'float32, bfloat16 or float16'} tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if x.dim() != 2 or (shape is not None and x.shape != shape) or not 1 <= x.shape[1] <= 1 << 30:
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {tuple(shape) if shape is not None else '[rows, vocabulary]'}")
    if device is not None and x.device != device:
        raise ValueError(f"{name} is on {x.device}, p on {device}")
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def draft_verify(p, draft, cu, accept, pick, q=None, max_drafts=None, status=None):
    """Which drafted tokens stay, and the token after them. Returns tokens int64 [B, max_drafts + 1] (the drafts
    taken, the token drawn, then -1) and counts int32 [B] (how many tokens those are).

    p [T, vocab]     the target's probabilities after each row's token (f32, bf16 or f16; they need not add up to 1)
    draft [T] int64  the token proposed to follow each row
    cu [B + 1] int32 sequence b has the rows cu[b] .. cu[b + 1] - 1, one more than drafts; its last row's draft,
                     accept and q are not read. A sequence without rows gets no token and count 0
    accept [T], pick [B] f32   random numbers in [0, 1)
    q [T, vocab]     the probabilities that the drafts were drawn from, of p's type; None: they were not drawn
    max_drafts       the most that a sequence has (by default T - B, or 0)

    Draft x is taken while accept * q[x] < p[x] (without q: accept < p[x]). Then one token is drawn: where a draft was
    refused from max(p - q, 0) of its row (without q: from p without the draft), after the last one from p. It is the first
    at which the sum of the weights up to it exceeds pick times their whole sum, in 64 bits. Weights that are no
    numbers count as 0; if nothing is left it is drawn from p.

    status: a device.StatusWord that gets BS_DEV_ERR_BOUNDS where rows do not exist or are more than max_drafts + 1 (the
    sequence gets no token) or a draft is no token (it is refused), and BS_DEV_ERR_COUNT where p's row has no
    probability at all (the token is 0)."""
    p = _rows("p", p, None, None, None)
    index, device, (t, vocab) = p.get_device(), p.device, p.shape
    if q is not None:
        q = _rows("q", q, p.shape, p.dtype, device)
    draft = _vector("draft", draft, t, torch.int64, device)
    accept = _vector("accept", accept, t, torch.float32, device)
    cu = _vector("cu", cu, None, torch.int32, device)
    b = cu.shape[0] - 1
    if not 0 <= b <= 1 << 20:
        raise ValueError(f"cu has {b + 1} numbers, expected 1 to {(1 << 20) + 1}")
    pick = _vector("pick", pick, b, torch.float32, device)
    if max_drafts is None:
        max_drafts = min(max(0, t - b), MOST_DRAFTS)
    if not 0 <= max_drafts <= MOST_DRAFTS:
        raise ValueError(f"max_drafts must be 0 to {MOST_DRAFTS}, got {max_drafts}")
    if t > 1 << 30:
        raise ValueError(f"{t} rows: at most {1 << 30}")
    if index < 0:
        raise RuntimeError(f"draft_verify runs on an AMD GPU (MI355X); p is on {device}")
    tokens = torch.empty((b, max_drafts + 1), dtype=torch.int64, device=device)
    counts = torch.empty((b,), dtype=torch.int32, device=device)
    if b:
        L = _native.lib()
        n = L.bs_draft_verify_work_bytes(b, vocab)
        work = torch.empty(n, dtype=torch.uint8, device=device)
        batch = _BATCH.pack(p.data_ptr(), q.data_ptr() if q is not None else 0, draft.data_ptr(), accept.data_ptr(), cu.data_ptr(),
                            pick.data_ptr(), tokens.data_ptr(), counts.data_ptr(), p.stride(0), q.stride(0) if q is not None else 0,
                            _TYPES[p.dtype], t, vocab, b, max_drafts)
        with torch.cuda.device(index):
            rc = L.bs_draft_verify(batch, work.data_ptr(), n, status.ptr if status else None, _stream(index))
        if rc:
            _native.check(rc, "bs_draft_verify")
    return tokens, counts


__all__ = ["MOST_DRAFTS", "draft_verify"]
