"""What a derivative would have to pass: the operators on tensors have none and refuse it."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

recording = torch.is_grad_enabled


def tangents(*tensors) -> bool:
    """Whether forward-mode differentiation goes through any of the tensors (None: no tensor). torch.no_grad() does not end
    it, and such a tensor does not say that it requires a gradient. Callers look at forward_ad._current_level first: 0.05 us of
    a call that takes 10, asked for here 0.2."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
