"""Operators without a backward pass refuse what a gradient would have to pass, instead of dropping it."""
from __future__ import annotations

import pytest
import torch

from bigsmall_amd.fp8 import Fp8Weight


def _weight():
    return torch.zeros(200, 300).to(torch.float8_e4m3fn), torch.ones(2, 3)


def test_weights_whose_scales_or_codes_are_learned():
    codes, scales = _weight()
    learned = torch.nn.Parameter(scales)
    for c, s in ((codes, learned), (codes, learned * 2), (torch.nn.Parameter(codes), scales)):
        with pytest.raises(RuntimeError, match="backward"):
            Fp8Weight(c, s)
        with torch.no_grad():
            w = Fp8Weight(c, s)
        assert not w.scales.requires_grad and not w.codes.requires_grad
        Fp8Weight(c.detach(), s.detach())
