"""Operators without a backward pass refuse what a gradient would have to pass, instead of dropping it."""
from __future__ import annotations

import pytest
import torch

from bigsmall_amd.fp8 import Fp8Weight
from test_paged_kv_cpu import _batch, _parts, on_gpu  # noqa: F401 (a fixture)


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


def test_dual_tensors_are_refused(on_gpu, monkeypatch):  # noqa: F811
    """Forward-mode differentiation goes on under torch.no_grad() and marks no tensor as requiring a gradient."""
    from torch.autograd import forward_ad

    from bigsmall_amd import fp8
    from bigsmall_amd.fp8 import fp8_linear, fp8_quantise
    from bigsmall_amd.paged_kv import KVPool, kv_append, kv_attend
    monkeypatch.setattr(fp8, "_gpu", lambda index, what: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    codes, scales = _weight()
    weight = Fp8Weight(codes, scales)
    pool, batch = KVPool(*_parts()), _batch()
    x, wide, slopes = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 300, dtype=torch.bfloat16), torch.zeros(2)

    def calls(d):
        return (lambda: Fp8Weight(codes, d(scales)), lambda: fp8_quantise(d(wide)), lambda: fp8_linear(d(wide), weight),
                lambda: kv_append(pool, batch, d(x), x, x), lambda: kv_append(pool, batch, x, d(x), x), lambda: kv_append(pool, batch, None, x, d(x)),
                lambda: kv_attend(pool, batch, d(x)), lambda: kv_attend(pool, batch, x, slopes=d(slopes)))

    with forward_ad.dual_level():
        for grad in (True, False):
            for call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
                with pytest.raises(RuntimeError, match="no derivative forwards"), torch.set_grad_enabled(grad):
                    call()
        # others pass as outside of it: on to the library, which here has nothing to call
        for call in calls(lambda t: t)[1:]:
            with pytest.raises(AssertionError, match="was called"):
                call()
