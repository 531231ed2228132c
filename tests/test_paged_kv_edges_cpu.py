"""The paged KV cache's host side at the edges of what its calls take."""
from __future__ import annotations

import pytest
import torch

from bigsmall_amd.paged_kv import KVPool, kv_append, kv_attend
from test_paged_kv_cpu import _batch, _parts, on_gpu  # noqa: F401 (a fixture)


def test_calls_refuse_rows_that_are_not_the_steps(on_gpu):
    pool, batch = KVPool(*_parts()), _batch(total=2)
    for n in (0, 1, 3):
        x = torch.zeros(n, 2, 64, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_append(pool, batch, x, x, x)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_append(pool, batch, None, x, x)
        with pytest.raises(ValueError, match="the step has 2"):
            kv_attend(pool, batch, x)
