"""The paged 8-bit KV cache on the GPU at the edges of what its calls take."""
from __future__ import annotations

import pytest
import torch

from paged_kv_reference import PAGE
from test_gpu_paged_kv import Rig, _check_attend, _say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,starts,claimed", [(64, [129 * PAGE - 20], 128), (64, [155 * PAGE - 1], 128), (128, [41 * PAGE - 63], 40),
                                              (64, [51 * PAGE - 30], 40), (64, [51 * PAGE - 7, 45 * PAGE - 40], 40),
                                              (256, [129 * PAGE - 5, 40], 128)])
def test_unfinished_page_counts_once_when_the_batch_says_too_little(d, starts, claimed):
    """Caches of more pages than the batch says, split, the last page unfinished: some parts are left without pages."""
    import bigsmall_amd as bs
    _say("too little", d, starts, claimed)
    rig = Rig(starts, [1] * len(starts), 2, d, torch.int8, seed=claimed + d)
    rig.pool.v_tail.mul_(3.0)                       # a tail counted twice is far off
    q = rig.rows(4)
    batch = bs.KVBatch(rig.batch.start, rig.batch.cu, rig.batch.table, rig.batch.tails, 1, claimed * PAGE)
    out, lse = bs.kv_attend(rig.pool, batch, q.cuda(), return_lse=True)
    _check_attend(rig, q, out, lse, d ** -0.5)
