"""The paged 8-bit KV cache on the GPU at the edges of what its calls take."""
from __future__ import annotations

import math

import pytest
import torch

import paged_kv_reference as ref
from paged_kv_reference import PAGE
from test_gpu_paged_kv import Rig, _check_attend, _cpu, _say

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


@pytest.mark.parametrize("start,new", [(100, 1), (5000, 1), (10, 1), (130, 40)])
@pytest.mark.parametrize("tail", [-1, 6])
def test_attend_skips_a_tail_that_does_not_exist(start, new, tail):
    """Single tokens and prompts alike: the rows see the full pages, and no other sequence's tail; the status says so."""
    import bigsmall_amd as bs
    from bigsmall_amd import _native
    from bigsmall_amd.device import StatusWord
    d, hk = 64, 2
    _say("no such tail", start, new, tail)
    rig = Rig([start] * 3, [new] * 3, hk, d, torch.int8, seed=start)
    q = rig.rows(hk * 2)
    tails = rig.batch.tails.clone()
    tails[1, 1] = tail
    batch = bs.KVBatch(rig.batch.start, rig.batch.cu, rig.batch.table, tails, new, start + new)
    st = StatusWord("cuda")
    out, lse = bs.kv_attend(rig.pool, batch, q.cuda(), return_lse=True, status=st)
    assert int(st.t) == _native.BS_DEV_ERR_BOUNDS
    full, mine, pool = (start + new) // PAGE * PAGE, slice(new, 2 * new), _cpu(rig.pool)
    got, got_l = out[mine].cpu().double(), lse[mine].cpu().double()
    if full:
        for i in range(new):                        # every row sees all full pages, as one that stood at their end would
            o, l, tol, ltol = ref.attend(pool, rig.pages[1], rig.tails[1], full - 1, q[mine][i:i + 1], d ** -0.5)
            assert bool(((got[i] - o[0]).abs() <= tol[0]).all()) and bool(((got_l[i] - l[0]).abs() <= ltol[0]).all()), i
    else:
        assert not bool(got.any()) and bool((got_l == -math.inf).all())
    good = bs.kv_attend(rig.pool, rig.batch, q.cuda())           # the others are as ever
    assert torch.equal(out[:new], good[:new]) and torch.equal(out[2 * new:], good[2 * new:])
