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


def _capped(pool, pages, tail, start, q, scale, cap):
    """ref.attend for causal rows with a cap, its bound without the cap in it: a score before the cap is off by at most
    2^-20 of the sum A of its terms' absolute values, which the cap (slope 1 at most) does not widen, and cap * tanh by
    2^-20 of its own value, which is A at most, again."""
    n, hq, d = q.shape
    hk = pool[0].shape[1]
    group, length = hq // hk, start + n
    see = torch.arange(length)[None] <= start + torch.arange(n)[:, None]
    out, tol = torch.zeros(2, n, hq, d, dtype=torch.float64)
    lse, off = torch.zeros(2, n, hq, dtype=torch.float64)
    for head in range(hq):
        k, v = ref.cached(pool, pages, tail, length, head // group)
        x = cap * torch.tanh((q[:, head].double() @ k.T) * scale / cap)
        a = (q[:, head].double().abs() @ k.abs().T) * abs(scale)
        lse[:, head] = torch.logsumexp(x.masked_fill(~see, -math.inf), 1)
        w = torch.exp(x - lse[:, head, None]).masked_fill(~see, 0.0)
        off[:, head] = 2.0 ** -20 * (2 * a.masked_fill(~see, 0.0).amax(1) + 16)
        out[:, head] = w @ v
        tol[:, head] = 2.0 ** -8 * out[:, head].abs() + (2.0 ** -11 + 2 * off[:, head, None]) * (w @ v.abs()) + \
            2.0 ** -36 * w.amax(1, keepdim=True) * (see.double() @ v.abs())
    return out, lse, tol, off


@pytest.mark.parametrize("cap", [0.25, 50.0, 100.0, 1000.0, 1e4, 1e5, 1e9, 1e30, 1e60, 1e-50])
@pytest.mark.parametrize("starts,news,d,scale", [([700, 64, 13], [1, 1, 1], 64, 0.125), ([300, 0, 5], [90, 65, 1], 64, 0.125),
                                                 ([300, 20], [70, 1], 256, 0.3), ([500, 3], [2, 1], 128, -1.0)])
def test_caps_of_every_size(cap, starts, news, d, scale):
    """Scores far below the cap come out as they went in, not off by the cap's own rounding; scores above it are held."""
    import bigsmall_amd as bs
    _say("cap", cap, starts, news, d, scale)
    rig = Rig(starts, news, 1, d, torch.int8, seed=d)
    q = rig.rows(2)
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), scale=scale, softcap=cap, return_lse=True)
    pool, out, lse = _cpu(rig.pool), out.cpu().double(), lse.cpu().double()
    for b, n in enumerate(news):
        at = slice(int(rig.cu[b]), int(rig.cu[b]) + n)
        o, l, tol, ltol = _capped(pool, rig.pages[b], rig.tails[b], starts[b], q[at], scale, cap)
        assert bool(((lse[at] - l).abs() <= ltol).all()), (b, float(((lse[at] - l).abs() / ltol).max()))
        assert bool(((out[at] - o).abs() <= tol).all()), (b, float(((out[at] - o).abs() / tol.clamp(min=1e-30)).max()))


def test_cache_refuses_rows_that_are_not_the_steps():
    """Fewer or more rows than a step has: refused before anything is written; numbers that do not exist reach a status."""
    import bigsmall_amd as bs
    from bigsmall_amd.device import StatusWord
    cache = bs.PagedKVCache(1, 1, 64, pages=4, sequences=2)
    a, b = cache.add(), cache.add()
    step = cache.step({a: 3, b: 2})
    x = torch.ones(7, 1, 64, dtype=torch.bfloat16, device="cuda")
    for n in (0, 3, 4, 6, 7):
        with pytest.raises(ValueError, match="5"):
            cache.append(0, step, None, x[:n], x[:n])
        with pytest.raises(ValueError, match="5"):
            cache.attend(0, step, x[:n])
    assert not bool(cache.pools[0].k_tail.any())
    st = StatusWord("cuda")
    out = torch.empty(5, 1, 64, dtype=torch.bfloat16, device="cuda")
    assert cache.append(0, step, x[:5], x[:5], x[:5], out=out, status=st) is out and torch.equal(out, x[:5])
    k, v = cache.read(0, a, status=st)
    assert torch.equal(k[0], x[:3, 0]) and torch.equal(v[0], x[:3, 0]) and int(st.t) == 0


@pytest.mark.parametrize("bad", [[66], [3], [64, 127, 129], list(range(64, 130))])
def test_append_reports_any_sequence_of_a_long_step(bad):
    """Starts that make no sense, wherever they stand in a step of 130 sequences: reported, and the others appended."""
    import bigsmall_amd as bs
    from bigsmall_amd import _native
    from bigsmall_amd.device import StatusWord
    n, d = 130, 64
    rig = Rig([5] * n, [1] * n, 1, d, torch.int8, seed=6)
    k, v = rig.rows(1), rig.rows(1)
    start = rig.batch.start.clone()
    start[bad] = 1 << 28
    st = StatusWord("cuda")
    before = _cpu(rig.pool)
    bs.kv_append(rig.pool, rig.batch, None, k.cuda(), v.cuda(), status=st)
    assert int(st.t) == 0
    rig.pool.k_tail.copy_(before[4])
    batch = bs.KVBatch(start, rig.batch.cu, rig.batch.table, rig.batch.tails, 1, 6)
    bs.kv_append(rig.pool, batch, None, k.cuda(), v.cuda(), status=st)
    assert int(st.t) == _native.BS_DEV_ERR_BOUNDS
    after = rig.pool.k_tail.cpu()
    for b in range(n):
        want = before[4][rig.tails[b]].clone()
        if b not in bad:
            want[:, 5] = k[b]
        assert torch.equal(after[rig.tails[b]].view(torch.uint8), want.view(torch.uint8)), b


@pytest.mark.parametrize("unaligned", [False, True])
def test_strides_of_dimensions_of_one(unaligned):
    """One token, or one head, out of a wider buffer: the stride of a dimension of one says nothing and is not looked at."""
    import bigsmall_amd as bs
    hk, group, d = 2, 4, 128
    rig = Rig([70], [1], hk, d, torch.int8, seed=1)
    rope = bs.Rope.from_theta(d, 100)
    rows = rig.rows(hk * group + 2 * hk).cuda()
    wide = torch.zeros(2, rows.shape[1] * d + 3, dtype=torch.bfloat16, device="cuda")
    at = int(unaligned)
    one = wide[:, :-3].unflatten(1, (-1, d))[at:at + 1]
    one.copy_(rows)
    q, k, v = one.split([hk * group, hk, hk], 1)
    assert q.stride(0) % 8 and q.is_contiguous() and bool(q.data_ptr() % 16) == unaligned
    want = bs.kv_append(rig.pool, rig.batch, q.clone(), k.clone(), v.clone(), rope)
    want_tails = rig.pool.k_tail.clone()
    rig.pool.k_tail[rig.tails[0], :, 70 % PAGE] = 0
    got = bs.kv_append(rig.pool, rig.batch, q, k, v, rope)
    assert torch.equal(got, want) and torch.equal(rig.pool.k_tail.view(torch.uint8), want_tails.view(torch.uint8))
    if not unaligned:
        wide_out = torch.empty_like(wide)
        out = wide_out[:, :-3].unflatten(1, (-1, d))[:1, :hk * group]
        assert bs.kv_append(rig.pool, rig.batch, q, k, v, rope, out=out) is out and torch.equal(out, want)
    assert torch.equal(bs.kv_attend(rig.pool, rig.batch, q), bs.kv_attend(rig.pool, rig.batch, q.clone()))
    # one head whose stride is odd
    rig = Rig([70], [3], 1, d, torch.int8, seed=2)
    x = rig.rows(1).cuda()
    odd = x.as_strided(x.shape, (d, 5, 1))
    assert torch.equal(bs.kv_attend(rig.pool, rig.batch, odd), bs.kv_attend(rig.pool, rig.batch, x))


@pytest.mark.parametrize("cap", [40.0, 100.0, 2000.0])
@pytest.mark.parametrize("starts,news,d,scale", [([700, 64, 13], [1, 3, 1], 64, 0.125), ([300, 0, 5], [90, 65, 1], 80, -0.4), ([300, 20], [70, 1], 256, 0.3)])
def test_large_caps_beside_biases_and_masks(cap, starts, news, d, scale):
    import bigsmall_amd as bs
    _say("cap and masks", cap, starts, news, d, scale)
    rig = Rig(starts, news, 2, d, torch.float8_e4m3fn, seed=d + 1)
    q = rig.rows(4)
    pos = torch.cat([s + torch.arange(n) for s, n in zip(starts, news)])
    options = dict(softcap=cap, slopes=torch.tensor([0.5, 0.0, 0.25, 0.01]), window=130, first=(pos // 37 * 37).to(torch.int32),
                   prefix=torch.tensor([40, 100, 3][:len(starts)], dtype=torch.int32))
    gpu = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), scale=scale, return_lse=True, **gpu)
    _check_attend(rig, q, out, lse, scale, **options)
