"""The paged 8-bit KV cache on the GPU against its definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import paged_kv_reference as ref
from paged_kv_reference import PAGE, QMAX

pytestmark = pytest.mark.gpu

KINDS = [torch.int8, torch.float8_e4m3fn]


def _say(*a):
    print(*a, flush=True)


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _bf16(shape, g, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)


def _cpu(pool):
    return [getattr(pool, n).cpu() for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")]


class Rig:
    """A pool with random contents and one step over sequences of given lengths."""

    def __init__(self, starts, news, hk, d, kind, seed=0, extra_pages=5, junk=True):
        import bigsmall_amd as bs
        g = _gen(seed)
        self.starts, self.news = starts, news
        b = len(starts)
        ends = [s + n for s, n in zip(starts, news)]
        need = [(e + PAGE - 1) // PAGE for e in ends]
        m = max(1, max(need))
        pages = sum(need) + extra_pages
        perm = torch.randperm(pages, generator=g).tolist()
        self.pages = []
        for n in need:
            self.pages.append([perm.pop() for _ in range(n)])
        table = torch.full((b, m), -7, dtype=torch.int32)          # entries that no token needs are no page
        for i, p in enumerate(self.pages):
            table[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
            if ends[i] % PAGE:
                table[i, len(p) - 1] = -9                          # an unfinished page has no page yet
        tails = torch.randperm(2 * b, generator=g).view(b, 2).to(torch.int32)
        for i in range(b):
            if ends[i] // PAGE == starts[i] // PAGE:
                tails[i, 1] = tails[i, 0]
        self.tail_in, self.tails = tails[:, 0].tolist(), tails[:, 1].tolist()
        q = QMAX[kind]
        x = (torch.randn(2, pages, hk, PAGE * d, generator=g) * q / 4).clamp(-q, q)
        x = x.round().to(torch.int8) if kind == torch.int8 else x.to(kind)
        scale = (0.5 + torch.rand(2, pages, hk, generator=g)) * 4 / q
        kt, vt = _bf16((2 * b, hk, PAGE, d), g), _bf16((2 * b, hk, d, PAGE), g)
        if junk:            # what lies after a sequence's end may be anything
            for i in range(b):
                used = ends[i] % PAGE if tails[i, 0] == tails[i, 1] else starts[i] % PAGE
                kt[tails[i, 0], :, used:] = math.nan
                vt[tails[i, 0], :, :, used:] = math.nan
                if tails[i, 0] != tails[i, 1]:
                    kt[tails[i, 1], :, ends[i] % PAGE:] = math.inf
                    vt[tails[i, 1], :, :, ends[i] % PAGE:] = -math.inf
        self.pool = bs.KVPool(x[0].view(pages, hk, PAGE, d).cuda(), x[1].view(pages, hk, d, PAGE).cuda(), scale[0].cuda(),
                              scale[1].cuda(), kt.cuda(), vt.cuda())
        self.start = torch.tensor(starts, dtype=torch.int32)
        self.cu = torch.tensor([0] + news).cumsum(0).to(torch.int32)
        self.batch = bs.KVBatch(self.start.cuda(), self.cu.cuda(), table.cuda(), tails.cuda(), max(news), max(ends))
        self.total, self.g, self.table = sum(news), g, table

    def rows(self, heads, scale=1.0):
        return _bf16((self.total, heads, self.pool.head_dim), self.g, scale)


def _check_attend(rig, q, out, lse, scale, **options):
    pool = _cpu(rig.pool)
    prefix, first = options.pop("prefix", None), options.pop("first", None)
    out, lse = out.cpu().double(), lse.cpu().double()
    for b, n in enumerate(rig.news):
        if not n:
            continue
        at = slice(int(rig.cu[b]), int(rig.cu[b]) + n)
        o, l, tol, ltol = ref.attend(pool, rig.pages[b], rig.tails[b], rig.starts[b], q[at], scale,
                                     prefix=int(prefix[b]) if prefix is not None else 0,
                                     first=first[at] if first is not None else None, **options)
        assert torch.equal(torch.isnan(out[at]), torch.isnan(o)), (b, "NaN")
        off = (out[at] - o).abs() - tol
        assert not bool((off > 0).any()), (b, float(off.nan_to_num(-1).max()))
        assert torch.equal(lse[at] == -math.inf, l == -math.inf), (b, "rows that see nothing")
        seen = l != -math.inf
        off = ((lse[at] - l).abs() - ltol)[seen]
        assert not bool((off > 0).any()), (b, "lse", float(off.nan_to_num(-1).max()))


# ---- append

def _turned(rig, x, rope, interleaved, fn):
    out = []
    for b, n in enumerate(rig.news):
        for i in range(n):
            t, pos = int(rig.cu[b]) + i, rig.starts[b] + i
            out.append(fn(x[t], rope[0][pos], rope[1][pos], interleaved))
    return torch.stack(out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,group,rot,interleaved", [(64, 1, 64, False), (80, 2, 40, True), (80, 3, 40, False), (96, 4, 96, False),
                                                     (128, 4, 128, False), (128, 1, 64, True), (256, 2, 256, False), (256, 1, 8, False)])
def test_append_matches_the_definition(kind, d, group, rot, interleaved):
    import bigsmall_amd as bs
    _say("append", kind, d, group, rot, interleaved)
    starts, news = [0, 63, 64, 1, 60, 0, 127, 10, 0, 191], [1, 1, 1, 63, 70, 200, 1, 5, 64, 130]
    hk = 2
    rig = Rig(starts, news, hk, d, kind, seed=d + rot)
    q, k, v = rig.rows(hk * group), rig.rows(hk), rig.rows(hk, 3.0)
    v[5] = 0                                              # zeros among them
    rope = bs.Rope.from_theta(rot, 400, 10000.0, interleaved)
    angles = (rope.cos.cpu(), rope.sin.cpu())
    before = _cpu(rig.pool)
    got = bs.kv_append(rig.pool, rig.batch, q.cuda(), k.cuda(), v.cuda(), rope).cpu().double()
    after = _cpu(rig.pool)
    # q: bit for bit the f32 definition, and one rounding to 8 bits away from 64 bits
    assert torch.equal(got, _turned(rig, q, angles, interleaved, ref.rotate32).double())
    want = _turned(rig, q, angles, interleaved, ref.rotate)
    size = q.double().abs().amax(-1, keepdim=True)
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * size).all())
    kr = _turned(rig, k, angles, interleaved, ref.rotate32)
    pages_written = set()
    qmax = QMAX[kind]
    for b, n in enumerate(news):
        s, e = starts[b], starts[b] + n
        for p in range(s // PAGE, (e - 1) // PAGE + 1):
            lo, hi = max(s, p * PAGE), min(e, (p + 1) * PAGE)
            rows = slice(int(rig.cu[b]) + lo - s, int(rig.cu[b]) + hi - s)
            new_k, new_v = kr[rows].transpose(0, 1), v[rows].transpose(0, 1)       # [hk, n, d]
            if (p + 1) * PAGE <= e:
                page = rig.pages[b][p]
                pages_written.add(page)
                cut = lo - p * PAGE
                old = rig.tail_in[b]
                full_k = torch.cat([before[4][old, :, :cut], new_k], 1)
                full_v = torch.cat([before[5][old, :, :, :cut].transpose(1, 2), new_v], 1)
                for name, x, codes, scales in (("k", full_k, after[0][page], after[2][page]),
                                               ("v", full_v, after[1][page].transpose(1, 2), after[3][page])):
                    for h in range(hk):
                        want_codes, want_scale = ref.quantise32(x[h], kind)
                        assert float(scales[h]) == float(want_scale), (b, p, name, h)
                        assert torch.equal(codes[h].double() if kind == torch.int8 else codes[h].float(),
                                           want_codes.double() if kind == torch.int8 else want_codes.float()), (b, p, name, h)
                        # and in 64 bits: within half a step of the value, three f32 roundings aside
                        y, sc = ref.values(codes[h], scales[h]), float(scales[h])
                        half = torch.full_like(y, sc / 2) if kind == torch.int8 else (y.abs() / 15).clamp(min=sc * 2.0 ** -10)
                        assert bool(((y - x[h].double()).abs() <= half + 3 * 2.0 ** -24 * qmax * sc).all()), (b, p, name, h)
            else:
                tail = rig.tails[b]
                cut = slice(lo - p * PAGE, hi - p * PAGE)
                assert torch.equal(after[4][tail, :, cut], new_k) and torch.equal(after[5][tail, :, :, cut].transpose(1, 2), new_v)
                if lo > p * PAGE:                     # what was there before stays
                    assert torch.equal(after[4][tail, :, :lo - p * PAGE], before[4][rig.tail_in[b], :, :lo - p * PAGE])
    keep = [p for p in range(before[0].shape[0]) if p not in pages_written]
    for x, y in zip(before[:4], after[:4]):
        assert torch.equal(x[keep].view(torch.uint8), y[keep].view(torch.uint8))
    # again: the same bytes
    again = bs.kv_append(rig.pool, rig.batch, q.cuda(), k.cuda(), v.cuda(), rope).cpu().double()
    assert torch.equal(again, got)
    for x, y in zip(after, _cpu(rig.pool)):
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", KINDS)
def test_cache_does_not_depend_on_the_chunks(kind):
    import bigsmall_amd as bs
    g = _gen(5)
    n, hk, d = 300, 2, 128
    q, k, v = (_bf16((n, h, d), g).cuda() for h in (4, hk, hk))
    rope = bs.Rope.from_theta(d, n)
    seen = []
    for chunks in ([300], [1] * 300, [64, 64, 64, 64, 44], [63, 2, 130, 1, 104], [299, 1]):
        cache = bs.PagedKVCache(1, hk, d, pages=8, sequences=2, kind=kind)
        other, seq, at, rotated = cache.add(), cache.add(), 0, []
        for c in chunks:
            step = cache.step({seq: c})
            rotated.append(cache.append(0, step, q[at:at + c], k[at:at + c], v[at:at + c], rope))
            at += c
        assert cache.length(seq) == n
        seen.append((torch.cat(rotated), *cache.read(0, seq)))
    for s in seen[1:]:
        for a, b in zip(seen[0], s):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
def test_append_extremes(kind):
    """Pages of zeros, of the smallest and of huge values: finite scales, values within a step or held to 2^60."""
    import bigsmall_amd as bs
    x = torch.zeros(PAGE * 5, 1, 64, dtype=torch.bfloat16)
    x[PAGE:2 * PAGE] = 2.0 ** -130
    x[2 * PAGE:3 * PAGE] = 2.0 ** 100
    x[3 * PAGE:4 * PAGE] = -(2.0 ** -20)
    x[4 * PAGE:] = 3.0e38
    cache = bs.PagedKVCache(1, 1, 64, pages=8, sequences=1, kind=kind)
    seq = cache.add()
    cache.append(0, cache.step({seq: 5 * PAGE}), None, x.cuda(), (-x).cuda())
    assert bool(torch.isfinite(cache.pools[0].k_scale).all()) and bool((cache.pools[0].v_scale[:5] >= 0).all())
    k, v = cache.read(0, seq)
    for y, sign in ((k.cpu().double(), 1), (v.cpu().double(), -1)):
        y = y[0] * sign
        assert not bool(y[:2 * PAGE].any())
        for p, value in ((2, 2.0 ** 60), (3, -(2.0 ** -20)), (4, 2.0 ** 60)):
            assert bool(((y[p * PAGE:(p + 1) * PAGE] - value).abs() <= abs(value) * 2.0 ** -7).all()), p


# ---- attend

MASKS = ["causal", "window", "documents", "everything"]


def _options(rig, heads, mask, g):
    o = {}
    if mask in ("window", "everything"):
        o["window"] = 70
    if mask in ("documents", "everything"):
        pos = torch.cat([s + torch.arange(n) for s, n in zip(rig.starts, rig.news)])
        first = (pos // 37 * 37).to(torch.int32)
        first[torch.rand(len(first), generator=g) < 0.2] = 1 << 29         # rows that see nothing
        first[0] = -5
        o["first"] = first
        o["prefix"] = torch.randint(0, 100, (len(rig.starts),), generator=g).to(torch.int32)
    if mask == "everything":
        o["slopes"] = torch.rand(heads, generator=g) * 0.3
        o["softcap"] = 5.0
    return o


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,group", [(64, 1), (80, 3), (96, 4), (128, 4), (128, 8), (256, 2), (128, 1), (64, 16), (128, 24)])
@pytest.mark.parametrize("mask", MASKS)
def test_attend_matches_the_definition(kind, d, group, mask):
    import bigsmall_amd as bs
    _say("attend", kind, d, group, mask)
    hk = 2
    rig = Rig([0, 63, 64, 130, 0, 5, 700, 191, 64], [1, 1, 1, 1, 130, 64, 3, 0, 64], hk, d, kind, seed=d * 10 + group)
    q = rig.rows(hk * group)
    o = _options(rig, hk * group, mask, rig.g)
    gpu = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in o.items()}
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), return_lse=True, **gpu)
    _check_attend(rig, q, out, lse, d ** -0.5, **o)
    assert torch.equal(bs.kv_attend(rig.pool, rig.batch, q.cuda(), **gpu), out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("starts,news,hk,group,d", [
    ([9000], [1], 1, 4, 128), ([4095, 4096, 17], [1, 1, 1], 2, 8, 64), ([20011], [2], 1, 2, 256), ([6000, 0], [40, 1], 1, 4, 96),
    ([3000], [150], 1, 6, 128), ([1], [700], 1, 5, 64), ([0, 2000, 13], [400, 1, 33], 2, 4, 80), ([0], [300], 1, 1, 256)])
def test_attend_long_caches_and_prompts(kind, starts, news, hk, group, d):
    import bigsmall_amd as bs
    _say("attend", kind, starts, news, hk, group, d)
    rig = Rig(starts, news, hk, d, kind, seed=sum(starts))
    q = rig.rows(hk * group, 2.0)
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), scale=0.07, return_lse=True)
    _check_attend(rig, q, out, lse, 0.07)
    first = torch.full((rig.total,), max(starts) // 2, dtype=torch.int32)       # the shorter sequences see nothing
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), scale=0.07, first=first.cuda(), softcap=30.0, return_lse=True)
    _check_attend(rig, q, out, lse, 0.07, first=first, softcap=30.0)


@pytest.mark.parametrize("start,new,d", [(20011, 2, 64), (17000, 20, 64), (16500, 1, 128)])
def test_attend_when_the_batch_says_too_little(start, new, d):
    """One workgroup for a cache of over 256 pages, and the kernel for few rows with many and for many with few."""
    import bigsmall_amd as bs
    rig = Rig([start], [new], 1, d, torch.int8, seed=start)
    q = rig.rows(2)
    for most_new, longest in ((1, 1), (1, start), (500, 1), (500, start + new)):
        batch = bs.KVBatch(rig.batch.start, rig.batch.cu, rig.batch.table, rig.batch.tails, most_new, longest)
        out, lse = bs.kv_attend(rig.pool, batch, q.cuda(), return_lse=True)
        _check_attend(rig, q, out, lse, d ** -0.5)


def test_cache_under_a_gpu_default_device():
    import bigsmall_amd as bs
    g = _gen(9)
    k = _bf16((70, 1, 64), g).cuda()
    outs = []
    for device in ("cpu", "cuda"):
        torch.set_default_device(device)
        try:
            cache = bs.PagedKVCache(1, 1, 64, pages=4, sequences=1)
            seq = cache.add()
            step = cache.step({seq: 70})
            q = cache.append(0, step, k, k, k, bs.Rope.from_theta(64, 100))
            outs.append((cache.attend(0, step, q), *cache.read(0, seq)))
        finally:
            torch.set_default_device("cpu")
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("most", [1, 90])
def test_attend_many_sequences_of_all_lengths(most):
    """More workgroups than run at once, sequences without new rows and of one token among them."""
    import bigsmall_amd as bs
    g = _gen(21)
    b, hk = 140, 4
    starts = torch.randint(0, 300, (b,), generator=g).tolist()
    news = torch.randint(0, 2, (b,), generator=g).tolist() if most == 1 else (torch.randint(0, most + 1, (b,), generator=g) // 10).tolist()
    starts[3], news[3], news[7], news[-1] = 0, 1, most, 0
    rig = Rig(starts, news, hk, 64, torch.int8, seed=5)
    q = rig.rows(hk * 2)
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), return_lse=True)
    _check_attend(rig, q, out, lse, 64 ** -0.5)
    # what the batch says of its sizes chooses the launches, not the results
    for most_new, longest in ((1, 1), (most, 20000), (400, 400), (max(news), max(news))):
        other = bs.KVBatch(rig.batch.start, rig.batch.cu, rig.batch.table, rig.batch.tails, most_new, longest)
        out, lse = bs.kv_attend(rig.pool, other, q.cuda(), return_lse=True)
        _check_attend(rig, q, out, lse, 64 ** -0.5)


@pytest.mark.parametrize("news", [[1, 1], [70, 130]])
def test_attend_scales_of_very_different_pages(news):
    """Pages whose values differ by many powers of two, zero pages among them, and rows of q as different."""
    import bigsmall_amd as bs
    rig = Rig([640, 448], news, 1, 64, torch.int8, seed=3)
    pages = rig.pages[0] + rig.pages[1]
    for i, p in enumerate(pages):
        rig.pool.v_scale[p] *= 2.0 ** [-47, 0, -20, 20, 0, 10, -30, 3][i % 8]
        if i % 5 == 4:
            rig.pool.v[p] = 0
            rig.pool.v_scale[p] = 2.0 ** -40 / 127
    q = rig.rows(4)
    q[:, 1] *= 2.0 ** -60
    q[:, 2] *= 2.0 ** 5
    q[:, 3] = 0
    out, lse = bs.kv_attend(rig.pool, rig.batch, q.cuda(), return_lse=True)
    _check_attend(rig, q, out, lse, 64 ** -0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 90])
def test_poisoned_tokens_reach_only_rows_that_see_them(kind, n):
    """NaN and infinities in k, v and q: rows that see such a token (or a full page with one) are NaN, all others are
    what they are without it."""
    import bigsmall_amd as bs
    hk, d, length = 1, 64, 200
    g = _gen(11)
    k, v = _bf16((length, hk, d), g), _bf16((length, hk, d), g)
    q = _bf16((n, 2, d), g)
    k[70, 0, 3] = math.nan            # page 1
    v[197, 0, 5] = math.inf           # the tail
    cache = bs.PagedKVCache(1, hk, d, pages=8, sequences=2, kind=kind)
    seq = cache.add()
    cache.append(0, cache.step({seq: length - n}), None, k[:length - n].cuda(), v[:length - n].cuda())
    step = cache.step({seq: n})
    cache.append(0, step, None, k[length - n:].cuda(), v[length - n:].cuda())
    pos = torch.arange(length - n, length)
    for first in (0, 64, 128, 192, 198):
        f = torch.minimum(torch.full((n,), first), pos).to(torch.int32)
        if n > 1:
            q[1] = math.inf
        out = bs.kv_attend(cache.pools[0], step, q.cuda(), first=f.cuda()).cpu()
        # a row inside page 1 sees part of the page: its scale is NaN
        bad = ((f < 128) & (pos >= 64)) | ((f <= 197) & (pos >= 197))
        if n > 1:
            bad[1] = True
        assert torch.equal(torch.isnan(out).all(-1).all(-1), bad) and torch.equal(torch.isnan(out).any(-1).any(-1), bad), first


def test_strides_alignment_and_streams():
    """q, k, v as parts of one projection's output, rows that start at odd places, and a stream of its own."""
    import bigsmall_amd as bs
    hk, group, d = 2, 4, 128
    rig = Rig([10, 100, 0], [1, 40, 64], hk, d, torch.int8, seed=1)
    g = rig.g
    fused = _bf16((rig.total, (hk * group + 2 * hk), d), g).cuda()
    q, k, v = fused.split([hk * group, hk, hk], 1)
    rope = bs.Rope.from_theta(d, 200)
    want_q = bs.kv_append(rig.pool, rig.batch, q.contiguous(), k.contiguous(), v.contiguous(), rope)
    want = _cpu(rig.pool)
    want_o = bs.kv_attend(rig.pool, rig.batch, want_q)
    odd = torch.empty(fused.numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view(fused.shape)
    odd.copy_(fused)
    wide = torch.empty(rig.total, fused.shape[1], 2 * d, dtype=torch.bfloat16, device="cuda")
    wide[:, :, ::2] = fused
    heads_first = fused.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (fused, odd, wide[:, :, ::2], heads_first):
        q, k, v = x.split([hk * group, hk, hk], 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for t in ("k", "v"):
                getattr(rig.pool, t).zero_()
            got_q = bs.kv_append(rig.pool, rig.batch, q, k, v, rope)
            got_o = bs.kv_attend(rig.pool, rig.batch, got_q)
            assert bs.kv_append(rig.pool, rig.batch, got_q, k, v) is got_q      # nothing turns: q as it is
            bs.kv_append(rig.pool, rig.batch, q, k, v, rope, out=got_q)
        side.synchronize()
        assert torch.equal(got_q, want_q)
        for i, (a, b) in enumerate(zip(want, _cpu(rig.pool))):
            if i >= 2:
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        used = [p for b, s in enumerate(rig.starts) for p in rig.pages[b][s // PAGE:(s + rig.news[b]) // PAGE]]
        assert torch.equal(rig.pool.k[used].cpu(), want[0][used]) and torch.equal(rig.pool.v[used].cpu(), want[1][used])
    # in place
    q = fused[:, :hk * group].contiguous()
    assert bs.kv_append(rig.pool, rig.batch, q, fused[:, 8:10], fused[:, 10:], rope, out=q) is q
    assert torch.equal(q, want_q)


def test_page_numbers_past_4_gib():
    """Pages whose bytes lie past 2^31 and 2^32 from the pool's start."""
    import bigsmall_amd as bs
    hk, d, pages = 8, 128, 66000
    k = torch.zeros(pages, hk, PAGE, d, dtype=torch.int8, device="cuda")
    v = torch.zeros(pages, hk, d, PAGE, dtype=torch.int8, device="cuda")
    scale = torch.ones(2, pages, hk, device="cuda")
    tails = torch.zeros(2, 2, hk, PAGE * d, dtype=torch.bfloat16, device="cuda")
    pool = bs.KVPool(k, v, scale[0], scale[1], tails[0].view(2, hk, PAGE, d), tails[1].view(2, hk, d, PAGE))
    table = torch.tensor([[65999, 33000, 3, 65537]], dtype=torch.int32)
    args = (torch.tensor([0], dtype=torch.int32).cuda(), torch.tensor([0, 250], dtype=torch.int32).cuda(), table.cuda(),
            torch.tensor([[0, 1]], dtype=torch.int32).cuda())
    batch = bs.KVBatch(*args, 250, 250)
    g = _gen(2)
    x = _bf16((250, hk, d), g)
    y = _bf16((250, hk, d), g)
    bs.kv_append(pool, batch, None, x.cuda(), y.cuda())
    got_k, got_v = bs.kv_read(pool, batch.table[0], 250, batch.tails[0, 1:])
    for got, put in ((got_k, x), (got_v, y)):
        for h in range(hk):
            want = put[:, h].clone()                       # the last 58 tokens are in the tail
            for p in range(3):
                codes, scale_h = ref.quantise32(want[64 * p:64 * p + 64], torch.int8)
                want[64 * p:64 * p + 64] = (codes.float() * scale_h).to(torch.bfloat16)
            assert torch.equal(got[h].cpu(), want), h
    low = [0, 1, 2, 3]
    small = [t[[65999, 33000, 3, 65537]].cpu() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]
    q = _bf16((250, hk, d), g)
    out, lse = bs.kv_attend(pool, batch, q.cuda(), return_lse=True)
    o, l, tol, ltol = ref.attend(small + [pool.k_tail.cpu(), pool.v_tail.cpu()], low, 1, 0, q, d ** -0.5)
    assert bool(((out.cpu().double() - o).abs() <= tol).all()) and bool(((lse.cpu().double() - l).abs() <= ltol).all())


def test_step_captured_into_a_graph():
    """Append and attend replayed from a graph, with other work between the replays, against the eager results."""
    import bigsmall_amd as bs
    hk, group, d = 2, 4, 64
    rig = Rig([1500, 63, 0, 200], [1, 1, 1, 1], hk, d, torch.float8_e4m3fn, seed=8)
    rope = bs.Rope.from_theta(d, 2000)
    static = [rig.rows(h).cuda() for h in (hk * group, hk, hk)]

    def step():
        q = bs.kv_append(rig.pool, rig.batch, *static, rope)
        return q, bs.kv_attend(rig.pool, rig.batch, q)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        fresh = [rig.rows(h).cuda() for h in (hk * group, hk, hk)]
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [c.clone() for c in captured]
        junk = torch.randn(1 << 20, device="cuda").sum()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert bool(torch.isfinite(junk))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 777])
@pytest.mark.parametrize("d", [64, 80, 256])
def test_read(kind, n, d):
    import bigsmall_amd as bs
    rig = Rig([0], [n], 3, d, kind, seed=n)
    pool = _cpu(rig.pool)
    k, v = bs.kv_read(rig.pool, rig.batch.table[0], n, rig.batch.tails[0, 1:])
    assert k.shape == v.shape == (3, n, d) and k.dtype == torch.bfloat16
    for h in range(3):
        for got, want in zip((k, v), ref.cached(pool, rig.pages[0], rig.tails[0], n, h)):
            # code * scale in f32, then rounded to bf16
            assert bool(((got[h].cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all())


def test_numbers_that_do_not_exist_are_reported():
    """A page, a tail and lengths out of range set the status and leave other sequences right."""
    import bigsmall_amd as bs
    from bigsmall_amd import _native
    from bigsmall_amd.device import StatusWord
    rig = Rig([100, 100, 100, 100], [70, 70, 70, 70], 1, 64, torch.int8, seed=4)
    q, k, v = (rig.rows(1).cuda() for _ in range(3))
    st = StatusWord("cuda")
    good = bs.kv_attend(rig.pool, rig.batch, q, status=st)
    bs.kv_append(rig.pool, rig.batch, q, k, v, status=st)
    good = bs.kv_attend(rig.pool, rig.batch, q, status=st)
    assert int(st.t) == 0
    want = _cpu(rig.pool)
    for what in ("page", "tail", "start", "cu"):
        st.reset()
        start, cu, table, tails = (t.clone() for t in (rig.batch.start, rig.batch.cu, rig.batch.table, rig.batch.tails))
        if what == "page":
            table[1, 1] = rig.pool.n_pages
        elif what == "tail":
            tails[1, 1] = -1
        elif what == "start":
            start[1] = 1 << 28
        else:
            cu[1:3] = torch.tensor([70, 50])           # the second sequence ends before it begins
        batch = bs.KVBatch(start, cu, table, tails, 70, 170)
        bs.kv_append(rig.pool, batch, q, k, v, status=st)
        assert int(st.t) == _native.BS_DEV_ERR_BOUNDS, what
        st.reset()
        out = bs.kv_attend(rig.pool, batch, q, status=st)
        assert int(st.t) == _native.BS_DEV_ERR_BOUNDS, what
        rows = slice(0, 50) if what == "cu" else slice(0, 70)
        assert torch.equal(out[rows], good[rows]) and torch.equal(out[210:], good[210:]), what
        if what != "cu":
            for a, b in zip(want, _cpu(rig.pool)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), what
    st.reset()
    bs.kv_read(rig.pool, torch.full((2,), -1, dtype=torch.int32, device="cuda"), 100, torch.tensor([99], dtype=torch.int32).cuda(), status=st)
    assert int(st.t) == _native.BS_DEV_ERR_BOUNDS
