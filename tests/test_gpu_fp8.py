"""fp8_quantise and fp8_linear on the GPU against their definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _x(t, k, dtype, g):
    x = torch.randn(t, k, generator=g) * (0.25 + torch.rand(t, 1, generator=g) * 4)
    x[:, ::37] *= 20
    return x.to(dtype)


def _w(n, k, g):
    codes = (torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, (0.5 + torch.rand(-(-n // 128), -(-k // 128), generator=g)) * 1e-3


def _same_rows(rows, x):
    codes, scales = ref.quantise(x)
    assert torch.equal(rows.codes.cpu().float().double(), codes)
    got = rows.scales.cpu()
    assert got.shape == scales.shape and torch.equal(torch.isnan(got), torch.isnan(scales))
    fine = ~torch.isnan(scales)
    assert torch.equal(got[fine], scales[fine].float())               # one rounding


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k", [(1, 1), (1, 128), (3, 127), (17, 129), (16, 512), (33, 1000), (5, 1001), (130, 640), (2, 4096)])
def test_quantise(t, k, dtype):
    import bigsmall_amd as bs
    x = _x(t, k, dtype, _gen(t * 1000 + k))
    _same_rows(bs.fp8_quantise(x.cuda()), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_borders(dtype):
    """Every pair of significands: quotients that are borders between two codes, and those next to them."""
    import bigsmall_amd as bs
    bits = 8 if dtype == torch.bfloat16 else 11
    tops = torch.arange(1 << (bits - 1), 1 << bits) if bits == 8 else torch.randint(1 << 10, 1 << 11, (256,), generator=_gen(1))
    tops = torch.cat([tops, torch.arange(7 << (bits - 4), 1 << bits, 7 << (bits - 6))])     # multiples of 7: 448 / a is short
    x = torch.zeros(len(tops), (1 << (bits - 1)) // 127 * 128 + 128)
    values = torch.arange(1 << (bits - 1), 1 << bits).float()
    at = torch.arange(len(values)) // 127 * 128 + 1 + torch.arange(len(values)) % 127
    for i, a in enumerate(tops.tolist()):
        x[i, ::128] = a
        x[i, at] = torch.where(values <= a, values, values / 2) * 2.0 ** -(i % 7)
    x[1::2] *= -1
    _same_rows(bs.fp8_quantise(x.to(dtype).cuda()), x.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_extremes(dtype):
    import bigsmall_amd as bs
    x = torch.zeros(9, 300).to(dtype)
    info = torch.finfo(dtype)
    x[1, 5] = info.max
    x[1, 6] = -info.max / 3
    x[2, 130] = info.smallest_normal
    x[2, 131] = info.smallest_normal * info.eps            # the smallest there is
    x[3] = 1.0
    x[4, 0], x[4, 299] = math.inf, 1.0
    x[5, 128], x[5, 0] = math.nan, 2.0
    x[6, 299] = -math.inf
    x[7] = info.smallest_normal
    x[8, 7] = 3.0
    if dtype == torch.bfloat16:
        x[8, 140], x[8, 141] = 2.0 ** -101, -2.0 ** -108   # below the smallest scale's largest value
        x[8, 280], x[8, 281] = 2.0 ** 101, 2.0 ** 93       # beyond which both sides are scaled down
    _same_rows(bs.fp8_quantise(x.cuda()), x)


def _check(y, rows, w, ws, dtype, device="cpu"):
    want, tol = ref.linear(rows.codes.to(device).float().double(), rows.scales.to(device).double(), w.to(device), ws.to(device), dtype)
    off = (y.to(device).double() - want).abs()
    worst = float((off / tol).max())
    assert worst <= 1, worst


SHAPES = [(1, 16, 128), (1, 128, 128), (2, 1, 1), (3, 7, 100), (15, 129, 129), (16, 64, 256), (17, 130, 300), (31, 257, 1000), (33, 48, 640),
          (64, 320, 384), (65, 17, 1024), (100, 1000, 200), (128, 128, 512), (129, 256, 128), (200, 255, 900), (257, 513, 260),
          (300, 384, 1300), (1, 4096, 2000), (8, 1000, 4096), (40, 512, 3200), (700, 640, 256), (1, 1, 14336), (1000, 300, 640)]


@pytest.mark.parametrize("t,n,k", SHAPES)
def test_linear(t, n, k):
    import bigsmall_amd as bs
    g = _gen(t + n + k)
    dtype = TYPES[(t + n) % 2]
    x = _x(t, k, dtype, g).cuda()
    w, ws = _w(n, k, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    rows = bs.fp8_quantise(x)
    y = bs.fp8_linear(x, weight)
    assert y.dtype == dtype and y.shape == (t, n)
    _check(y, rows, w, ws, dtype)
    other = TYPES[1 - TYPES.index(dtype)]
    z = bs.fp8_linear(rows, weight, dtype=other)              # quantised once, the other type out
    assert z.dtype == other
    _check(z, rows, w, ws, other)
    assert t <= 16 or torch.equal(bs.fp8_linear(rows, weight), y)      # (few rows: another kernel, other sums)


# Sizes for each way in which a product is cut up (tiles of 32 by 16 to 256 by 256, one to several turns), odd and even numbers of
# blocks, and more than 64 blocks to a wave, whose scales come 64 at a time.
LARGE = [(61, 4090, 4000), (64, 4097, 3000), (50, 8000, 1000), (64, 14000, 700), (250, 7001, 800), (129, 4097, 900), (500, 4100, 700), (900, 4000, 9000),
         (1100, 3500, 1500), (1500, 4000, 256), (1300, 4500, 1000), (300, 14001, 400), (2300, 5000, 520), (3000, 4100, 200), (2100, 4609, 130),
         (2050, 4999, 9000), (1300, 9000, 8500), (250, 7001, 8500), (2, 33, 70000), (5, 70, 40000), (20, 2000, 40000), (16, 14336, 33000), (300, 500, 34000)]


@pytest.mark.parametrize("t,n,k", LARGE)
def test_linear_large(t, n, k):
    import bigsmall_amd as bs
    g = _gen(t + n + k)
    dtype = TYPES[(t + k) % 2]
    x = _x(t, k, dtype, g).cuda()
    w, ws = _w(n, k, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    y = bs.fp8_linear(x, weight)
    rows = bs.fp8_quantise(x)
    _check(y, rows, w, ws, dtype, "cuda")
    assert torch.equal(bs.fp8_linear(rows, weight), y)


# More tiles of 256 by 256 than compute units, so that a workgroup has several: of one, two, three and more blocks; tiles that are
# stored whole before ones that are not and after them (4,608 = 18 * 256; odd rows of y).
MANY = [(4200, 4300, 128), (8192, 4096, 128), (4350, 4608, 384), (4200, 4300, 256), (9000, 4608, 130), (4608, 4611, 520), (8200, 4107, 70),
        (4100, 4400, 8400)]


@pytest.mark.parametrize("t,n,k", MANY)
def test_linear_many_tiles(t, n, k):
    import bigsmall_amd as bs
    g = _gen(t + n + k)
    dtype = TYPES[n % 2]
    x = _x(t, k, dtype, g).cuda()
    w, ws = _w(n, k, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    rows = bs.fp8_quantise(x)
    y = bs.fp8_linear(rows, weight)
    _check(y, rows, w, ws, dtype, "cuda")
    for _ in range(3):
        assert torch.equal(bs.fp8_linear(rows, weight), y)


def test_each_block_has_its_scale():
    """Exact numbers: code 1 in one place each, so a result names the scales that made it."""
    import bigsmall_amd as bs
    t, n, k = 37, 400, 700
    scales = 2.0 ** torch.arange(-12, 12).float()[:4 * 6].reshape(4, 6)
    for j in range(6):
        w = torch.zeros(n, k)
        w[:, j * 128 + 3] = 1.0
        x = torch.zeros(t, k)
        x[:, j * 128 + 3] = 448.0 * (1 + torch.arange(t) % 3)
        y = bs.fp8_linear(x.bfloat16().cuda(), bs.Fp8Weight(w.to(torch.float8_e4m3fn).cuda(), scales.cuda()))
        want = x[:, j * 128 + 3, None] * scales.repeat_interleave(128, 0)[:n, j]
        assert torch.equal(y.cpu().float(), want)


@pytest.mark.parametrize("t", [1, 16, 70, 300])
def test_what_is_not_finite_stays_in_its_row(t):
    import bigsmall_amd as bs
    g = _gen(t)
    w, ws = _w(200, 500, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    x = _x(t, 500, torch.bfloat16, g)
    clean = bs.fp8_linear(x.cuda(), weight).cpu()
    x[t // 2, 499] = math.nan
    if t > 2:
        x[0, 0] = math.inf
    y = bs.fp8_linear(x.cuda(), weight).cpu()
    bad = torch.zeros(t, dtype=torch.bool)
    bad[t // 2] = True
    if t > 2:
        bad[0] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad])
    assert float(bs.fp8_linear(torch.zeros(t, 500, dtype=torch.float16).cuda(), weight).abs().max()) == 0


@pytest.mark.parametrize("t,n,k", [(8192, 4096, 128), (4350, 4608, 384), (1300, 4700, 300), (1300, 4700, 600)])
def test_what_is_not_finite_stays_in_its_tile(t, n, k):
    """Rows that are no numbers in every group of 16 of some tiles; workgroups that go on with another tile leave them behind."""
    import bigsmall_amd as bs
    g = _gen(t + k)
    x = _x(t, k, torch.bfloat16, g)
    w, ws = _w(n, k, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    want = bs.fp8_linear(x.cuda(), weight)
    bad = torch.zeros(t, dtype=torch.bool)
    for first in (0, 256, 1024, t - 40):
        bad[first:first + 256:5] = True
    x[bad, k - 1] = math.inf
    x[bad & (torch.arange(t) % 2 == 0), 0] = math.nan
    y = bs.fp8_linear(x.cuda(), weight).cpu()
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], want.cpu()[~bad])


@pytest.mark.parametrize("t", [1, 20, 150])
def test_strides_and_shapes(t):
    import bigsmall_amd as bs
    g = _gen(t)
    n, k = 260, 384
    w, ws = _w(n, k, g)
    plain = bs.Fp8Weight(w.cuda(), ws.cuda())
    x = _x(t, k, torch.bfloat16, g).cuda()
    y = bs.fp8_linear(x, plain)
    wide = torch.full((t, k + 24), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:8 + k] = x
    assert torch.equal(bs.fp8_linear(wide[:, 8:8 + k], plain), y)                  # rows apart, aligned
    wide[:, 3:3 + k] = x
    assert torch.equal(bs.fp8_linear(wide[:, 3:3 + k], plain), y)                  # at no multiple of 16 bytes
    assert torch.equal(bs.fp8_linear(x.T.contiguous().T, plain), y)                # columns apart
    assert torch.equal(bs.fp8_linear(x.view(1, t, 1, k), plain), y.view(1, t, 1, n))
    assert torch.equal(bs.fp8_linear(x[:1].expand(t, k), plain), y[:1].expand(t, n))
    one = bs.fp8_linear(x[0], plain)
    assert one.shape == (n,)
    none = bs.fp8_linear(x[:0], plain)
    assert none.shape == (0, n)
    # weights: a slice of a wider one in place, one that is copied, scales that are a view
    big = torch.full((n + 3, k + 256), math.nan).to(torch.float8_e4m3fn).cuda()
    big[3:, 128:128 + k].view(torch.uint8).copy_(w.cuda().view(torch.uint8))
    part = bs.Fp8Weight(big[3:, 128:128 + k], ws.cuda().T.contiguous().T)
    assert part.codes.data_ptr() == big[3:, 128:].data_ptr()
    assert torch.equal(bs.fp8_linear(x, part), y)
    odd = torch.zeros(n, k + 5, dtype=torch.uint8).view(torch.float8_e4m3fn).cuda()
    odd[:, 5:].view(torch.uint8).copy_(w.cuda().view(torch.uint8))
    assert torch.equal(bs.fp8_linear(x, bs.Fp8Weight(odd[:, 5:], ws.cuda())), y)
    assert torch.equal(bs.fp8_linear(x, bs.Fp8Weight(w.cuda().view(torch.uint8).T.contiguous().T.view(torch.float8_e4m3fn), ws.cuda())), y)


@pytest.mark.parametrize("t", [1, 40, 260])
def test_graph_and_streams(t):
    import bigsmall_amd as bs
    g = _gen(t)
    w, ws = _w(512, 1024, g)
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    xs = [_x(t, 1024, torch.bfloat16, g).cuda() for _ in range(4)]
    want = [bs.fp8_linear(x, weight) for x in xs]
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        early = bs.fp8_linear(static, weight)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(early, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bs.fp8_linear(static, weight)
    for x, y in zip(xs, want):
        static.copy_(x)
        graph.replay()
        assert torch.equal(out, y)
        assert torch.equal(bs.fp8_linear(x, weight), y)
        torch.cuda.synchronize()


def test_gradients_are_refused_while_recorded():
    import bigsmall_amd as bs
    w, ws = _w(64, 128, _gen(0))
    weight = bs.Fp8Weight(w.cuda(), ws.cuda())
    x = torch.ones(2, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    for call in (lambda: bs.fp8_quantise(x), lambda: bs.fp8_linear(x, weight)):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    with torch.no_grad():
        assert not bs.fp8_linear(x, weight).requires_grad
