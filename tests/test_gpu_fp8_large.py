"""Products by the tile of 256 by 256 where a workgroup goes through several tiles of many blocks, on numbers whose sums are exact
in any order: a block that is missing, doubled or of another tile shows in every result."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# rows of x, rows of the weight, columns: an odd and an even number of blocks, more than 64 of them, whole tiles and such that end
# inside, rows of the result that start at multiples of 16 bytes and such that do not
SEVERAL_TILES = [(4096, 8192, 4097), (5100, 13000, 4000), (8100, 8104, 8500), (8100, 8099, 4200), (8192, 8192, 640)]


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def _case(t, n, k, dtype):
    """x and a weight of small whole numbers, the first of each block of x 448 (so that its scale is 1), scales powers of two:
    group by group, block by block and in the end all sums are multiples of 1/2 below 2^21."""
    g = torch.Generator(device="cuda").manual_seed(t + n + k)

    def whole(rows, cols, most):
        return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda")

    x = whole(t, k, 8).to(dtype)
    x[:, ::128] = 448.0 * (1 - 2 * (x[:, ::128] < 0).to(dtype))
    codes = whole(n, k, 4).to(torch.float32).to(torch.float8_e4m3fn)
    scales = torch.exp2(whole(-(-n // 128), -(-k // 128), 1).float())
    w = codes.float() * scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x, codes, scales, (x.double() @ w.double().T).to(dtype)


@pytest.mark.parametrize("t,n,k", SEVERAL_TILES)
def test_exact_sums(t, n, k):
    import bigsmall_amd as bs
    x, codes, scales, want = _case(t, n, k, (torch.bfloat16, torch.float16)[k % 2])
    weight = bs.Fp8Weight(codes, scales)
    rows = bs.fp8_quantise(x)
    assert bool((rows.scales == 1).all())
    assert torch.equal(bs.fp8_linear(rows, weight), want)
    assert torch.equal(bs.fp8_linear(x, weight), want)


@pytest.mark.parametrize("t,n,k", SEVERAL_TILES[:3])
def test_what_is_not_finite_stays_in_its_rows(t, n, k):
    """Rows that are no numbers, in the first, a middle and the last block of some tiles, and not in the tile that comes next."""
    import bigsmall_amd as bs
    x, codes, scales, want = _case(t, n, k, torch.bfloat16)
    bad = torch.zeros(t, dtype=torch.bool, device="cuda")
    for first in (0, 512, 1024, 2560, t - 40):
        bad[first:first + 256:7] = True
    at = torch.nonzero(bad)[:, 0]
    x[at[0::3], 0], x[at[1::3], k // 2], x[at[2::3], k - 1] = math.nan, math.inf, -math.inf
    y = bs.fp8_linear(x, bs.Fp8Weight(codes, scales))
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], want[~bad])
