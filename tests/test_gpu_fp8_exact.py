"""st_fp8_gemm to the last bit, in every tile: whole numbers up to 8 and scales
of 1/2, 1 and 2. Products of an eight are within 2^6 of each other, so the 8-bit
instruction cuts none, and every sum is a multiple of 1/2 below 2^23: f32 holds
it whatever the order, and f16 y is its one rounding. A product, scale, row or
column out of its place shows, however long K is."""
import math
import random

import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import B, F8, blocks, check_product, rows_of, spread, weight_of
from shady_thinker_amd._lib import launches

pytestmark = pytest.mark.gpu

F32, F16, F64 = torch.float32, torch.float16, torch.float64
DEV = "cuda:0"


def case(seed, m, k, n):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pick = lambda lo, hi, *shape: torch.randint(lo, hi, shape, device=DEV, generator=g).float()
    return (pick(-8, 9, m, k).to(F8), 2.0 ** pick(-1, 2, blocks(k), m), pick(-8, 9, n, k).to(F8), 2.0 ** pick(0, 2, blocks(n), blocks(k)))


def exact(x8, sx, w8, sw):
    x = x8.to(F64) * spread(sx.to(F64), x8.shape[1])
    w = w8.to(F64) * sw.to(F64).repeat_interleave(B, 0)[:w8.shape[0]].repeat_interleave(B, 1)[:, :w8.shape[1]]
    return torch.mm(x, w.t())


def gemm(gpu, c, dtype):
    x8, sx, w8, sw = c
    m, n = x8.shape[0], w8.shape[0]
    buf = torch.full((m * n + 64,), 7.0, dtype=dtype, device=DEV)
    y = buf[:m * n].view(m, n)
    launches()
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    assert (buf[m * n:] == 7.0).all()
    return y, launches()


TILES16, TILES32 = (1, 2, 3, 4, 5, 7), (1, 2, 3, 4, 6)


@pytest.mark.parametrize("m,k,n", [(65, 400, 300), (130, 144, 136), (200, 2064, 513), (300, 11008, 260), (1030, 272, 776)])
@pytest.mark.parametrize("tile,splits,dtype", [(t, s, d) for d, tiles in ((F16, TILES16), (F32, TILES32)) for t in tiles
                                               for s in ((1, 4) if t != 7 else (1,))])
def test_tiles(gpu, tune, m, k, n, tile, splits, dtype):
    tune(FP8_TILE=tile, FP8_SPLITS=splits)
    c = case(m + k + n, m, k, n)
    y, ran = gemm(gpu, c, dtype)
    assert ran[0] == ("fp8_wide_kernel" if tile == 7 else "fp8_ring_kernel")
    assert torch.equal(y, exact(*c).to(dtype))


@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 33, 49, 64])
@pytest.mark.parametrize("k,n", [(400, 300), (11008, 515), (272, 13830), (16512, 8200)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_few_tokens(gpu, tune, m, k, n, dtype):
    tune(FP8_TILE=0)
    c = case(m + k + n, m, k, n)
    y, ran = gemm(gpu, c, dtype)
    assert ran == ["fp8_mv_kernel"] and torch.equal(y, exact(*c).to(dtype))


# The 256 x 256 kernel: a workgroup for each CU takes tiles one after the other,
# an XCD's CUs (32) a run of an eighth of them, those of the last round halved
# along the tokens where that gives every CU one.
@pytest.mark.parametrize("m,n", [
    (2500, 3500),   # 140 tiles: a whole one each
    (4096, 4096),   # 256: each CU one, none left
    (2500, 7600),   # 300: one, then halves
    (5100, 5130),   # 420: one, then whole ones
    (5100, 10240),  # 800: three, then halves
    (330, 3000)])   # 24: halves, some past the last token
@pytest.mark.parametrize("k", [144, 272, 384, 1040])
def test_wide(gpu, tune, m, n, k):
    tune(FP8_TILE=7)
    c = case(m + k + n, m, k, n)
    y, ran = gemm(gpu, c, F16)
    assert ran == ["fp8_wide_kernel"] and torch.equal(y, exact(*c).to(F16))


@pytest.mark.parametrize("m,k,n", [(2500, 11008, 3500), (5100, 8320, 4100), (2500, 16512, 7600), (200, 24704, 520), (2600, 8192, 7000)])
def test_wide_long(gpu, tune, m, k, n):
    """More blocks of K than the 64 whose scales a wave holds, also where the
    next tile's begin in the other half."""
    tune(FP8_TILE=7)
    c = case(m + k + n, m, k, n)
    y, ran = gemm(gpu, c, F16)
    assert ran == ["fp8_wide_kernel"] and torch.equal(y, exact(*c).to(F16))


@pytest.mark.parametrize("m", [130, 500])
@pytest.mark.parametrize("tile", TILES16)
def test_every_place(gpu, tune, m, tile):
    """One-hot rows return the weight's columns, f16 y its one rounding."""
    tune(FP8_TILE=tile)
    k, n = 400, 300
    w8 = (torch.randn(n, k, generator=torch.Generator().manual_seed(5)) * 40).to(F8).to(DEV)
    sw = torch.rand(blocks(n), blocks(k), generator=torch.Generator().manual_seed(6)).to(DEV) + 0.5
    w = w8.double() * sw.double().repeat_interleave(B, 0)[:n].repeat_interleave(B, 1)[:, :k]
    for k0 in range(0, k, m):
        at = torch.arange(m, device=DEV)
        cols = (at + k0) % k
        x = torch.zeros(m, k, device=DEV)
        x[at, cols] = 2.0 ** (at % 5 - 2).float()
        sx = 2.0 ** (torch.arange(blocks(k), device=DEV)[:, None] - at % 3).float()
        y, _ = gemm(gpu, (x.to(F8), sx, w8, sw), F16)
        f = (sx[cols // B, at] * x[at, cols]).double()
        # (a power of two times an e4m3 value times sw: one f32 rounding, then f16's)
        assert torch.equal(y, (w[:, cols].t() * f[:, None]).float().half())


@pytest.mark.parametrize("m,n", [(130, 150), (300, 520), (2500, 3500)])
@pytest.mark.parametrize("tile", TILES16)
def test_not_finite(gpu, tune, m, n, tile):
    """NaN rows, scales and weights reach their own row and column alone, from
    the last row and column too, which tiles repeat or leave empty."""
    tune(FP8_TILE=tile)
    k = 272
    x8, sx, w8, sw = case(3, m, k, n)
    want = exact(x8, sx, w8, sw).half()
    rows, cols = [2, 3, 4, m - 1], [7, 8, n - 1]
    x8.view(torch.uint8)[[2, m - 1], 265] = 0x7F
    sx[1, 3], sx[0, 4] = math.nan, math.inf
    w8.view(torch.uint8)[[7, n - 1], 270] = 0xFF
    w8.view(torch.uint8)[8, :8] = 0x7F
    y, _ = gemm(gpu, (x8, sx, w8, sw), F16)
    assert torch.isnan(y[[2, 3, m - 1]]).all() and torch.isnan(y[:, cols]).all() and not torch.isfinite(y[4]).any()
    fine_r = torch.ones(m, dtype=torch.bool, device=DEV)
    fine_c = torch.ones(n, dtype=torch.bool, device=DEV)
    fine_r[rows], fine_c[cols] = False, False
    assert torch.equal(y[fine_r][:, fine_c], want[fine_r][:, fine_c])


# ----------------------------------------------- exact products for f16 y, by choice
@pytest.mark.parametrize("m,k,n", [(65, 2752, 515), (300, 1040, 260), (1030, 272, 776)])
@pytest.mark.parametrize("tile,splits", [(-1, -1), (1, 1), (2, 4), (3, 1), (4, 4), (6, 1), (6, 4), (5, -1), (7, -1)])
def test_exact_products(gpu, tune, m, k, n, tile, splits):
    """FP8_EXACT: f16 y within the bound of f32 sums, whatever the batch; tiles of
    the 8-bit instruction alone (5, 7) give way."""
    tune(FP8_EXACT=1, FP8_TILE=tile, FP8_SPLITS=splits)
    x8, sx = rows_of(torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(DEV) * (1.0 + 999.0 * (torch.arange(k, device=DEV) % 128 == 5)))
    w8, sw = weight_of(torch.randn(n, k, generator=torch.Generator().manual_seed(n)).to(DEV))
    y, ran = gemm(gpu, (x8, sx, w8, sw), F16)
    assert ran[0] == "fp8_ring_kernel"
    check_product(y, x8, sx, w8, sw, many=False)


@pytest.mark.parametrize("m", [1, 64, 65, 300])
@pytest.mark.parametrize("tile", [-1, 1, 2, 3, 4, 6])
def test_exact_products_that_cancel(gpu, tune, m, tile):
    """1 - 1 + 2^-14 of neighbouring k is 2^-14."""
    tune(FP8_EXACT=1, FP8_TILE=tile)
    x, w = torch.zeros(m, 272, device=DEV), torch.zeros(200, 272, device=DEV)
    x[:, 160:163], w[:, 160:163] = torch.tensor([1.0, -1.0, 2.0**-7], device=DEV), torch.tensor([1.0, 1.0, 2.0**-7], device=DEV)
    y, _ = gemm(gpu, (x.to(F8), torch.ones(3, m, device=DEV), w.to(F8), torch.ones(2, 3, device=DEV)), F16)
    assert (y == 2.0**-14).all()


@pytest.mark.parametrize("seed", range(48))
def test_drawn(gpu, seed):
    """Sizes spread over the range, tile and slices by the estimates; a part of
    a larger batch's rows."""
    rng = random.Random(seed)
    spread_over = lambda lo, hi, step=1: max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)
    m, k, n = rng.choice([spread_over(1, 64), spread_over(65, 4096)]), spread_over(16, 12000, 16), spread_over(1, 12000)
    dtype, skip = rng.choice([F16, F32]), rng.randint(0, 5)
    x8, sx, w8, sw = case(seed, m + skip, k, n)
    y = torch.full((m + 1, n), 7.0, dtype=dtype, device=DEV)
    with gpu.tuning(FP8_EXACT=rng.choice([0, 1])):
        sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx)[skip:], sta.Fp8Weight.of(w8, sw), y[:m])
    assert torch.equal(y[:m], exact(x8[skip:], sx[:, skip:], w8, sw).to(dtype)) and (y[m] == 7.0).all()
