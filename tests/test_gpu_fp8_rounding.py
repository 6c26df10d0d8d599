"""Quantised rows bit for bit: a block's scale is max |x| times the f32 nearest
to 1 / 448, its values the f32 quotients x / scale rounded to e4m3. The CPU's
f32 product, quotient and conversion are rounded once each, to nearest, even."""
import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import B, F8, spread

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
DEV = "cuda:0"


def rows32(y):
    """y [M, K] float32 on the CPU as (data, scale)."""
    m, k = y.shape
    most = torch.nn.functional.pad(y.abs(), (0, -k % B)).view(m, -1, B).amax(-1).t().contiguous()
    scale = (most * torch.tensor(1.0 / 448.0, dtype=F32)).clamp(min=2.0**-126)
    return (y / spread(scale, k)).clamp(-448, 448).to(F8), scale


def same(rows, y):
    data, scale = rows32(y)
    assert torch.equal(rows.scale.cpu(), scale)
    got, want = rows.data.cpu().view(torch.uint8), data.view(torch.uint8)
    assert torch.equal(got, want), ((got != want).sum(), y[got != want][:4])


def values(kind, m, k, dtype):
    g = torch.Generator().manual_seed(m + k)
    if kind == "whole":  # (quotients at the middle of two values are common)
        x = torch.randint(-200, 201, (m, k), generator=g).float()
    else:
        x = torch.randn(m, k, generator=g) * 2.0 ** torch.randint(-6, 7, (m, 1), generator=g)
    x[:, 3::7] *= 0.0  # (zeros of both signs)
    if kind == "tiny" and dtype is F32:
        x = x * 2.0**-122  # (scales about the least one, subnormal values)
    return x.to(dtype)


@pytest.mark.parametrize("m,k", [(1, 16), (77, 2752), (515, 4112), (1024, 11008)])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kind", ["whole", "normal", "tiny"])
def test_quotients(gpu, m, k, dtype, kind):
    x = values(kind, m, k, dtype)
    rows = sta.Fp8Rows(gpu, m, k)
    sta.fp8_quant(gpu, x.to(DEV), rows)
    same(rows, x.float())


@pytest.mark.parametrize("m,d", [(1, 4096), (31, 2576), (515, 5120), (7, 16400)])
@pytest.mark.parametrize("res", [F32, F16])
def test_norm_quotients(gpu, m, d, res):
    """The rows beside y are y's."""
    r, x = values("normal", m, d, res).to(DEV), values("whole", m, d, F16).to(DEV)
    y, rows = torch.empty(m, d, device=DEV), sta.Fp8Rows(gpu, m, d)
    sta.add_rmsnorm(gpu, r, torch.linspace(0.5, 1.5, d, device=DEV), x, y, rows)
    same(rows, y.cpu())


def test_a_block_with_an_infinity(gpu):
    """Its other values are 0, also the large ones."""
    x = torch.full((2, 2 * B), 3.0e38)
    x[0, 3], x[1, B + 5] = float("inf"), float("-inf")
    rows = sta.Fp8Rows(gpu, 2, 2 * B)
    sta.fp8_quant(gpu, x.to(DEV), rows)
    d = rows.data.float().cpu()
    assert (d != 0).view(2, 2, B).sum(-1).tolist() == [[1, B], [B, 1]] and d[0, 3] == 448 and d[1, B + 5] == -448
    assert torch.isinf(rows.scale.cpu()).tolist() == [[True, False], [False, True]]
