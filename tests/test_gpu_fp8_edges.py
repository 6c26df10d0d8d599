"""Calls of the 8-bit floating point operators that their documentation allows
at its edges: the sum in the buffer of x, tiles and columns past a launch."""
import pytest
import torch

import shady_thinker_amd as sta
from shady_thinker_amd._lib import launches

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
DEV = "cuda:0"


def rand(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


@pytest.mark.parametrize("m,d", [(1, 4096), (300, 2576), (5, 16400)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_sum_in_the_buffer_of_x(gpu, m, d, dtype):
    """residual_out may be x: the bits of a buffer of its own."""
    r, x, w = rand(1, m, d, dtype=dtype), rand(2, m, d, dtype=dtype), rand(3, d)
    want, rows, again = torch.empty_like(r), sta.Fp8Rows(gpu, m, d), sta.Fp8Rows(gpu, m, d)
    sta.add_rmsnorm(gpu, r, w, x, rows=rows, residual_out=want)
    sta.add_rmsnorm(gpu, r, w, x, rows=again, residual_out=x)
    assert torch.equal(x, want) and torch.equal(rows.scale, again.scale)
    assert torch.equal(rows.data.view(torch.uint8), again.data.view(torch.uint8))


def test_tiles_that_do_not_fit_a_launch(gpu, tune):
    """65 tokens and 2^28 columns, f32 y: 64 x 64 would be 2^32 threads, more than
    a launch has; the setting gives way to a tile that fits."""
    m, k, n, b = 65, 16, 1 << 28, 1 << 16
    tune(FP8_TILE=1)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-8, 9, (m, k), device=DEV, generator=g).float()
    part = torch.randint(-8, 9, (b, k), device=DEV, generator=g).float()
    w = part.to(torch.float8_e4m3fn).view(torch.uint8).repeat(n // b, 1).view(torch.float8_e4m3fn)
    scale = 2.0 ** (torch.arange(n // 128, device=DEV)[:, None] % 3).float()
    y = torch.empty(m, n, device=DEV)
    launches()
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x.to(torch.float8_e4m3fn), torch.ones(1, m, device=DEV)), sta.Fp8Weight.of(w, scale), y)
    assert launches() == ["fp8_ring_kernel"]
    want = x @ part.t()  # (whole numbers: exact)
    for n0 in (0, n // 2, n - b):
        assert torch.equal(y[:, n0:n0 + b], want * scale[n0 // 128:(n0 + b) // 128, 0].repeat_interleave(128))


@pytest.mark.parametrize("xs,ys", [((272,), (150,)), ((2, 3, 272), (2, 3, 150)), ((4, 272), (700,))])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_linear_of_any_shape(gpu, xs, ys, dtype):
    """linear() takes x and y of any shape that holds the rows, as for the other
    weights; what lies behind them is left alone."""
    w8 = (rand(1, 150, 272) * 20).to(torch.float8_e4m3fn)
    w, x, y = sta.Fp8Weight.of(w8, rand(2, 2, 3).abs()), rand(3, *xs), torch.full(ys, 7.0, dtype=dtype, device=DEV)
    m = x.numel() // 272
    rows, want = sta.Fp8Rows(gpu, m, 272), torch.empty(m, 150, dtype=dtype, device=DEV)
    sta.linear(gpu, x, w, y)
    sta.fp8_quant(gpu, x.view(m, 272), rows)
    sta.fp8_gemm(gpu, rows, w, want)
    assert torch.equal(y.view(-1)[:m * 150], want.view(-1)) and (y.view(-1)[m * 150:] == 7.0).all()
