"""Calls of the 8-bit floating point operators that their documentation allows
at its edges: the sum in x's buffer."""
import pytest
import torch

import shady_thinker_amd as sta

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
