"""Calls of the 8-bit floating point operators that are refused, on the CPU:
scales that overlap, outputs in the buffers of inputs."""
import ctypes

import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import F8
from shady_thinker_amd._lib import ST_F16, ST_F32, lib

ST_ERR_INVALID = 1  # (st_status)


@pytest.mark.parametrize("m,blocks,scale", [
    (3, 2, lambda: torch.ones(1, 3).expand(2, 3)),  # (a token's scale for all of its blocks)
    (1, 2, lambda: torch.ones(1, 1).expand(2, 1)),
    (3, 3, lambda: torch.ones(7).as_strided((3, 3), (2, 1)))])
def test_scales_that_overlap(m, blocks, scale):
    """A block's scales begin where the one before's end, or later: the calls
    read and write [blocks, M] of them from the first one on."""
    with pytest.raises(ValueError, match="scale"):
        sta.Fp8Rows.of(torch.zeros(m, 128 * blocks).to(F8), scale())


def test_scales_side_by_side():
    wide = torch.ones(2, 9)
    assert sta.Fp8Rows.of(torch.zeros(3, 256).to(F8), wide[:, 4:7]).stride == 9
    assert sta.Fp8Rows.of(torch.zeros(1, 256).to(F8), torch.ones(2, 1)).stride == 1
    assert sta.Fp8Rows.of(torch.zeros(3, 128).to(F8), torch.ones(3).as_strided((1, 3), (0, 1))).stride == 3  # (one block: no next one)


# ------------------------------------------- buffers that are one, C entry points
CTX = ctypes.create_string_buffer(1024)  # (never used: every call below is refused before)
M, K, N = 3, 144, 40
A = [4096 * i for i in range(1, 9)]  # (addresses)
NORM = dict(ctx=CTX, residual=A[0], res_dtype=ST_F32, res_stride=K, x=A[1], x_dtype=ST_F32, x_stride=K, residual_out=A[2], out_stride=K,
            weight=A[3], eps=1e-6, y=A[4], y_dtype=ST_F32, y_stride=K, y8=A[5], y_scale=A[6], scale_stride=M, m=M, d=K, flags=0)
QUANT = dict(ctx=CTX, a=A[0], b=A[1], dtype=ST_F16, a_stride=K, b_stride=K, y8=A[2], y_scale=A[3], scale_stride=M, m=M, k=K)
GEMM = dict(ctx=CTX, x=A[0], x_scale=A[1], scale_stride=M, w=A[2], w_scale=A[3], y=A[4], y_dtype=ST_F32, m=M, k=K, n=N)


def refused(fn, args, match):
    assert getattr(lib(), fn)(*args.values()) == ST_ERR_INVALID
    assert lib().st_last_error().decode().startswith(fn) and match in lib().st_last_error().decode()


@pytest.mark.parametrize("kw", [dict(x_dtype=ST_F16), dict(x_stride=2 * K), dict(out_stride=2 * K), dict(res_dtype=ST_F16)])
def test_sum_over_another_kind_of_x(kw):
    """A row's sum would cover other rows of x, before their workgroups read them."""
    refused("st_add_rmsnorm", {**NORM, "residual_out": A[1], **kw}, "residual_out in x's buffer")


@pytest.mark.parametrize("out", ["y8", "y_scale"])
@pytest.mark.parametrize("other", ["residual", "x", "residual_out", "weight", "y"])
def test_norm_rows_over_other_buffers(out, other):
    refused("st_add_rmsnorm", {**NORM, out: NORM[other]}, "buffer")


@pytest.mark.parametrize("kw", [dict(y_scale=A[5]), dict(y=A[3]), dict(residual_out=A[3])])
def test_norm_other_buffers(kw):
    refused("st_add_rmsnorm", {**NORM, **kw}, "buffer")


@pytest.mark.parametrize("kw", [dict(y8=A[0]), dict(y8=A[1]), dict(y_scale=A[0]), dict(y_scale=A[1]), dict(y_scale=A[2])])
def test_quant_over_inputs(kw):
    refused("st_fp8_quant", {**QUANT, **kw}, "buffer")


@pytest.mark.parametrize("other", ["x", "x_scale", "w", "w_scale"])
def test_product_over_inputs(other):
    refused("st_fp8_gemm", {**GEMM, "y": GEMM[other]}, "buffer")
