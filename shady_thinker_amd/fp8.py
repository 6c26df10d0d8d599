"""Linears in 8-bit floating point: rows of e4m3 activations, the norm and the
activation that make them, and their product with block-scaled weights.

No reference counterpart but for the norms (src/model.rs:685-691, 799-802,
820-823: rmsnorm.wgsl, add_rmsnorm.wgsl). Entry points of libshady_hip like
the other linears, on torch device tensors and torch's current stream:

* `Fp8Rows`: quantised rows, e4m3 with a scale for each token and 128 dims;
* `add_rmsnorm`: residual addition and norm, to such rows, to f32 / f16, or both;
* `fp8_quant`: rows, or silu(a) * b, to such rows;
* `fp8_gemm`: rows times an `Fp8Weight` (weights.py), any number of tokens.

Errors raise ValueError / TypeError (arguments) or ShadyHipError (a call).
"""
from __future__ import annotations

import torch

from ._lib import ST_F16, ST_F32, ST_FLAG_NORM_PLUS_ONE, call
from .weights import FP8_BLOCK, Fp8Weight, fp8_blocks

_F32, _F16, _F8 = torch.float32, torch.float16, torch.float8_e4m3fn
_DT = {_F32: ST_F32, _F16: ST_F16}


def _on(gpu, t, name: str) -> None:
    if t.device != gpu.device:
        raise ValueError(f"{name}: on {t.device}, the context's device is {gpu.device}")


def _act_rows(gpu, t, name: str, m: int, k: int) -> tuple[int, int, int]:
    """(address, dtype, elements from one row to the next) of `t` [m, k],
    float32 or float16, a row's elements side by side."""
    d = _DT.get(t.dtype)
    if d is None:
        raise TypeError(f"{name}: dtype {t.dtype} (need float32 or float16)")
    if t.shape != (m, k):
        raise ValueError(f"{name}: shape {tuple(t.shape)} (need [{m}, {k}])")
    _on(gpu, t, name)
    s = t.stride()
    if s[1] != 1 and k > 1:
        raise ValueError(f"{name}: strides {s} (need rows of adjacent elements)")
    return t.data_ptr(), d, s[0] if m > 1 else max(s[0], k)


class Fp8Rows:
    """M quantised rows of K dims: data e4m3 [M, K], scale f32 [ceil(K / 128),
    M] (the scales of one block of dims side by side by token; a part of
    wider rows will do). Row m's dim k is data[m, k] * scale[k // 128, m]."""

    def __init__(self, gpu, m: int, k: int):
        """Allocates rows on the context's device; what they hold is undefined."""
        if m < 1 or k < 16 or k % 16:
            raise ValueError(f"Fp8Rows: {m} rows of {k} dims (a multiple of 16)")
        self._take(torch.empty(m, k, dtype=_F8, device=gpu.device), torch.empty(fp8_blocks(k), m, device=gpu.device))

    @classmethod
    def of(cls, data, scale) -> "Fp8Rows":
        """Rows over the caller's tensors."""
        self = cls.__new__(cls)
        self._take(data, scale)
        return self

    def _take(self, data, scale):
        if data.dtype is not _F8 or scale.dtype is not _F32:
            raise TypeError(f"Fp8Rows: data {data.dtype} (need float8_e4m3fn), scale {scale.dtype} (need float32)")
        if data.dim() != 2 or not data.is_contiguous() or data.shape[1] % 16 or data.numel() == 0:
            raise ValueError(f"Fp8Rows: data {tuple(data.shape)} (need contiguous [M, K], K a multiple of 16)")
        m, k = data.shape
        if scale.shape != (fp8_blocks(k), m) or (m > 1 and scale.stride(1) != 1) or scale.device != data.device:
            raise ValueError(f"Fp8Rows: scale {tuple(scale.shape)}, strides {scale.stride()}, on {scale.device} (need "
                             f"[{fp8_blocks(k)}, {m}], a block's side by side, on {data.device})")
        self.data, self.scale, self.M, self.K = data, scale, m, k
        self.stride = max(scale.stride(0), m) if scale.shape[0] > 1 else m
        self._at, self._scale_at, self.device = data.data_ptr(), scale.data_ptr(), data.device

    def __getitem__(self, rows: slice) -> "Fp8Rows":
        """Rows [a:b] of these, sharing their memory."""
        return Fp8Rows.of(self.data[rows], self.scale[:, rows])

    def dequantise(self):
        """The values, float32 [M, K] (torch ops)."""
        s = self.scale.t().repeat_interleave(FP8_BLOCK, 1)[:, : self.K]
        return self.data.float() * s


def add_rmsnorm(gpu, residual, weight, x=None, y=None, rows: Fp8Rows | None = None, residual_out=None, eps: float = 1e-6,
                one_plus: bool = False) -> None:
    """residual_out = residual + x (None: in place; x None: no addition), and
    the RMS norm of that sum times weight [D] f32 (one_plus: 1 + weight) into
    y [M, D] (float32 or float16), into `rows` (quantised), or both: the
    reference's rmsnorm and add_rmsnorm (src/model.rs:685-691, 799-802).

    residual, residual_out (one dtype) and x [M, D] float32 or float16, rows
    of adjacent elements. The norm is of the sum before it is rounded to the
    residual's type."""
    if residual.dim() != 2:
        raise ValueError(f"residual: shape {tuple(residual.shape)} (need [M, D])")
    m, d = residual.shape
    rp, rd, rs = _act_rows(gpu, residual, "residual", m, d)
    xp = op = yp = qp = sp = None
    xd = xs = os_ = yd = ys = ss = 0
    if x is not None:
        xp, xd, xs = _act_rows(gpu, x, "x", m, d)
        if residual_out is None:
            op, os_ = rp, rs
        else:
            if residual_out.dtype is not residual.dtype:
                raise TypeError(f"residual_out: dtype {residual_out.dtype} (need the residual's, {residual.dtype})")
            op, _, os_ = _act_rows(gpu, residual_out, "residual_out", m, d)
    elif residual_out is not None:
        raise ValueError("residual_out without x")
    if weight.dtype is not _F32 or weight.numel() != d or not weight.is_contiguous():
        raise ValueError(f"weight: {weight.dtype} {tuple(weight.shape)} (need contiguous float32 [{d}])")
    _on(gpu, weight, "weight")
    if y is not None:
        yp, yd, ys = _act_rows(gpu, y, "y", m, d)
    if rows is not None:
        if rows.M != m or rows.K != d:
            raise ValueError(f"rows: [{rows.M}, {rows.K}] (need [{m}, {d}])")
        _on(gpu, rows, "rows")
        qp, sp, ss = rows._at, rows._scale_at, rows.stride
    elif y is None:
        raise ValueError("add_rmsnorm: neither y nor rows")
    gpu.sync_stream()
    call("st_add_rmsnorm", gpu.handle, rp, rd, rs, xp, xd, xs, op, os_, weight.data_ptr(), eps, yp, yd, ys, qp, sp, ss, m, d,
         ST_FLAG_NORM_PLUS_ONE if one_plus else 0)


def fp8_quant(gpu, a, rows: Fp8Rows, b=None) -> None:
    """rows = a, or silu(a) * b, quantised; a and b [M, K] float32 or float16
    (one dtype), rows of adjacent elements (the halves of a gate|up row will
    do)."""
    ap, ad, as_ = _act_rows(gpu, a, "a", rows.M, rows.K)
    bp, bs = None, 0
    if b is not None:
        if b.dtype is not a.dtype:
            raise TypeError(f"b: dtype {b.dtype} (need a's, {a.dtype})")
        bp, _, bs = _act_rows(gpu, b, "b", rows.M, rows.K)
    _on(gpu, rows, "rows")
    gpu.sync_stream()
    call("st_fp8_quant", gpu.handle, ap, bp, ad, as_, bs, rows._at, rows._scale_at, rows.stride, rows.M, rows.K)


def fp8_gemm(gpu, rows: Fp8Rows, w: Fp8Weight, y) -> None:
    """y [M, N] (float32 or float16) = rows . w^T, M of any size."""
    if rows.K != w.K:
        raise ValueError(f"rows of {rows.K} dims, a weight of {w.K}")
    d = _DT.get(y.dtype)
    if d is None:
        raise TypeError(f"y: dtype {y.dtype} (need float32 or float16)")
    if y.numel() != rows.M * w.N or not y.is_contiguous():
        raise ValueError(f"y: {tuple(y.shape)}, strides {y.stride()} (need contiguous [{rows.M}, {w.N}])")
    _on(gpu, y, "y")
    _on(gpu, rows, "rows")
    _on(gpu, w.w, "w")
    gpu.sync_stream()
    call("st_fp8_gemm", gpu.handle, rows._at, rows._scale_at, rows.stride, w.w.data_ptr(), w.scale.data_ptr(), y.data_ptr(), d, rows.M,
         w.K, w.N)
