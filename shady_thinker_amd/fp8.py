"""Linears in 8-bit floating point: rows of e4m3 activations, the norm and the
activation that make them, and their product with block-scaled weights.

No reference counterpart but for the norms (src/model.rs:685-691, 799-802,
820-823: rmsnorm.wgsl, add_rmsnorm.wgsl). Entry points of libshady_hip like
the other linears, on torch device tensors and torch's current stream:

* `Fp8Rows`: quantised rows, e4m3 with a scale for each token and 128 dims;
* `add_rmsnorm`: residual addition and norm, to such rows, to f32 / f16, or both;
* `fp8_quant`: rows, or silu(a) * b, to such rows;
* `fp8_gemm`: rows times an `Fp8Weight` (weights.py), any number of tokens;
* `ResidualNorms`: the residual and norms of a model as a DecoderStack's hooks.

Errors raise ValueError / TypeError (arguments) or ShadyHipError (a call).
"""
from __future__ import annotations

import torch

from ._lib import ST_F16, ST_F32, ST_FLAG_NORM_PLUS_ONE, call
from .weights import FP8_BLOCK, Fp8Weight, fp8_blocks

_F32, _F16, _F8 = torch.float32, torch.float16, torch.float8_e4m3fn
_DT = {_F32: ST_F32, _F16: ST_F16}


# As in model.py, what is right in the common case is found by few cheap
# tensor queries (a small call's kernel takes 3 us); what they do not pass goes
# to a function that finds a permitted form or says what is wrong.
def _device(gpu) -> int:
    i = gpu.device.index
    return -1 if i is None else i


def _elsewhere(gpu, name: str, device):
    raise ValueError(f"{name}: on {device}, the context's device is {gpu.device}")


def _row_stride(gpu, t, name: str, m: int, k: int) -> int:
    """Elements from one row to the next of a `t` [m, k] that the quick checks
    did not pass: a part of wider rows, or refused."""
    if t.dtype not in _DT:
        raise TypeError(f"{name}: dtype {t.dtype} (need float32 or float16)")
    if t.shape != (m, k):
        raise ValueError(f"{name}: shape {tuple(t.shape)} (need [{m}, {k}])")
    if t.get_device() != _device(gpu):
        _elsewhere(gpu, name, t.device)
    s = t.stride()
    if s[1] != 1:
        raise ValueError(f"{name}: strides {s} (need rows of adjacent elements)")
    return s[0] if m > 1 else max(s[0], k)


class Fp8Rows:
    """M quantised rows of K dims: data e4m3 [M, K], scale f32 [ceil(K / 128),
    M] (the scales of one block of dims side by side by token; a part of
    wider rows will do). Row m's dim k is data[m, k] * scale[k // 128, m].
    Calls use the memory that both have when the rows are made: it is theirs as
    long as the rows are used (no set_, resize_ or other .data)."""

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
        self.stride = scale.stride(0) if scale.shape[0] > 1 else m
        if self.stride < m:
            raise ValueError(f"Fp8Rows: scale {tuple(scale.shape)}, strides {scale.stride()}: a block's scales overlap the next one's")
        self._data, self._scale, self.M, self.K = data, scale, m, k
        self._at, self._scale_at, self._device = data.data_ptr(), scale.data_ptr(), data.get_device()

    @property
    def data(self):
        return self._data

    @property
    def scale(self):
        return self._scale

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
    shape, dev = residual.shape, _device(gpu)
    if len(shape) != 2:
        raise ValueError(f"residual: shape {tuple(shape)} (need [M, D])")
    m, d = shape
    rd = _DT.get(residual.dtype)
    rs = os_ = xs = ys = d
    if rd is None or residual.get_device() != dev or not residual.is_contiguous():
        rs = os_ = _row_stride(gpu, residual, "residual", m, d)
    rp = residual.data_ptr()
    xp = op = yp = qp = sp = None
    xd = yd = ss = 0
    if x is not None:
        xd = _DT.get(x.dtype)
        if xd is None or x.shape != shape or x.get_device() != dev or not x.is_contiguous():
            xs = _row_stride(gpu, x, "x", m, d)
        xp, op = x.data_ptr(), rp
        if residual_out is not None:
            if residual_out.dtype is not residual.dtype:
                raise TypeError(f"residual_out: dtype {residual_out.dtype} (need the residual's, {residual.dtype})")
            os_ = d
            if residual_out.shape != shape or residual_out.get_device() != dev or not residual_out.is_contiguous():
                os_ = _row_stride(gpu, residual_out, "residual_out", m, d)
            op = residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out without x")
    if weight.dtype is not _F32 or weight.numel() != d or not weight.is_contiguous():
        raise ValueError(f"weight: {weight.dtype} {tuple(weight.shape)} (need contiguous float32 [{d}])")
    if weight.get_device() != dev:
        _elsewhere(gpu, "weight", weight.device)
    if y is not None:
        yd = _DT.get(y.dtype)
        if yd is None or y.shape != shape or y.get_device() != dev or not y.is_contiguous():
            ys = _row_stride(gpu, y, "y", m, d)
        yp = y.data_ptr()
    if rows is not None:
        if rows.M != m or rows.K != d or rows._device != dev:
            raise ValueError(f"rows: [{rows.M}, {rows.K}] on {rows.data.device} (need [{m}, {d}] on {gpu.device})")
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
    m, k, dev = rows.M, rows.K, rows._device
    if dev != _device(gpu):
        _elsewhere(gpu, "rows", rows.data.device)
    ad, as_, bp, bs = _DT.get(a.dtype), k, None, k
    if ad is None or a.shape != (m, k) or a.get_device() != dev or not a.is_contiguous():
        as_ = _row_stride(gpu, a, "a", m, k)
    if b is not None:
        if b.dtype is not a.dtype:
            raise TypeError(f"b: dtype {b.dtype} (need a's, {a.dtype})")
        if b.shape != (m, k) or b.get_device() != dev or not b.is_contiguous():
            bs = _row_stride(gpu, b, "b", m, k)
        bp = b.data_ptr()
    gpu.sync_stream()
    call("st_fp8_quant", gpu.handle, a.data_ptr(), bp, ad, as_, bs, rows._at, rows._scale_at, rows.stride, m, k)


def fp8_gemm(gpu, rows: Fp8Rows, w: Fp8Weight, y) -> None:
    """y [M, N] (float32 or float16) = rows . w^T, M of any size. float16 y of
    more than 64 tokens: the 8-bit matrix instruction cuts small products beside
    large ones (st_fp8_gemm in the header says how far), unless
    gpu.set_tune("FP8_EXACT", 1), at up to twice the time."""
    m, k, n, dev = rows.M, w.K, w.N, rows._device
    d = _DT.get(y.dtype)
    if (d is None or rows.K != k or y.shape != (m, n) or not y.is_contiguous() or y.get_device() != dev or w._device != dev
            or _device(gpu) != dev):
        if d is None:
            raise TypeError(f"y: dtype {y.dtype} (need float32 or float16)")
        raise ValueError(f"y {tuple(y.shape)}, strides {y.stride()}, on {y.device} = rows [{m}, {rows.K}] on {rows.data.device} . weight "
                         f"[{n}, {k}] on {w.w.device}: need a contiguous [{m}, {n}], all on {gpu.device}")
    gpu.sync_stream()
    call("st_fp8_gemm", gpu.handle, rows._at, rows._scale_at, rows.stride, w._at, w._scale_at, y.data_ptr(), d, m, k, n)


class ResidualNorms:
    """The residual stream of a model and the norms before its linears, as a
    DecoderStack's hooks (src/model.rs:685-691, 799-802, 820-823): one launch
    before each layer's attention side, one before its MLP, one before the
    lm_head. Layers that read quantised rows get them from the norm.

    A subclass adds `embed(b)`, which fills `residual` [batch, hidden] (float32)
    at the start of a step, and may be a PagedAttention too. attention and mlp:
    each layer's norm weights [hidden] float32; last: the lm_head's; one_plus:
    they hold w - 1."""

    fills_rows = True

    def init_norms(self, gpu, stack, batch: int, attention, mlp, last, eps: float = 1e-6, one_plus: bool = False) -> None:
        n = len(stack.layers)
        if len(attention) != n or len(mlp) != n:
            raise ValueError(f"ResidualNorms: {len(attention)} and {len(mlp)} norm weights for {n} layers")
        self.residual = torch.zeros(batch, stack.layers[0].hidden, device=gpu.device)
        self._norms = (gpu, eps, one_plus)
        self._attention_norms, self._mlp_norms, self._last_norm = attention, mlp, last
        self._fp8 = [L.fp8 for L in stack.layers] + [isinstance(stack.lm_head, Fp8Weight)]

    def embed(self, b) -> None:
        raise NotImplementedError("ResidualNorms: embed(b) fills the residual")

    def _norm(self, weight, x, fp8, y, rows) -> None:
        gpu, eps, one_plus = self._norms
        add_rmsnorm(gpu, self.residual, weight, x, None if fp8 else y, rows if fp8 else None, eps=eps, one_plus=one_plus)

    def pre_attention(self, i, b) -> None:
        if i == 0:
            self.embed(b)
        self._norm(self._attention_norms[i], b.down if i else None, self._fp8[i], b.x, b.x8)

    def post_attention(self, i, b) -> None:
        self._norm(self._mlp_norms[i], b.o, self._fp8[i], b.xm, b.xm8)

    def final(self, b) -> None:
        self._norm(self._last_norm, b.down, self._fp8[-1], b.x, b.x8)
