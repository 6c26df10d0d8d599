"""Calls of the 8-bit floating point operators that are refused, on the CPU:
scales that overlap, outputs in the buffers of inputs, layers that are not
built, the shapes that linear() takes."""
import ctypes

import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import F8, weight_of
from shady_thinker_amd._lib import ST_F16, ST_F32, ST_FLAG_TILED, lib

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


# --------------------------------------------------- layers that are not built
def fp8_weight(n, k):
    return sta.Fp8Weight.of(*weight_of(torch.ones(n, k)))


def gptq_weight(n, k):
    return sta.GptqWeight(torch.zeros(n * k // 8, dtype=torch.int32), torch.zeros(k // 128, n, dtype=torch.float16), None, None, k, n, 128,
                          ST_FLAG_TILED)


DELTA = {"linear_attn.in_proj_qkv": (384, 256), "linear_attn.in_proj_z": (128, 256), "linear_attn.out_proj": (256, 128)}
MLP = {"mlp.gate_proj": (512, 256), "mlp.up_proj": (512, 256), "mlp.down_proj": (256, 512)}
ATTENTION = {f"self_attn.{p}_proj": (256, 256) for p in "qkvo"}


@pytest.mark.parametrize("e4m3", [{*DELTA, *MLP}, {*DELTA}, {*MLP}, {"linear_attn.out_proj"}, {"mlp.down_proj"}])
def test_delta_net_layers_in_e4m3(e4m3):
    """A hybrid model's linear attention in e4m3 is refused by its name."""
    linears = {f"model.layers.4.{name}": (fp8_weight if name in e4m3 else gptq_weight)(*s) for name, s in {**DELTA, **MLP}.items()}
    with pytest.raises(TypeError, match=r"DeltaNetLinears: model\.layers\.4\.\S+ is an e4m3 weight"):
        sta.layer_from_linears(linears, 4)


@pytest.mark.parametrize("e4m3", [{*MLP}, {"self_attn.o_proj"}])
def test_mixed_layers(e4m3):
    linears = {f"model.layers.0.{name}": (fp8_weight if name in e4m3 else gptq_weight)(*s) for name, s in {**ATTENTION, **MLP}.items()}
    with pytest.raises(TypeError, match=r"DecoderLinears: model\.layers\.0\.\S+ is an e4m3 weight"):
        sta.layer_from_linears(linears, 0)


def test_layers_of_e4m3_by_hand():
    g, f = [gptq_weight(*s) for s in (*DELTA.values(), *MLP.values())], [fp8_weight(*s) for s in (*DELTA.values(), *MLP.values())]
    sta.DeltaNetLinears(*g)
    for i in range(6):
        with pytest.raises(TypeError, match="is an e4m3 weight"):
            sta.DeltaNetLinears(*g[:i], f[i], *g[i + 1:])
    g, f = [gptq_weight(*s) for s in (*ATTENTION.values(), *MLP.values())], [fp8_weight(*s) for s in (*ATTENTION.values(), *MLP.values())]
    sta.DecoderLinears(*g)
    for i in range(7):
        with pytest.raises(TypeError, match="is an e4m3 weight"):
            sta.DecoderLinears(*g[:i], f[i], *g[i + 1:])
        with pytest.raises(TypeError, match="need e4m3"):
            sta.Fp8DecoderLinears(*f[:i], g[i], *f[i + 1:])


# --------------------------------------------------------------------- linear()
class NoGpu:
    handle = None
    device = torch.device("cpu")

    def sync_stream(self):
        pass


@pytest.mark.parametrize("xs,ys", [((144,), (40,)), ((3, 144), (3, 40)), ((2, 3, 144), (2, 3, 40)), ((3, 144), (130,))])
def test_linear_shapes(monkeypatch, xs, ys):
    seen = []
    monkeypatch.setattr(sta.fp8, "call", lambda name, *a: seen.append((name, a[-3:])))
    sta.linear(NoGpu(), torch.zeros(xs), fp8_weight(40, 144), torch.zeros(ys))
    m = torch.zeros(xs).numel() // 144
    assert seen[0][0] == "st_fp8_quant" and seen[0][1][-2:] == (m, 144) and seen[1] == ("st_fp8_gemm", (m, 144, 40))


def test_linear_of_a_part_of_wider_rows(monkeypatch):
    seen = []
    monkeypatch.setattr(sta.fp8, "call", lambda name, *a: seen.append(a))
    sta.linear(NoGpu(), torch.zeros(3, 288)[:, :144], fp8_weight(40, 144), torch.zeros(3, 40))
    assert seen[0][4] == 288  # (a_stride)


@pytest.mark.parametrize("x,y", [
    (torch.zeros(3, 143), torch.zeros(3, 40)), (torch.zeros(3, 144), torch.zeros(3, 39)), (torch.zeros(3, 144).int(), torch.zeros(3, 40)),
    (torch.zeros(144, 3).t(), torch.zeros(3, 40)), (torch.zeros(2, 2, 288)[..., :144], torch.zeros(4, 40)), (torch.zeros(3, 144), torch.zeros(40, 3).t()), (torch.zeros(3, 144), torch.zeros(3, 40).double())])
def test_linear_refusals(monkeypatch, x, y):
    monkeypatch.setattr(sta.fp8, "call", lambda *a: None)
    with pytest.raises((ValueError, TypeError)):
        sta.linear(NoGpu(), x, fp8_weight(40, 144), y)
