"""Refusals and host logic of the 8-bit floating point calls (CPU, no GPU):
the Python helpers' with a stand-in for the context, and the C entry points'
own, which look at their arguments before they touch the context or a GPU."""
import ctypes

import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import F8, rows_of, weight_of
from shady_thinker_amd._lib import ST_BF16, ST_F16, ST_F32, lib

ST_ERR_INVALID, ST_ERR_SHAPE, ST_ERR_ALIGN = 1, 2, 3  # (st_status)
F32, F16 = torch.float32, torch.float16
M, K, N = 3, 144, 40


class NoGpu:
    handle = None
    device = torch.device("cpu")

    def sync_stream(self):
        pass


G = NoGpu()


def rows(m=M, k=K):
    return sta.Fp8Rows(G, m, k)


def weight(n=N, k=K):
    return sta.Fp8Weight.of(*weight_of(torch.ones(n, k)))


# ------------------------------------------------------------ Python helpers
@pytest.mark.parametrize("m,k", [(0, 16), (1, 0), (1, 8), (2, 130)])
def test_rows_sizes(m, k):
    with pytest.raises(ValueError):
        sta.Fp8Rows(G, m, k)


@pytest.mark.parametrize("data,scale", [
    (torch.zeros(M, K, dtype=torch.uint8), torch.zeros(2, M)), (torch.zeros(M, K).to(F8), torch.zeros(2, M, dtype=F16)),
    (torch.zeros(M, K).to(F8), torch.zeros(M, 2)), (torch.zeros(M, K).to(F8), torch.zeros(1, M)), (torch.zeros(M * K).to(F8), torch.zeros(2, M)),
    (torch.zeros(M, 2 * K).to(F8)[:, :K], torch.zeros(2, M)), (torch.zeros(M, 136).to(F8), torch.zeros(2, M)),
    (torch.zeros(M, K).to(F8), torch.zeros(M, 2).t()), (torch.zeros(0, K).to(F8), torch.zeros(2, 0)),
    (torch.zeros(M, K).to(F8), torch.zeros(2, M, device="meta"))])
def test_rows_refusals(data, scale):
    with pytest.raises((ValueError, TypeError)):
        sta.Fp8Rows.of(data, scale)


def test_rows_slices():
    y = torch.randn(9, 300 // 16 * 16)
    r = sta.Fp8Rows.of(*rows_of(y))
    assert torch.allclose(r.dequantise(), y, rtol=2.0**-4, atol=y.abs().max().item() / 448 * 2.0**-10)
    part = r[2:7]
    assert (part.M, part.K, part.stride) == (5, r.K, 9)
    assert torch.equal(part.dequantise(), r.dequantise()[2:7])
    assert r[4:5].stride == 9 and r[4:5].M == 1


@pytest.mark.parametrize("w,scale", [
    (torch.zeros(N, K, dtype=torch.int8), torch.zeros(1, 2)), (torch.zeros(N, K).to(F8), torch.zeros(1, 2, dtype=torch.bfloat16)),
    (torch.zeros(N, K).to(F8), torch.zeros(2, 1)), (torch.zeros(N, K).to(F8), torch.zeros(2)), (torch.zeros(N, K + 8).to(F8), torch.zeros(1, 2)),
    (torch.zeros(N * K).to(F8), torch.zeros(1, 2)), (torch.zeros(K, N).to(F8).t(), torch.zeros(1, 2)),
    (torch.zeros(N, K).to(F8), torch.zeros(1, 4)[:, ::2])])
def test_weight_refusals(w, scale):
    with pytest.raises((ValueError, TypeError)):
        sta.Fp8Weight.of(w, scale)


def test_tensors_stay():
    """What a handle's pointers are of is not exchanged, and a weight is what it
    says, however it is made."""
    r, w = rows(), weight()
    for obj, name in ((r, "data"), (r, "scale"), (w, "w"), (w, "scale"), (w, "K")):
        with pytest.raises(AttributeError):
            setattr(obj, name, getattr(obj, name))
    for k, n in ((K + 16, N), (K, N + 1), (N, K)):
        with pytest.raises(ValueError):
            sta.Fp8Weight(w.w, w.scale, k, n)


def test_weight_upload_and_cat():
    a, b = weight_of(torch.randn(256, K)), weight_of(torch.randn(40, K))
    w = sta.Fp8Weight.cat([sta.Fp8Weight.upload(G, *a), sta.Fp8Weight.upload(G, b[0], b[1].to(torch.bfloat16))])
    assert (w.N, w.K, tuple(w.scale.shape), w.nbytes) == (296, K, (3, 2), 296 * K + 24)
    assert torch.equal(w.w.float(), torch.cat([a[0].float(), b[0].float()])) and torch.equal(w.scale[:2], a[1])
    with pytest.raises(ValueError):
        sta.Fp8Weight.cat([weight(40), weight(128)])
    with pytest.raises(ValueError):
        sta.Fp8Weight.cat([weight(128), weight(128, 160)])


def norm(**kw):
    a = dict(residual=torch.zeros(M, K), weight=torch.zeros(K), x=torch.zeros(M, K), y=torch.zeros(M, K), rows=rows())
    a.update(kw)
    sta.add_rmsnorm(G, a.pop("residual"), a.pop("weight"), **a)


@pytest.mark.parametrize("kw", [
    dict(residual=torch.zeros(M * K)), dict(residual=torch.zeros(M, K, dtype=torch.bfloat16)), dict(residual=torch.zeros(K, M).t()),
    dict(weight=torch.zeros(K - 1)), dict(weight=torch.zeros(K, dtype=F16)), dict(weight=torch.zeros(2 * K)[::2]), dict(x=torch.zeros(M, K - 16)),
    dict(x=torch.zeros(M + 1, K)), dict(x=torch.zeros(M, K, dtype=torch.int8)), dict(x=None, residual_out=torch.zeros(M, K)),
    dict(residual_out=torch.zeros(M, K, dtype=F16)), dict(residual_out=torch.zeros(M, 2 * K)), dict(y=torch.zeros(M, 2 * K)[:, ::2]),
    dict(y=torch.zeros(M, K, dtype=torch.float64)), dict(y=None, rows=None), dict(rows=rows(M + 1)), dict(rows=rows(M, K + 16))])
def test_norm_refusals(kw):
    with pytest.raises((ValueError, TypeError)):
        norm(**kw)


@pytest.mark.parametrize("kw", [
    dict(a=torch.zeros(M, K + 16)), dict(a=torch.zeros(M, K, dtype=torch.bfloat16)), dict(a=torch.zeros(M, 2 * K)[:, ::2]),
    dict(b=torch.zeros(M, K, dtype=F16)), dict(b=torch.zeros(M - 1, K))])
def test_quant_refusals(kw):
    a = dict(a=torch.zeros(M, K), rows=rows(), b=torch.zeros(M, K))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        sta.fp8_quant(G, **a)


@pytest.mark.parametrize("kw", [
    dict(rows=rows(M, K + 16)), dict(y=torch.zeros(M, N + 1)), dict(y=torch.zeros(M + 1, N)), dict(y=torch.zeros(M, N, dtype=torch.bfloat16)),
    dict(y=torch.zeros(N, M).t())])
def test_gemm_refusals(kw):
    a = dict(rows=rows(), w=weight(), y=torch.zeros(M, N))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        sta.fp8_gemm(G, **a)


def test_tensors_elsewhere():
    """Host tensors, or another device's, do not reach a context's calls."""

    class Other(NoGpu):
        device = torch.device("cuda", 1)

    g = Other()
    x, w = torch.zeros(M, K), torch.zeros(K)
    for f in (lambda: sta.add_rmsnorm(g, x, w, y=x), lambda: sta.add_rmsnorm(g, x, w, rows=rows()), lambda: sta.fp8_quant(g, x, rows()),
              lambda: sta.fp8_gemm(g, rows(), weight(), torch.zeros(M, N))):
        with pytest.raises(ValueError, match="cuda:1"):
            f()


# ------------------------------------------------------------- C entry points
CTX = ctypes.create_string_buffer(1024)  # (never used: every call below is refused before)
P, ODD, Z = 4096, 4100, None


def st(fn, *args):
    rc = getattr(lib(), fn)(*args)
    assert rc and lib().st_last_error().decode().startswith(fn)
    return rc


NORM = dict(ctx=CTX, residual=P, res_dtype=ST_F32, res_stride=K, x=P, x_dtype=ST_F32, x_stride=K, residual_out=P, out_stride=K, weight=P,
            eps=1e-6, y=P, y_dtype=ST_F32, y_stride=K, y8=P, y_scale=P, scale_stride=M, m=M, d=K, flags=0)


@pytest.mark.parametrize("kw,rc", [
    (dict(ctx=Z), ST_ERR_INVALID), (dict(residual=Z), ST_ERR_INVALID), (dict(weight=Z), ST_ERR_INVALID), (dict(x=Z), ST_ERR_INVALID),
    (dict(residual_out=Z), ST_ERR_INVALID), (dict(y8=Z), ST_ERR_INVALID), (dict(y_scale=Z), ST_ERR_INVALID),
    (dict(y=Z, y8=Z, y_scale=Z), ST_ERR_INVALID), (dict(res_dtype=ST_BF16), ST_ERR_INVALID), (dict(x_dtype=7), ST_ERR_INVALID),
    (dict(y_dtype=-1), ST_ERR_INVALID), (dict(flags=8), ST_ERR_INVALID), (dict(m=0), ST_ERR_SHAPE), (dict(d=K + 8), ST_ERR_SHAPE),
    (dict(d=0), ST_ERR_SHAPE), (dict(d=32784), ST_ERR_SHAPE), (dict(res_stride=K - 16), ST_ERR_SHAPE), (dict(x_stride=0), ST_ERR_SHAPE),
    (dict(out_stride=-K), ST_ERR_SHAPE), (dict(y_stride=K - 4), ST_ERR_SHAPE), (dict(scale_stride=M - 1), ST_ERR_SHAPE),
    (dict(res_stride=K + 2), ST_ERR_ALIGN), (dict(x_stride=K + 1), ST_ERR_ALIGN), (dict(y_dtype=ST_F16, y_stride=K + 4), ST_ERR_ALIGN),
    (dict(residual=ODD), ST_ERR_ALIGN), (dict(x=ODD), ST_ERR_ALIGN), (dict(residual_out=ODD), ST_ERR_ALIGN), (dict(weight=ODD), ST_ERR_ALIGN),
    (dict(y=ODD), ST_ERR_ALIGN), (dict(y8=ODD), ST_ERR_ALIGN), (dict(y_scale=4097), ST_ERR_ALIGN),
    (dict(x=2 * P, y=2 * P, y_stride=2 * K), ST_ERR_INVALID), (dict(x=2 * P, y=2 * P, y_dtype=ST_F16), ST_ERR_INVALID),
    (dict(x=2 * P, y=3 * P, out_stride=2 * K), ST_ERR_INVALID), (dict(x=2 * P, y=P), ST_ERR_INVALID),
    (dict(x=2 * P, y=4 * P, residual_out=4 * P), ST_ERR_INVALID), (dict(x=Z, residual_out=Z, y=P, y_stride=2 * K), ST_ERR_INVALID),
    (dict(x=2 * P, y=3 * P, m=1 << 22, scale_stride=1 << 22), ST_ERR_SHAPE)])
def test_c_norm(kw, rc):
    assert st("st_add_rmsnorm", *{**NORM, **kw}.values()) == rc


QUANT = dict(ctx=CTX, a=P, b=P, dtype=ST_F16, a_stride=K, b_stride=K, y8=P, y_scale=P, scale_stride=M, m=M, k=K)


@pytest.mark.parametrize("kw,rc", [
    (dict(ctx=Z), ST_ERR_INVALID), (dict(a=Z), ST_ERR_INVALID), (dict(y8=Z), ST_ERR_INVALID), (dict(y_scale=Z), ST_ERR_INVALID),
    (dict(dtype=ST_BF16), ST_ERR_INVALID), (dict(m=0), ST_ERR_SHAPE), (dict(m=-1), ST_ERR_SHAPE), (dict(k=K + 8), ST_ERR_SHAPE),
    (dict(k=0), ST_ERR_SHAPE), (dict(a_stride=K - 8), ST_ERR_SHAPE), (dict(b_stride=0), ST_ERR_SHAPE), (dict(scale_stride=0), ST_ERR_SHAPE),
    (dict(m=2**31 - 1, k=1 << 22, a_stride=1 << 22, b_stride=1 << 22, scale_stride=2**31), ST_ERR_SHAPE),
    (dict(m=1 << 24, scale_stride=1 << 24), ST_ERR_SHAPE), (dict(a_stride=K + 4), ST_ERR_ALIGN),
    (dict(b_stride=K + 1), ST_ERR_ALIGN), (dict(a=ODD), ST_ERR_ALIGN), (dict(b=ODD), ST_ERR_ALIGN), (dict(y8=ODD), ST_ERR_ALIGN),
    (dict(y_scale=4098), ST_ERR_ALIGN)])
def test_c_quant(kw, rc):
    assert st("st_fp8_quant", *{**QUANT, **kw}.values()) == rc


GEMM = dict(ctx=CTX, x=P, x_scale=P, scale_stride=M, w=P, w_scale=P, y=P, y_dtype=ST_F32, m=M, k=K, n=N)


@pytest.mark.parametrize("kw,rc", [
    (dict(ctx=Z), ST_ERR_INVALID), (dict(x=Z), ST_ERR_INVALID), (dict(x_scale=Z), ST_ERR_INVALID), (dict(w=Z), ST_ERR_INVALID),
    (dict(w_scale=Z), ST_ERR_INVALID), (dict(y=Z), ST_ERR_INVALID), (dict(y_dtype=ST_BF16), ST_ERR_INVALID), (dict(m=0), ST_ERR_SHAPE),
    (dict(n=0), ST_ERR_SHAPE), (dict(k=0), ST_ERR_SHAPE), (dict(k=K + 8), ST_ERR_SHAPE), (dict(k=(1 << 22) + 16), ST_ERR_SHAPE),
    (dict(scale_stride=M - 1), ST_ERR_SHAPE), (dict(m=2**31 - 1, n=2**31 - 1, scale_stride=2**31), ST_ERR_SHAPE),
    (dict(m=2**31 - 1, scale_stride=2**31), ST_ERR_SHAPE), (dict(n=2**31 - 1), ST_ERR_SHAPE), (dict(m=1 << 18, n=1 << 18, scale_stride=1 << 18), ST_ERR_SHAPE),
    (dict(x=ODD), ST_ERR_ALIGN),
    (dict(w=ODD), ST_ERR_ALIGN), (dict(y=ODD), ST_ERR_ALIGN), (dict(x_scale=4097), ST_ERR_ALIGN), (dict(w_scale=4098), ST_ERR_ALIGN)])
def test_c_gemm(kw, rc):
    assert st("st_fp8_gemm", *{**GEMM, **kw}.values()) == rc


# ------------------------------------------------------- layers and checkpoints
def parts(h=256, q=256, kv=128, i=384):
    mk = lambda n, k: weight(n, k)
    return dict(q=mk(q, h), k=mk(kv, h), v=mk(kv, h), o=mk(h, q), gate=mk(i, h), up=mk(i, h), down=mk(h, i))


def test_layer_construction():
    layer = sta.Fp8DecoderLinears(**parts())
    assert (layer.qkv.N, layer.splits, layer.gate_up.N, layer.hidden, layer.inter, layer.attn_dim) == (512, (256, 128, 128), 768, 256, 384, 256)
    assert layer.nbytes() > 0
    for name, w in (("k", weight(128, 272)), ("o", weight(272, 256)), ("up", weight(256, 256)), ("down", weight(256, 400)), ("q", weight(64, 256))):
        with pytest.raises(ValueError):
            sta.Fp8DecoderLinears(**{**parts(), name: w})


def test_layer_by_names():
    names = {"q": "self_attn.q_proj", "k": "self_attn.k_proj", "v": "self_attn.v_proj", "o": "self_attn.o_proj", "gate": "mlp.gate_proj",
             "up": "mlp.up_proj", "down": "mlp.down_proj"}
    linears = {f"model.layers.3.{names[n]}": w for n, w in parts().items()}
    assert isinstance(sta.layer_from_linears(linears, 3), sta.Fp8DecoderLinears)
    linears.pop("model.layers.3.mlp.up_proj")
    with pytest.raises(KeyError):
        sta.layer_from_linears(linears, 3)


def test_stack_refusals():
    layer = sta.Fp8DecoderLinears(**parts())
    with pytest.raises(ValueError):
        sta.DecoderStack([layer], weight(100, 272))
    with pytest.raises(ValueError):
        sta.DecoderStack([layer, sta.Fp8DecoderLinears(**parts(i=256))], weight(100, 256))
    stack = sta.DecoderStack([layer], weight(100, 256))
    with pytest.raises(ValueError):
        sta.ResidualNorms().init_norms(G, stack, 1, [], [torch.ones(256)], torch.ones(256))
    with pytest.raises(NotImplementedError):
        sta.ResidualNorms().embed(None)


def save(path, tensors, config=None):
    import json

    from safetensors.torch import save_file

    save_file(tensors, path / "model.safetensors")
    if config is not None:
        (path / "config.json").write_text(json.dumps(config))


def test_checkpoint_refusals(tmp_path):
    w, s = weight_of(torch.randn(40, 144))
    good = {"a.weight": w, "a.weight_scale_inv": s}
    save(tmp_path, good, {"quantization_config": {"weight_block_size": [128, 128]}})
    linears, bf16 = sta.load_fp8_checkpoint(G, str(tmp_path))
    assert list(linears) == ["a"] and torch.equal(linears["a"].w.float(), w.float()) and not bf16
    save(tmp_path, good, {"quantization_config": None})
    assert list(sta.load_fp8_checkpoint(G, str(tmp_path))[0]) == ["a"]
    for bad, config in (({"a.weight": w}, None), ({"a.weight_scale_inv": s}, None), ({**good, "a.weight_scale_inv": s[:, :1].contiguous()}, None),
                        (good, {"quantization_config": {"weight_block_size": [64, 128]}}),
                        (good, {"quantization_config": {"weight_block_size": None}}), ({**good, "a.weight_scale_inv": s.half()}, None)):
        (tmp_path / "config.json").unlink(missing_ok=True)
        save(tmp_path, bad, config)
        with pytest.raises((ValueError, TypeError)):
            sta.load_fp8_checkpoint(G, str(tmp_path))
