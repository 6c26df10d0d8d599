"""The 8-bit floating point operators in the framework's own paths: a layer's
decode and prefill, a DecoderStack with and without ResidualNorms, eager and
captured, the example."""
import os
import sys

import numpy as np
import pytest
import torch

import shady_thinker_amd as sta
from fp8_util import U, check_product, check_rows, weight_of
from test_gpu_fp8 import norm_err, rand, silu64, silu_err

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))

pytestmark = pytest.mark.gpu

H, Q, KV, I, V = 400, 256, 128, 384, 1003
F32, F16 = torch.float32, torch.float16


def fp8_layer(seed):
    mk = lambda s, n, k: sta.Fp8Weight.of(*weight_of(rand(seed + s, n, k) / k**0.5))
    return sta.Fp8DecoderLinears(mk(0, Q, H), mk(1, KV, H), mk(2, KV, H), mk(3, H, Q), mk(4, I, H), mk(5, I, H), mk(6, H, I))


def gptq_layer(gpu, seed):
    rng = np.random.default_rng(seed)

    def mk(k, n):
        qw = rng.integers(0, 2**32, (k // 8, n), dtype=np.uint32)
        return sta.GptqWeight.upload(gpu, qw, (rng.uniform(0.5, 1.0, (k // 64, n)) * 0.2 / k**0.5).astype(np.float16), 64)

    return sta.DecoderLinears(mk(384, Q), mk(384, KV), mk(384, KV), mk(Q, 384), mk(384, I), mk(384, I), mk(I, 384))


def prod(rows, w, y):
    check_product(y, rows.data, rows.scale, w.w, w.scale)


@pytest.mark.parametrize("m,dtype", [(1, F32), (32, F32), (7, F16), (100, F16), (300, F16)])
def test_layer(gpu, m, dtype):
    """decode and prefill: from float activations, and from quantised rows the same bits."""
    L = fp8_layer(10)
    x, attn, xm = rand(1, m, H, dtype=dtype), rand(2, m, Q, dtype=dtype), rand(3, m, H, dtype=dtype)
    mk = lambda n: torch.empty(m, n, dtype=dtype, device=gpu.device)
    qkv, o, gu, down = mk(Q + 2 * KV), mk(H), mk(2 * I), mk(H)
    (L.decode if dtype is F32 else L.prefill)(gpu, x, attn, qkv, o, gu, down, xm)
    rx, ra, rm, rh = (sta.Fp8Rows(gpu, m, n) for n in (H, Q, H, I))
    sta.fp8_quant(gpu, x, rx), sta.fp8_quant(gpu, attn, ra), sta.fp8_quant(gpu, xm, rm)
    prod(rx, L.qkv, qkv), prod(ra, L.o, o), prod(rm, L.gate_up, gu)
    sta.fp8_quant(gpu, gu[:, :I], rh, gu[:, I:])
    prod(rh, L.down, down)
    again = [torch.empty_like(t) for t in (qkv, o, gu, down)]
    L.decode(gpu, rx, ra, *again, rm)
    assert all(torch.equal(a, b) for a, b in zip(again, (qkv, o, gu, down)))
    L.decode(gpu, rx, ra, *again)  # (the MLP reads x)
    prod(rx, L.gate_up, again[2])


class Norms(sta.ResidualNorms):
    def __init__(self, gpu, stack, batch, x0):
        h = stack.layers[0].hidden
        mk = lambda s: 1.0 + 0.1 * rand(s, h)
        n = len(stack.layers)
        self.init_norms(gpu, stack, batch, [mk(50 + i) for i in range(n)], [mk(70 + i) for i in range(n)], mk(90), one_plus=False)
        self.x0, self.seen = x0, []

    def embed(self, b):
        self.residual.copy_(self.x0)

    def attention(self, i, b):
        self.seen.append((self.residual.clone(), b.x8 and (b.x8.data.clone(), b.x8.scale.clone()), b.x.clone()))
        b.attn.copy_(b.qkv[:, :b.attn.shape[1]])


def norm64(r, w):
    r = r.double().cpu()
    return r / torch.sqrt((r * r).mean(-1, keepdim=True) + 1e-6) * w.double().cpu()


@pytest.mark.parametrize("batch", [1, 5, 32])
@pytest.mark.parametrize("head", ["fp8", "bf16"])
def test_stack_step(gpu, batch, head):
    """One step of an e4m3 layer with ResidualNorms, each operation against 64
    bits of what it read."""
    L = fp8_layer(20)
    lm = sta.Fp8Weight.of(*weight_of(rand(30, V, H))) if head == "fp8" else rand(30, 1000, H).to(torch.bfloat16)
    stack = sta.DecoderStack([L], lm)
    assert stack.vocab == (V if head == "fp8" else 1000) and stack.nbytes() > 0
    hooks = Norms(gpu, stack, batch, rand(40, batch, H))
    b = stack.buffers(gpu, batch)
    stack.step(gpu, b, hooks)
    (r0, (d0, s0), _), = hooks.seen
    assert torch.equal(r0, hooks.x0)
    check_rows(d0, s0, norm64(r0, hooks._attention_norms[0]), norm_err(H))
    check_product(b.qkv, d0, s0, L.qkv.w, L.qkv.scale)
    check_rows(b.attn8.data, b.attn8.scale, b.attn.double().cpu(), 0.0)
    prod(b.attn8, L.o, b.o)
    r1 = r0.double().cpu() + b.o.double().cpu()
    check_rows(b.xm8.data, b.xm8.scale, norm64(r1, hooks._mlp_norms[0]), norm_err(H))
    prod(b.xm8, L.gate_up, b.gate_up)
    g = b.gate_up[:, :I]
    check_rows(b.h8.data, b.h8.scale, silu64(g.double().cpu()) * b.gate_up[:, I:].double().cpu(), silu_err(g))
    prod(b.h8, L.down, b.down)
    r2 = r1 + b.down.double().cpu()
    assert ((hooks.residual.double().cpu() - r2).abs() <= 4 * U * (r1.abs() + r2.abs())).all()
    if head == "fp8":
        prod(b.x8, lm, b.logits)
    else:
        want = b.x.double().cpu() @ lm.double().cpu().t()
        assert ((b.logits.double().cpu() - want).norm() / want.norm()) < 1e-5


def test_stack_without_norms(gpu):
    """Hooks that fill b.x and b.xm: the step quantises them."""
    L = fp8_layer(20)
    stack = sta.DecoderStack([L, fp8_layer(21)], sta.Fp8Weight.of(*weight_of(rand(30, V, H))))
    b = stack.buffers(gpu, 3)
    b.x.copy_(rand(1, 3, H)), b.xm.copy_(rand(2, 3, H)), b._attn_flat.copy_(rand(3, 3 * Q).view(-1))
    stack.step(gpu, b)
    rows = sta.Fp8Rows(gpu, 3, H)
    sta.fp8_quant(gpu, b.xm, rows)
    prod(rows, stack.layers[1].gate_up, b.gate_up)
    sta.fp8_quant(gpu, b.x, rows)
    prod(rows, stack.lm_head, b.logits)


def test_norms_of_other_layers(gpu):
    """ResidualNorms before GPTQ linears, and a stack of both kinds: float32
    rows for one, quantised ones for the other; captured, every replay the
    eager step's bits."""
    H2 = 384
    mk = lambda s, n, k: sta.Fp8Weight.of(*weight_of(rand(s, n, k) / k**0.5))
    f8 = sta.Fp8DecoderLinears(mk(0, Q, H2), mk(1, KV, H2), mk(2, KV, H2), mk(3, H2, Q), mk(4, I, H2), mk(5, I, H2), mk(6, H2, I))
    for layers in ([gptq_layer(gpu, 1)], [gptq_layer(gpu, 1), f8, gptq_layer(gpu, 2)], [f8, gptq_layer(gpu, 2)]):
        stack = sta.DecoderStack(layers, rand(30, 1000, H2).to(torch.bfloat16))
        hooks = Norms(gpu, stack, 4, rand(40, 4, H2))
        b = stack.buffers(gpu, 4)
        stack.step(gpu, b, hooks)
        for i, (r, rows, x) in enumerate(hooks.seen):
            want = norm64(r, hooks._attention_norms[i])
            if layers[i].fp8:
                check_rows(*rows, want, norm_err(H2))
            else:
                assert ((x.double().cpu() - want).abs() <= want.abs() * (norm_err(H2) + U)).all()
        want = b.logits.clone()
        hooks.attention = lambda i, b: b.attn.copy_(b.qkv[:, :b.attn.shape[1]])
        graph = stack.capture(gpu, b, hooks)
        for _ in range(3):
            b.logits.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(b.logits, want)
        graph.release()


@pytest.mark.parametrize("batch", [1, 3])
def test_example(gpu, batch):
    """examples/decode.py --fp8: the captured steps are the eager ones'."""
    import decode as ex

    stack, embedding = ex.build(gpu, fp8=True)
    prompts = torch.arange(batch * 5, dtype=torch.int32, device=gpu.device).view(batch, 5) * 37 % ex.VOCAB
    ids, lps, logits = ex.decode(gpu, stack, embedding, prompts, 20)
    want_ids, want_lps, want_logits = ex.decode(gpu, stack, embedding, prompts, 20, graph=False)
    assert torch.equal(ids, want_ids) and torch.equal(lps, want_lps) and torch.equal(logits, want_logits)
    assert torch.isfinite(logits).all() and torch.equal(ids[:, -1].long(), logits.argmax(-1))


def test_checkpoint(gpu, tmp_path):
    """A block-scaled checkpoint's linears, loaded and run as a layer."""
    from safetensors.torch import save_file

    names = {"self_attn.q_proj": (Q, H), "self_attn.k_proj": (KV, H), "self_attn.v_proj": (KV, H), "self_attn.o_proj": (H, Q),
             "mlp.gate_proj": (I, H), "mlp.up_proj": (I, H), "mlp.down_proj": (H, I)}
    tensors = {}
    for j, (name, (n, k)) in enumerate(names.items()):
        w, s = weight_of(rand(j, n, k))
        tensors[f"model.layers.0.{name}.weight"], tensors[f"model.layers.0.{name}.weight_scale_inv"] = w.cpu(), s.cpu()
    tensors["lm_head.weight"] = rand(9, 64, H).to(torch.bfloat16).cpu()
    tensors["model.norm.weight"] = torch.ones(H)
    save_file(tensors, tmp_path / "model.safetensors")
    linears, bf16 = sta.load_fp8_checkpoint(gpu, str(tmp_path))
    assert len(linears) == 7 and list(bf16) == ["lm_head.weight"]
    L = sta.layer_from_linears(linears, 0)
    assert isinstance(L, sta.Fp8DecoderLinears)
    x, y = rand(20, 2, H), torch.empty(2, L.qkv.N, device=gpu.device)
    rows = sta.Fp8Rows(gpu, 2, H)
    sta.fp8_quant(gpu, x, rows)
    sta.fp8_gemm(gpu, rows, L.qkv, y)
    parts = [f"model.layers.0.self_attn.{p}_proj.weight" for p in "qkv"]
    w = torch.cat([tensors[p].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
    check_product(y, rows.data, rows.scale, w, torch.cat([tensors[p + "_scale_inv"] for p in parts]))
