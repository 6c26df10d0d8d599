"""The operators of linears in 8-bit floating point, as measurable cases.

A weight is e4m3 [N, K] as a checkpoint holds it, with one float32 scale for
each block of 128 x 128; activations are rows of e4m3 with one float32 scale
for each token and 128 dims, side by side by token: scale [ceil(K / 128), T].
A block's scale is its largest magnitude / 448 (at least 2^-126), its values
x / scale rounded to e4m3. A case is one pass through one operator:

* "norm": residual + x, and its root-mean-square norm (of the sum before it is
  rounded to the residual's type), as e4m3 rows with scales, as float32 or
  float16, or both;
* "quant": rows, or silu(a) * b of two, as e4m3 rows with scales;
* "gemm": e4m3 rows times an e4m3 weight.

K and N need not be whole blocks (a shard's width, an odd vocabulary).
"""
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
F8 = torch.float8_e4m3fn
MOST8 = 448.0  # e4m3's largest value
LEAST = 2.0**-126  # the least scale
EPS = 1e-6


def listed():
    return [
        # one token of one user between two linears, f32 residual
        dict(name="norm_1", kind="norm", t=1, d=4096, res="f32", x="f32", y="", q=True, one_plus=False),
        # a decode batch; the normed rows also as they are (a layer whose other linears read f32), weights as w - 1
        dict(name="norm_31_both", kind="norm", t=31, d=2560, res="f32", x="f32", y="f32", q=True, one_plus=True),
        # a prompt of odd length, f16 all through
        dict(name="norm_4095", kind="norm", t=4095, d=5120, res="f16", x="f16", y="", q=True, one_plus=False),
        # one token's gate and up
        dict(name="silu_1", kind="quant", t=1, k=11008, x="f32", silu=True),
        # an attention output of a shard, whose width ends inside a block
        dict(name="quant_77", kind="quant", t=77, k=2752, x="f16", silu=False),
        # a prompt's gate and up
        dict(name="silu_4096", kind="quant", t=4096, k=11008, x="f16", silu=True),
        # the smallest linear of one token
        dict(name="gemm_1", kind="gemm", t=1, k=2560, n=2560, y="f32"),
        # gate and up of one token, side by side
        dict(name="gemm_1_wide", kind="gemm", t=1, k=4096, n=22016, y="f32"),
        # a decode batch on a shard, both sizes odd
        dict(name="gemm_31_odd", kind="gemm", t=31, k=2752, n=4099, y="f32"),
        # a short prompt
        dict(name="gemm_77", kind="gemm", t=77, k=5120, n=13824, y="f16"),
        # a prompt's down projection
        dict(name="gemm_512", kind="gemm", t=512, k=11008, n=4096, y="f16"),
        # a long prompt's gate and up
        dict(name="gemm_4096", kind="gemm", t=4096, k=4096, n=22016, y="f16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "quant", "gemm", "gemm", "gemm", "gemm"])
    t = rng.choice([1, rng.randint(2, 32), _log(rng, 33, 4096), _log(rng, 33, 4096)])
    if kind == "norm":
        d = rng.choice([2560, 4096, 5120, _log(rng, 128, 8192, 16)])
        res = rng.choice(["f32", "f16"])
        y, q = rng.choice([("", True), ("", True), ("f32", True), ("f16", True), ("f32", False), ("f16", False)])
        return dict(kind=kind, t=t, d=d, res=res, x=rng.choice([res, "f32", "f16"]), y=y, q=q, one_plus=rng.random() < 0.5)
    if kind == "quant":
        return dict(kind=kind, t=t, k=rng.choice([4096, 9728, 11008, _log(rng, 128, 11008, 16)]), x=rng.choice(["f32", "f16"]),
                    silu=rng.random() < 0.6)
    k = rng.choice([2560, 4096, 9728, _log(rng, 256, 13824, 16)])
    n = rng.choice([2560, 4096, 13824, 22016, _log(rng, 64, 22016)])
    while t * k * n > 4096 * 4096 * 22016:
        n //= 2
    return dict(kind=kind, t=t, k=k, n=n, y=rng.choice(["f32", "f16"]))


# ------------------------------------------------------------------ inputs
def _randn(seed, idx, *shape):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 4096 + idx)
    return torch.randn(*shape, device=DEV, generator=g)


def _dt(name):
    return {"f32": torch.float32, "f16": torch.float16}[name]


def _blocks(n):
    return -(-n // BLOCK)


def _channels(seed, idx, n):
    """A few channels are much larger than the others, as in a model's activations."""
    return 1.0 + 15.0 * (_randn(seed, idx, n) > 2.4)


def _rows8(t, k):
    """What a call writes quantised rows to."""
    return torch.empty(t, k, dtype=F8, device=DEV), torch.empty(_blocks(k), t, device=DEV)


def prepare(case, seed):
    c, st = case, dict(case=case)
    t = c["t"]
    if c["kind"] == "norm":
        d = c["d"]
        chan = _channels(seed, 1, d)
        st["residual"] = (4.0 * _randn(seed, 2, t, d) * chan).to(_dt(c["res"]))
        st["x"] = (_randn(seed, 3, t, d) * chan).to(_dt(c["x"]))
        st["weight"] = (0.0 if c["one_plus"] else 1.0) + 0.2 * _randn(seed, 4, d)
        st["residual_out"] = torch.empty_like(st["residual"])
        st["y"] = torch.empty(t, d, dtype=_dt(c["y"]), device=DEV) if c["y"] else None
        st["y8"], st["scale"] = _rows8(t, d) if c["q"] else (None, None)
    elif c["kind"] == "quant":
        k = c["k"]
        x = _randn(seed, 1, t, 2 * k if c["silu"] else k)
        st["x"] = (1.5 * x * _channels(seed, 2, x.shape[1])).to(_dt(c["x"]))
        st["y8"], st["scale"] = _rows8(t, k)
    else:
        k, n = c["k"], c["n"]
        st["x8"], st["x_scale"] = _quantise(_randn(seed, 1, t, k) * _channels(seed, 2, k))
        w = torch.nn.functional.pad(_randn(seed, 3, n, k) * (1.0 / math.sqrt(k)), (0, -k % BLOCK, 0, -n % BLOCK))
        w = w.view(_blocks(n), BLOCK, _blocks(k), BLOCK)
        scale = w.abs().amax((1, 3)) / MOST8
        st["w8"] = (w / scale[:, None, :, None]).to(F8).view(_blocks(n) * BLOCK, -1)[:n, :k].contiguous()
        st["w_scale"] = scale.contiguous()
        st["y"] = torch.empty(t, n, dtype=_dt(c["y"]), device=DEV)
    return st


# --------------------------------------------------------- the plain forms
def _quantise(y):
    """Rows of float32 as e4m3 [T, K] and scales [blocks, T]."""
    t, k = y.shape
    b = torch.nn.functional.pad(y, (0, -k % BLOCK)).view(t, -1, BLOCK)
    scale = (b.abs().amax(-1) / MOST8).clamp(min=LEAST)
    q = (b / scale[..., None]).clamp(-MOST8, MOST8).to(F8)
    return q.view(t, -1)[:, :k].contiguous(), scale.t().contiguous()


def _norm_plain(st, c):
    r = st["residual"].float() + st["x"].float()
    st["residual_out"].copy_(r)
    w = st["weight"] + 1.0 if c["one_plus"] else st["weight"]
    y = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * w
    if c["y"]:
        st["y"].copy_(y)
    if c["q"]:
        q, scale = _quantise(y)
        st["y8"].copy_(q)
        st["scale"].copy_(scale)
    return _norm_out(st)


def _norm_out(st):
    return {name: st[name] for name in ("residual_out", "y", "y8", "scale") if st[name] is not None}


def _quant_plain(st, c):
    x = st["x"].float()
    if c["silu"]:
        a, b = x[:, : c["k"]], x[:, c["k"] :]
        x = a / (1.0 + torch.exp(-a)) * b
    q, scale = _quantise(x)
    st["y8"].copy_(q)
    st["scale"].copy_(scale)
    return st["y8"], st["scale"]


def _gemm_plain(st, c):
    t, k, n = c["t"], c["k"], c["n"]
    kb, nb = (torch.arange(m, device=DEV) // BLOCK for m in (k, n))
    x = st["x8"].float() * st["x_scale"].t()[:, kb]
    w = st["w8"].float() * st["w_scale"][nb][:, kb]
    st["y"].copy_(torch.matmul(x, w.t()))
    return st["y"]


# ------------------------------------------------- the framework's kernels
_ctx = []


def _gpu():
    """The program's context of the framework (one for the process)."""
    if not _ctx:
        import shady_thinker_amd as sta

        _ctx.append(sta.GpuContext(0))
    return _ctx[0]


def _handle(st, name, make):
    """A handle that a program keeps beside its tensors."""
    if name not in st:
        st[name] = make()
    return st[name]


def _run_own(st, c):
    import shady_thinker_amd as sta

    gpu = _gpu()
    if c["kind"] == "norm":
        rows = _handle(st, "rows", lambda: sta.Fp8Rows.of(st["y8"], st["scale"])) if c["q"] else None
        sta.add_rmsnorm(gpu, st["residual"], st["weight"], st["x"], st["y"], rows, residual_out=st["residual_out"], eps=EPS,
                        one_plus=c["one_plus"])
        return _norm_out(st)
    if c["kind"] == "quant":
        rows, x, k = _handle(st, "rows", lambda: sta.Fp8Rows.of(st["y8"], st["scale"])), st["x"], c["k"]
        if c["silu"]:
            sta.fp8_quant(gpu, x[:, :k], rows, x[:, k:])
        else:
            sta.fp8_quant(gpu, x, rows)
        return st["y8"], st["scale"]
    rows = _handle(st, "rows", lambda: sta.Fp8Rows.of(st["x8"], st["x_scale"]))
    weight = _handle(st, "weight", lambda: sta.Fp8Weight.of(st["w8"], st["w_scale"]))
    sta.fp8_gemm(gpu, rows, weight, st["y"])
    return st["y"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    return {"norm": _norm_plain, "quant": _quant_plain, "gemm": _gemm_plain}[c["kind"]](state, c)


def work(case):
    c, t = case, case["t"]
    size = lambda name: {"": 0, "f16": 2, "f32": 4}[name]
    rows8 = lambda k: t * (k + 4 * _blocks(k))
    if c["kind"] == "norm":
        d = c["d"]
        return dict(bytes=t * d * (2 * size(c["res"]) + size(c["x"]) + size(c["y"])) + (rows8(d) if c["q"] else 0) + 4 * d, flops=6 * t * d)
    if c["kind"] == "quant":
        k = c["k"]
        return dict(bytes=t * k * size(c["x"]) * (2 if c["silu"] else 1) + rows8(k), flops=(8 if c["silu"] else 3) * t * k)
    k, n = c["k"], c["n"]
    return dict(bytes=rows8(k) + n * k + 4 * _blocks(n) * _blocks(k) + t * n * size(c["y"]), flops=2 * t * k * n)


# ------------------------------------------------------------ 64-bit values
def _rows64(y):
    """(what the 8 bits round, scale) of rows, block by block of the definition."""
    q, scale = torch.empty_like(y), []
    for k0 in range(0, y.shape[1], BLOCK):
        part = y[:, k0 : k0 + BLOCK]
        s = torch.maximum(part.abs().max(-1).values / MOST8, torch.tensor(LEAST, dtype=torch.float64, device=DEV))
        q[:, k0 : k0 + BLOCK] = part / s[:, None]
        scale.append(s)
    return q, torch.stack(scale)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "norm":
        r = st["residual"].double() + st["x"].double()
        gain = st["weight"].double() + (1.0 if c["one_plus"] else 0.0)
        y = r / torch.sqrt(r.pow(2).sum(-1, keepdim=True) / c["d"] + EPS) * gain
        got = dict(residual_out=r)
        if c["y"]:
            got["y"] = y
        if c["q"]:
            got["y8"], got["scale"] = _rows64(y)
        return got
    if c["kind"] == "quant":
        x = st["x"].double()
        return _rows64(torch.nn.functional.silu(x[:, : c["k"]]) * x[:, c["k"] :] if c["silu"] else x)
    y = torch.zeros(c["t"], c["n"], dtype=torch.float64, device=DEV)
    for b in range(_blocks(c["k"])):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        part = st["x8"][:, at].double() @ st["w8"][:, at].double().t()
        y += part * st["x_scale"][b].double()[:, None] * st["w_scale"][:, b].double().repeat_interleave(BLOCK)[: c["n"]]
    return y
