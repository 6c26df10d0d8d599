"""The operators between the quantized linears, as measurable cases.

A case is one pass through one operator, over a paged key-value cache or the
lm_head's logits:

* "store": norms of queries and keys for each head, their rotation, and the
  write of keys and values into the cache (f16, or int8 with a scale for each
  token and head; an int8 case reads the written tokens back, the values that
  the 8 bits stand for);
* "read": cached tokens read back, dequantised;
* "attn": attention of new rows over the cache: one token for each sequence,
  a few drafted ones, or prompts; causal, optionally with a sliding window, a
  tanh cap, a bias that depends on distance, an output gate;
* "logprobs": log probability and rank of given tokens, the entropy and the
  top alternatives of rows of logits.

The cache holds tiles of 16 tokens: keys [pages, heads, page/16, dim/8, 16, 8]
(eight dims of a token side by side), values [pages, heads, page/16, 2, dim, 8]
(eight tokens of a dim side by side: half h holds tokens 4h..4h+3 and
8+4h..8+4h+3 of the tile), scales [pages, heads, page].
"""
import math

import torch

own = False

DEV = "cuda:0"


def listed():
    return [
        # one token of one user: f32 projections, the step's smallest launch
        dict(name="store_1", kind="store", t=1, nh=32, nkv=8, hd=128, rot=128, page=16, x="f32", cache="f16",
             gated=False, one_plus=False, pairs=False),
        # a decode batch of the reference's gated width, partial rotation, int8 cache, written and read back
        dict(name="store_31_i8", kind="store", t=31, nh=16, nkv=4, hd=256, rot=64, page=32, x="f32", cache="i8",
             gated=True, one_plus=True, pairs=False),
        # a long prompt's projections (f16 from the prefill GEMM), odd length
        dict(name="store_2047", kind="store", t=2047, nh=32, nkv=8, hd=128, rot=128, page=64, x="f16", cache="f16",
             gated=True, one_plus=False, pairs=True),
        # a short shared prefix taken out of a cache
        dict(name="read_77", kind="read", t=77, nkv=8, hd=128, page=16, cache="f16", out="f16"),
        # a long document's cache moved out, dequantised
        dict(name="read_16384_i8", kind="read", t=16384, nkv=8, hd=128, page=64, cache="i8", out="f16"),
        # one user, a short chat
        dict(name="decode_1", kind="attn", b=1, q=1, kv=333, nh=32, nkv=8, hd=128, page=16, cache="f16", x="f32", cap=0.0,
             window=0, bias=False, gated=False),
        # one user, a long document, int8 cache
        dict(name="decode_1_long_i8", kind="attn", b=1, q=1, kv=65000, nh=32, nkv=8, hd=128, page=64, cache="i8", x="f32",
             cap=0.0, window=0, bias=False, gated=True),
        # batched serving, sequences of very different lengths, capped scores
        dict(name="decode_31", kind="attn", b=31, q=1, kv=8191, nh=32, nkv=8, hd=128, page=16, cache="f16", x="f32",
             cap=50.0, window=0, bias=False, gated=False),
        # drafted tokens of a few users checked together, wide heads, sliding window
        dict(name="verify_6x5", kind="attn", b=6, q=5, kv=4099, nh=16, nkv=4, hd=256, page=32, cache="f16", x="f32",
             cap=0.0, window=1024, bias=False, gated=True),
        # the largest prompt, from empty
        dict(name="prompt_4096", kind="attn", b=1, q=4096, kv=4096, nh=32, nkv=8, hd=128, page=64, cache="f16", x="f16",
             cap=0.0, window=0, bias=False, gated=False),
        # one user's next token: what the model thought of it, with alternatives
        dict(name="logprobs_1", kind="logprobs", m=1, vocab=151936, x="f32", top=20),
        # scoring a prompt
        dict(name="logprobs_512", kind="logprobs", m=512, vocab=151936, x="f32", top=5),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["store", "store", "read", "decode", "decode", "decode", "verify", "prompt", "prompt", "logprobs", "logprobs"])
    nh, nkv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 128), (16, 4, 256), (16, 2, 256), (24, 8, 128), (28, 4, 128),
                              (32, 4, 64), (8, 8, 64)])
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice(["f16", "f16", "i8"])
    if kind == "store":
        t = rng.choice([rng.randint(1, 32), _log(rng, 33, 2048)])
        return dict(kind=kind, t=t, nh=nh, nkv=nkv, hd=hd, rot=rng.choice([hd, hd, hd // 2, hd // 4]), page=page,
                    x=rng.choice(["f32", "f16"]), cache=cache, gated=rng.random() < 0.5, one_plus=rng.random() < 0.5,
                    pairs=rng.random() < 0.3)
    if kind == "read":
        return dict(kind=kind, t=_log(rng, 1, 16384), nkv=min(nkv, 8), hd=min(hd, 128), page=page, cache=cache,
                    out=rng.choice(["f16", "f32"]))
    if kind == "logprobs":
        return dict(kind=kind, m=_log(rng, 1, 512), vocab=_log(rng, 8192, 151936), x=rng.choice(["f32", "f32", "f16"]),
                    top=rng.choice([0, 1, 5, 20, 32]))
    opts = dict(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, rng.randint(16, 4096)]),
                bias=rng.random() < 0.25, gated=rng.random() < 0.5)
    if kind == "prompt":
        q = _log(rng, 9, 4096)
        b = rng.choice([1, 1, rng.randint(2, 4)]) if q <= 1024 else 1
        kv = min(q + rng.choice([0, _log(rng, 1, 8192)]), max(q, int(8.0e6 / (b * q)) + q // 2))
        return dict(kind="attn", b=b, q=q, kv=kv, nh=nh, nkv=nkv, hd=hd, page=page, cache=cache, x="f16", **opts)
    b = _log(rng, 1, 32)
    if kind == "verify":
        b = min(b, 8)
    q = rng.randint(2, 8) if kind == "verify" else 1
    kv = _log(rng, q, min(65000, 131072 // b))
    return dict(kind="attn", b=b, q=q, kv=kv, nh=nh, nkv=min(nkv, 8), hd=hd, page=page, cache=cache, x=rng.choice(["f32", "f32", "f16"]),
                **opts)


# ------------------------------------------------------------------ inputs
def _gen(seed, idx):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 4096 + idx)
    return g


def _randn(seed, idx, *shape):
    return torch.randn(*shape, device=DEV, generator=_gen(seed, idx))


def _dt(name):
    return {"f32": torch.float32, "f16": torch.float16}[name]


def _lens(c):
    """(rows, cached tokens with them) of each sequence: of one sequence the
    case's own, of several from those down to a tenth of them (a batch's
    users are at different places)."""
    b = c["b"]
    if b == 1:
        return [(c["q"], c["kv"])]
    got = []
    for i in range(b):
        q = max(1, c["q"] - (i % 3) * c["q"] // 4)
        got.append((q, max(q, round(c["kv"] * (1.0 - 0.9 * i / (b - 1))))))
    return got


def _empty_cache(seed, c, pages):
    """A cache as a running program has it: every slot holds some token."""
    nkv, hd, page = c["nkv"], c["hd"], c["page"]
    ks, vs = (pages, nkv, page // 16, hd // 8, 16, 8), (pages, nkv, page // 16, 2, hd, 8)
    chan = 1.0 + 3.0 * (torch.rand(hd, device=DEV, generator=_gen(seed, 10)) < 0.03)  # a few large key channels
    mean = 0.5 * _randn(seed, 11, nkv, hd)
    k = _randn(seed, 12, *ks) * chan.view(hd // 8, 1, 8)
    v = _randn(seed, 13, *vs) + mean.view(nkv, 1, 1, hd, 1)
    if c["cache"] == "f16":
        return dict(k=k.half(), v=v.half(), k_scale=None, v_scale=None)
    size = lambda i: 0.025 * (0.5 + torch.rand(pages, nkv, page, device=DEV, generator=_gen(seed, i)))
    whole = lambda t: (t * 36.0).round().clamp(-127, 127).to(torch.int8)
    return dict(k=whole(k), v=whole(v), k_scale=size(14), v_scale=size(15))


def prepare(case, seed):
    c = case
    st = dict(case=c)
    if c["kind"] == "logprobs":
        m, n = c["m"], c["vocab"]
        x = _randn(seed, 1, m, n) * 2.0
        near = torch.randint(0, n, (m, 16), device=DEV, generator=_gen(seed, 2))
        x.scatter_add_(1, near, 5.0 + 2.0 * _randn(seed, 3, m, 16))  # what the model holds likely
        some = torch.randint(0, n, (m,), device=DEV, generator=_gen(seed, 4))
        st["tokens"] = torch.where(torch.arange(m, device=DEV) % 4 == 3, some, near[:, 0]).to(torch.int32)
        st["logits"] = x.to(_dt(c["x"]))
        e = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device=DEV)
        st["out"] = dict(logprob=e(m), entropy=e(m), rank=e(m, dt=torch.int32), top_ids=e(m, c["top"], dt=torch.int32),
                         top_logprobs=e(m, c["top"]))
        return st
    nkv, hd, page = c["nkv"], c["hd"], c["page"]
    if c["kind"] in ("store", "read"):
        t = c["t"]
        pages = -(-t // page) + 3
        order = torch.randperm(pages, device=DEV, generator=_gen(seed, 1))
        at = torch.arange(t, device=DEV)
        slots = order[at // page] * page + at % page
        if t <= 32:  # a decode batch: every token in a page of another sequence
            slots = torch.randperm(pages * page, device=DEV, generator=_gen(seed, 2))[:t]
        st["slots"] = slots.to(torch.int32)
        st.update(_empty_cache(seed, c, pages))
        if c["kind"] == "read":
            st["k_out"], st["v_out"] = (torch.empty(t, nkv, hd, dtype=_dt(c["out"]), device=DEV) for _ in range(2))
            return st
        nh, rot = c["nh"], c["rot"]
        st["qw"] = nh * hd * (2 if c["gated"] else 1)
        chan = 1.0 + 7.0 * (torch.rand(st["qw"] + 2 * nkv * hd, device=DEV, generator=_gen(seed, 3)) < 0.01)
        st["qkv"] = (_randn(seed, 4, t, st["qw"] + 2 * nkv * hd) * chan).to(_dt(c["x"]))
        most = 8192
        st["positions"] = (at + 5 if t > 32 else torch.randint(0, most, (t,), device=DEV, generator=_gen(seed, 5))).to(torch.int32)
        angle = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(rot // 2, device=DEV, dtype=torch.float64) * 2 / rot)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        one = 0.0 if c["one_plus"] else 1.0
        st["q_weight"], st["k_weight"] = (one + 0.2 * _randn(seed, i, hd) for i in (6, 7))
        st["q_out"] = torch.empty(t, nh * hd, dtype=_dt(c["x"]), device=DEV)
        if c["cache"] == "i8":
            st["k_out"], st["v_out"] = (torch.empty(t, nkv, hd, dtype=torch.float16, device=DEV) for _ in range(2))
        return st
    lens = _lens(c)
    lens = [lens[i] for i in torch.randperm(c["b"], generator=torch.Generator().manual_seed(seed)).tolist()]
    need = [-(-kv // page) for _, kv in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, device=DEV, generator=_gen(seed, 1)).to(torch.int32)
    first = torch.tensor([sum(need[:i]) for i in range(c["b"])], device=DEV)
    j = torch.arange(max(need), device=DEV)
    mine = j[None, :] < torch.tensor(need, device=DEV)[:, None]
    st["table"] = torch.where(mine, order[(first[:, None] + j).clamp(max=pages - 1)], -1).contiguous()
    st["kv_len"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
    rows = sum(q for q, _ in lens)
    st["q_start"] = None
    if c["q"] > 1:
        st["q_start"] = torch.tensor([sum(q for q, _ in lens[:i]) for i in range(c["b"] + 1)], dtype=torch.int32, device=DEV)
    st.update(_empty_cache(seed, c, pages))
    nh = c["nh"]
    st["q"] = (1.5 * _randn(seed, 2, rows, nh * hd)).to(_dt(c["x"]))
    st["gate"] = _randn(seed, 3, rows, nh * hd).to(_dt(c["x"])) if c["gated"] else None
    st["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, nh + 1, device=DEV) / nh) if c["bias"] else None
    st["scale"] = 1.0 / math.sqrt(hd)
    st["out"] = torch.empty(rows, nh * hd, dtype=_dt(c["x"]), device=DEV)
    return st


# --------------------------------------------------------- the plain forms
def _tokens_k(k):
    """[..., heads, page/16, dim/8, 16, 8] -> [..., page, heads, dim]."""
    *b, h, t, d, _, _ = k.shape
    n = len(b)
    return k.permute(*range(n), n + 1, n + 3, n, n + 2, n + 4).reshape(*b, t * 16, h, d * 8)


def _tokens_v(v):
    """[..., heads, page/16, 2, dim, 8] -> [..., page, heads, dim]."""
    *b, h, t, _, d, _ = v.shape
    n = len(b)
    v = v.view(*b, h, t, 2, d, 2, 4)
    return v.permute(*range(n), n + 1, n + 4, n + 2, n + 5, n, n + 3).reshape(*b, t * 16, h, d)


def _slot(c, slots):
    """(page, tile of the page, token of the tile) of slots."""
    s = slots.long()
    return s // c["page"], s % c["page"] // 16, s % 16


def _read_plain(st, c, dtype):
    p, tile, tok = _slot(c, st["slots"])
    k = st["k"][p, :, tile, :, tok, :].float().flatten(2)
    v = st["v"].view(*st["v"].shape[:-1], 2, 4)[p, :, tile, tok // 4 % 2, :, tok // 8, tok % 4].float()
    if c["cache"] == "i8":
        at = st["slots"].long() % c["page"]
        k, v = k * st["k_scale"][p, :, at][..., None], v * st["v_scale"][p, :, at][..., None]
    return k.to(dtype), v.to(dtype)


def _rotate(y, c, cos, sin):
    a = c["rot"]
    r, rest = y[..., :a], y[..., a:]
    x0, x1 = (r[..., 0::2], r[..., 1::2]) if c["pairs"] else (r[..., : a // 2], r[..., a // 2 :])
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    r = torch.stack([y0, y1], -1).flatten(-2) if c["pairs"] else torch.cat([y0, y1], -1)
    return torch.cat([r, rest], -1)


def _store_plain(st, c):
    t, nh, nkv, hd = c["t"], c["nh"], c["nkv"], c["hd"]
    qkv = st["qkv"].float()
    q = qkv[:, : st["qw"]].view(t, nh, -1)[..., :hd]  # (gated: each head's query, then its gate)
    k, v = (qkv[:, st["qw"] + i * nkv * hd :][:, : nkv * hd].view(t, nkv, hd) for i in (0, 1))
    pos = st["positions"].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    norm = lambda x, w: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w + 1.0 if c["one_plus"] else w)
    q, k = (_rotate(norm(x, w), c, cos, sin) for x, w in ((q, st["q_weight"]), (k, st["k_weight"])))
    st["q_out"].copy_(q.flatten(1))
    p, tile, tok = _slot(c, st["slots"])
    at = st["slots"].long() % c["page"]
    if c["cache"] == "i8":
        for_scale = [x.abs().amax(-1) / 127.0 for x in (k, v)]
        st["k_scale"][p, :, at], st["v_scale"][p, :, at] = for_scale
        k, v = (torch.where(s[..., None] > 0, x / s[..., None], 0.0).round().clamp(-127, 127) for x, s in zip((k, v), for_scale))
    st["k"][p, :, tile, :, tok, :] = k.to(st["k"].dtype).view(t, nkv, hd // 8, 8)
    st["v"].view(*st["v"].shape[:-1], 2, 4)[p, :, tile, tok // 4 % 2, :, tok // 8, tok % 4] = v.to(st["v"].dtype)
    if c["cache"] == "f16":
        return dict(q=st["q_out"], k=st["k"], v=st["v"])
    k, v = _read_plain(st, c, torch.float16)
    return dict(q=st["q_out"], k=k, v=v)


def _attn_plain(st, c):
    nh, nkv, hd, b = c["nh"], c["nkv"], c["hd"], c["b"]
    table = st["table"].long()
    k, v = _tokens_k(st["k"][table]).float(), _tokens_v(st["v"][table]).float()  # [b, page index, page, heads, dim]
    if c["cache"] == "i8":
        k = k * st["k_scale"][table].transpose(2, 3)[..., None]
        v = v * st["v_scale"][table].transpose(2, 3)[..., None]
    k, v = (x.flatten(1, 2).permute(0, 2, 1, 3).contiguous() for x in (k, v))  # [b, heads, keys, dim]
    n = k.shape[2]
    kv = st["kv_len"].long()
    start = torch.arange(b + 1, device=DEV) if st["q_start"] is None else st["q_start"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(c["q"], device=DEV)
    row = (start[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)  # [b, q]: a sequence's rows (past its last: any)
    pos = (kv - count)[:, None] + i
    q = st["q"][row].float().view(b, c["q"], nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, hd)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st["scale"]).view(b, nkv, nh // nkv, c["q"], n)
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    j = torch.arange(n, device=DEV)
    away = j - pos[:, :, None]  # [b, q, keys]
    if st["slopes"] is not None:
        s = s + st["slopes"].view(nkv, -1, 1, 1) * away[:, None, None].float()
    seen = (away <= 0) & (j < kv[:, None, None])
    if c["window"]:
        seen &= away > -c["window"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    o = torch.matmul(s.view(b, nkv, -1, n), v).view(b, nkv, nh // nkv, c["q"], hd)
    o = o / s.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, c["q"], nh * hd)
    r = torch.arange(st["q"].shape[0], device=DEV)
    of = torch.searchsorted(start, r, right=True) - 1
    o = o[of, r - start[of]]
    if st["gate"] is not None:
        o = o / (1.0 + torch.exp(-st["gate"].float()))
    st["out"].copy_(o)
    return st["out"]


def _logprobs_plain(st, c):
    x, t = st["logits"].float(), st["tokens"].long()[:, None]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    s = e.sum(-1)
    log_s = s.log()
    j = torch.arange(c["vocab"], device=DEV)
    xt = x.gather(1, t)
    out = st["out"]
    out["logprob"].copy_(d.gather(1, t)[:, 0] - log_s)
    out["entropy"].copy_(log_s - (e * d).sum(-1) / s)
    out["rank"].copy_(((x > xt) | ((x == xt) & (j < t))).sum(-1))
    if c["top"]:
        # by value, equal ones by index: the bits of x in its order, then the index from above
        bits = x.contiguous().view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - j)
        ids = key.topk(c["top"], dim=-1).indices
        out["top_ids"].copy_(ids)
        out["top_logprobs"].copy_(d.gather(1, ids) - log_s[:, None])
    return out


# ------------------------------------------------- the framework's kernels
_ctx = []


def _gpu():
    """The program's context of the framework (one for the process)."""
    if not _ctx:
        import shady_thinker_amd as sta

        _ctx.append(sta.GpuContext(0))
    return _ctx[0]


def _cache(st, c):
    """The state's cache as the framework's handle of it."""
    import shady_thinker_amd as sta

    if "cache" not in st:
        st["cache"] = sta.KvCache.of(st["k"], st["v"], c["page"], st["k_scale"], st["v_scale"])
    return st["cache"]


def _run_own(st, c):
    import shady_thinker_amd as sta

    gpu = _gpu()
    if c["kind"] == "logprobs":
        o = st["out"]
        sta.token_logprobs(gpu, st["logits"], st["tokens"], o["logprob"], o["entropy"], o["rank"], o["top_ids"], o["top_logprobs"])
        return o
    cache = _cache(st, c)
    if c["kind"] == "read":
        sta.kv_read(gpu, cache, st["slots"], st["k_out"], st["v_out"])
        return st["k_out"], st["v_out"]
    if c["kind"] == "store":
        qkv, w, kw = st["qkv"], st["qw"], c["nkv"] * c["hd"]
        sta.qk_norm_rope_store(gpu, cache, qkv[:, :w], qkv[:, w : w + kw], qkv[:, w + kw :], st["q_out"], st["slots"], st["positions"],
                               st["cos"], st["sin"], st["q_weight"], st["k_weight"], eps=1e-6, one_plus=c["one_plus"], pairs=c["pairs"],
                               gated=c["gated"])
        if c["cache"] == "f16":
            return dict(q=st["q_out"], k=st["k"], v=st["v"])
        sta.kv_read(gpu, cache, st["slots"], st["k_out"], st["v_out"])
        return dict(q=st["q_out"], k=st["k_out"], v=st["v_out"])
    sta.paged_attention(gpu, cache, st["q"], st["out"], st["table"], st["kv_len"], st["q_start"], scale=st["scale"], cap=c["cap"],
                        window=c["window"], slopes=st["slopes"], gate=st["gate"])
    return st["out"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    if c["kind"] == "logprobs":
        return _logprobs_plain(state, c)
    if c["kind"] == "read":
        k, v = _read_plain(state, c, _dt(c["out"]))
        state["k_out"].copy_(k)
        state["v_out"].copy_(v)
        return state["k_out"], state["v_out"]
    return _store_plain(state, c) if c["kind"] == "store" else _attn_plain(state, c)


def work(case):
    c = case
    if c["kind"] == "logprobs":
        size = 2 if c["x"] == "f16" else 4
        return dict(bytes=c["m"] * (c["vocab"] * size + 16 + 8 * c["top"]), flops=6 * c["m"] * c["vocab"])
    nkv, hd = c["nkv"], c["hd"]
    token = 2 * nkv * (hd * 2 if c["cache"] == "f16" else hd + 4)  # a cached token's bytes
    if c["kind"] == "read":
        return dict(bytes=c["t"] * (token + 4 + 2 * nkv * hd * (2 if c["out"] == "f16" else 4)), flops=2 * c["t"] * nkv * hd)
    size = 2 if c["x"] == "f16" else 4
    if c["kind"] == "store":
        n = c["nh"] * hd
        back = token + 4 * nkv * hd if c["cache"] == "i8" else 0
        by = c["t"] * ((2 * n + 2 * nkv * hd) * size + token + 8 + 4 * c["rot"] + back)
        return dict(bytes=by, flops=8 * c["t"] * (n + 2 * nkv * hd))
    rows = pairs = read = 0
    for q, kv in _lens(c):
        w = c["window"] or kv
        rows += q
        read += min(kv, w + q - 1)
        full = max(0, min(q, kv - w + 1)) if w < kv else 0  # rows that see a whole window
        left = q - full  # the first ones, which see all before them
        pairs += full * w + left * (kv - q + 1) + left * (left - 1) // 2
    by = read * token + rows * c["nh"] * hd * size * (3 if c["gated"] else 2) + 4 * (read // c["page"] + 2 * c["b"])
    return dict(bytes=by, flops=4 * pairs * c["nh"] * hd)


# ------------------------------------------------------------ 64-bit values
def _place(c, slots):
    """Flat index of (token, head, dim) in keys and values, from the layout's definition."""
    nkv, hd, page = c["nkv"], c["hd"], c["page"]
    s = slots.long()[:, None, None]
    h = torch.arange(nkv, device=DEV)[None, :, None]
    d = torch.arange(hd, device=DEV)[None, None, :]
    tile = ((s // page) * nkv + h) * (page // 16) + s % page // 16
    t = s % 16
    return (tile * (hd // 8) + d // 8) * 128 + t * 8 + d % 8, (tile * 2 + t // 4 % 2) * hd * 8 + d * 8 + t // 8 * 4 + t % 4


def _scales(st, c, slots, name):
    s = slots.long()[:, None]
    h = torch.arange(c["nkv"], device=DEV)[None]
    return st[name].view(-1)[((s // c["page"]) * c["nkv"] + h) * c["page"] + s % c["page"]].double()[..., None]


def _read64(st, c, slots):
    ik, iv = _place(c, slots)
    k, v = st["k"].view(-1)[ik].double(), st["v"].view(-1)[iv].double()
    if c["cache"] == "i8":
        k, v = k * _scales(st, c, slots, "k_scale"), v * _scales(st, c, slots, "v_scale")
    return k, v


def _store64(st, c):
    t, nh, nkv, hd, rot = c["t"], c["nh"], c["nkv"], c["hd"], c["rot"]
    x = st["qkv"].double()
    w, kw = st["qw"], nkv * hd
    step = 2 * hd if c["gated"] else hd
    heads = {"q": torch.stack([x[:, i * step : i * step + hd] for i in range(nh)], 1), "k": x[:, w : w + kw].reshape(t, nkv, hd),
             "v": x[:, w + kw :].reshape(t, nkv, hd)}
    pos = st["positions"].long()
    co, si = st["cos"].double()[pos][:, None], st["sin"].double()[pos][:, None]
    for name in ("q", "k"):
        y = heads[name]
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + 1e-6) * ((1.0 if c["one_plus"] else 0.0) + st[name + "_weight"].double())
        z = y.clone()
        lo = torch.arange(rot // 2, device=DEV) * 2 if c["pairs"] else torch.arange(rot // 2, device=DEV)
        hi = lo + (1 if c["pairs"] else rot // 2)
        z[..., lo] = y[..., lo] * co - y[..., hi] * si
        z[..., hi] = y[..., hi] * co + y[..., lo] * si
        heads[name] = z
    q = heads["q"].reshape(t, nh * hd)
    if c["cache"] == "i8":
        held = []
        for y in (heads["k"], heads["v"]):
            s = y.abs().amax(-1, keepdim=True) / 127.0
            held.append(torch.round(y / s) * s)
        return dict(q=q, k=held[0], v=held[1])
    ik, iv = _place(c, st["slots"])
    k, v = st["k"].double(), st["v"].double()
    k.view(-1)[ik], v.view(-1)[iv] = heads["k"], heads["v"]
    return dict(q=q, k=k, v=v)


def _attn64(st, c):
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    out = torch.zeros(st["q"].shape[0], nh, hd, dtype=torch.float64, device=DEV)
    starts = list(range(c["b"] + 1)) if st["q_start"] is None else st["q_start"].tolist()
    for b, n in enumerate(st["kv_len"].tolist()):
        r0, r1 = starts[b], starts[b + 1]
        j = torch.arange(n, device=DEV)
        k, v = _read64(st, c, st["table"][b].long()[j // page] * page + j % page)
        p = torch.arange(n - (r1 - r0), n, device=DEV)[:, None]
        seen = j[None] <= p
        if c["window"]:
            seen &= j[None] > p - c["window"]
        for h in range(nh):
            q = st["q"][r0:r1, h * hd : (h + 1) * hd].double()
            s = q @ k[:, h * nkv // nh].t() * st["scale"]
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if st["slopes"] is not None:
                s = s + st["slopes"][h].double() * (j[None] - p)
            out[r0:r1, h] = torch.softmax(torch.where(seen, s, -math.inf), -1) @ v[:, h * nkv // nh]
    out = out.flatten(1)
    return out if st["gate"] is None else out * torch.sigmoid(st["gate"].double())


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "store":
        return _store64(st, c)
    if c["kind"] == "read":
        return _read64(st, c, st["slots"])
    if c["kind"] == "attn":
        return _attn64(st, c)
    lp = torch.log_softmax(st["logits"].double(), -1)
    t = st["tokens"].long()
    rows = torch.arange(c["m"], device=DEV)
    plogp = torch.where(lp > -math.inf, lp.exp() * lp, 0.0)
    ids = torch.sort(st["logits"].float(), dim=-1, descending=True, stable=True).indices[:, : c["top"]]
    return dict(logprob=lp[rows, t], entropy=-plogp.sum(-1), rank=None, top_ids=None, top_logprobs=lp.gather(1, ids))
