"""GPU parity of the cache and attention entry points (st_qk_norm_rope_store,
st_kv_read, st_paged_attention) through the Python helpers, against 64-bit
plain forms on the CPU (tests/attn_util.py).

Tolerances (relative 2-norm), from the arithmetic:
* f32 results of the store: a norm and a rotation in f32, a handful of
  roundings of 2^-24: 1e-6. f16: one rounding (2^-11, 2.1e-4 rms): 5e-4.
* int8: half a step of the head's scale, and 1e-3 of a step for f32.
* f32 attention: q and weights in 22 bits, scores up to about 2^5 in f32
  (2^-24 2^5 = 2e-6 of a weight): 1e-5. f16: output and weights rounded to
  f16 (2.1e-4 rms each): 1e-3.
"""
import math

import pytest
import torch

import shady_thinker_amd as sta
from shady_thinker_amd._lib import launches
from attn_util import attention, indices, norm_rope, rel, shapes

pytestmark = pytest.mark.gpu

F32, F16, I8 = torch.float32, torch.float16, torch.int8


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def tables(n, rot, theta=10000.0):
    a = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    return a.cos().float(), a.sin().float()


def cache_of(gpu, pages, heads, page, hd, dtype, fill=None):
    c = sta.KvCache(gpu, pages, page, heads, hd, dtype)
    for t in (c.k, c.v):
        t.fill_(77 if fill is None else fill)
    if dtype is I8:
        c.k_scale.fill_(3.0)
        c.v_scale.fill_(3.0)
    return c


# ------------------------------------------------------------------- store
STORE = [
    # hd, nh, nkv, T, page, x, q_out, cache, rot, pairs, gated, plus, norm, slots
    (128, 4, 2, 1, 16, F32, F32, F16, 128, False, False, False, True, "scatter"),
    (64, 3, 1, 5, 32, F32, F16, F16, 32, True, True, True, True, "scatter"),
    (256, 2, 2, 33, 64, F16, F16, F16, 64, False, True, False, True, "run0"),
    (128, 7, 1, 50, 16, F16, F32, F16, 96, False, False, True, True, "run5"),
    (128, 4, 4, 40, 128, F32, F32, I8, 128, False, True, False, True, "run5"),
    (64, 4, 2, 17, 16, F16, F16, I8, 64, True, False, False, True, "scatter"),
    (256, 2, 1, 3, 256, F32, F32, I8, 256, False, False, True, False, "scatter"),
    (128, 2, 2, 19, 32, F32, F32, F16, 0, False, False, False, False, "run0"),
    (128, 2, 2, 64, 32, F32, F32, F16, 128, False, False, False, True, "holes"),
    (128, 0, 2, 16, 32, F16, None, F16, 128, False, False, False, True, "run0"),
]


@pytest.mark.parametrize("hd,nh,nkv,T,page,xd,qd,cd,rot,pairs,gated,plus,norm,where", STORE)
def test_store(gpu, hd, nh, nkv, T, page, xd, qd, cd, rot, pairs, gated, plus, norm, where):
    g = rng(hd + T)
    wide = nh * hd * (2 if gated else 1)
    extra = 24  # the rows are parts of wider ones
    row = torch.randn(T, wide + 2 * nkv * hd + extra, generator=g).to(xd)
    row[:, wide:wide + 1] *= 30.0
    q, k, v = row[:, :wide], row[:, wide:wide + nkv * hd], row[:, wide + nkv * hd:wide + 2 * nkv * hd]
    pages = T // page + 4
    if where == "scatter":
        slots = torch.randperm(pages * page, generator=g)[:T]
    else:
        slots = torch.arange(T) + (5 if where == "run5" else 0) + page
    bad = torch.zeros(T, dtype=torch.bool)
    n_pos = 300
    pos = torch.randint(0, n_pos, (T,), generator=g)
    if where == "holes":  # padding, slots and positions out of range
        slots[3], slots[20], slots[21] = -1, pages * page, 2**31 - 1
        pos[40], pos[41] = -1, n_pos
        bad[[3, 20, 21, 40, 41]] = True
    cos, sin = tables(n_pos, rot) if rot else (None, None)
    qw, kw = (torch.randn(hd, generator=g) * 0.3 + (0.0 if plus else 1.0) for _ in range(2)) if norm else (None, None)
    c = cache_of(gpu, pages, nkv, page, hd, cd)
    D = lambda t, dt=None: None if t is None else t.to(gpu.device, dt or t.dtype)
    rd = D(row)
    q_out = torch.full((T, nh * hd), 5.0, dtype=qd, device=gpu.device) if nh else None
    sta.qk_norm_rope_store(gpu, c, rd[:, :wide] if nh else None, rd[:, wide:wide + nkv * hd], rd[:, wide + nkv * hd:wide + 2 * nkv * hd],
                           q_out, D(slots, torch.int32), D(pos, torch.int32) if rot else None, D(cos), D(sin), D(qw), D(kw), eps=1e-5,
                           one_plus=plus, pairs=pairs, gated=gated)
    safe = pos.clamp(0, n_pos - 1)
    heads = lambda t, n: t.double().view(T, n, -1)[..., :hd]
    kx = norm_rope(heads(k, nkv), kw, 1e-5, float(plus), cos, sin, safe, pairs)
    vx = heads(v, nkv)
    if nh:
        qx = norm_rope(heads(q, nh), qw, 1e-5, float(plus), cos, sin, safe, pairs).flatten(1)
        got = q_out.cpu()
        misplaced = (pos != safe) if rot else torch.zeros(T, dtype=torch.bool)
        assert got[misplaced].isnan().all()
        assert rel(got[~misplaced], qx[~misplaced]) < (1e-6 if qd is F32 else 5e-4)
    keep = ~bad
    ki, vi, si = indices(slots[keep], nkv, page, hd)
    kc, vc = c.k.cpu().flatten(), c.v.cpu().flatten()
    for raw, at, want, scales in ((kc, ki, kx[keep], c.k_scale), (vc, vi, vx[keep], c.v_scale)):
        got = raw[at].double()
        if cd is I8:
            s = scales.cpu().flatten()[si].double()[..., None]
            assert rel(s[..., 0], want.abs().amax(-1) / 127) < 1e-6
            assert ((got * s - want).abs() <= s * 0.501).all()
            assert got.abs().max() <= 127
        else:
            assert rel(got, want) < 5e-4
        untouched = torch.ones(raw.numel(), dtype=torch.bool)
        untouched[at.flatten()] = False
        assert (raw[untouched] == 77).all()
    if cd is I8:
        for scales in (c.k_scale, c.v_scale):
            rest = torch.ones(scales.numel(), dtype=torch.bool)
            rest[si.flatten()] = False
            assert (scales.cpu().flatten()[rest] == 3.0).all()


def test_store_int8_edge_heads(gpu):
    """A zero head, one with a NaN, one with an infinity, equal magnitudes."""
    T, hd = 4, 64
    x = torch.randn(T, hd, generator=rng(1))
    x[0] = 0.0
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    x[3] = torch.where(x[3] > 0, 2.0, -2.0)
    c = cache_of(gpu, 1, 1, 16, hd, I8)
    slots = torch.arange(T, dtype=torch.int32, device=gpu.device)
    xd = x.to(gpu.device)
    sta.qk_norm_rope_store(gpu, c, None, xd, xd, None, slots)
    ko, vo = (torch.empty(T, 1, hd, device=gpu.device) for _ in range(2))
    sta.kv_read(gpu, c, slots, ko, vo)
    for o in (ko.cpu()[:, 0], vo.cpu()[:, 0]):
        assert (o[0] == 0).all()
        assert o[1].isnan().all()
        assert not o[2].isfinite().any()
        assert rel(o[3], x[3]) < 1e-6


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("hd,nkv,T,page,cd,od,where", [
    (128, 2, 1, 16, F16, F16, "scatter"), (64, 3, 16, 16, F16, F32, "run0"), (256, 1, 45, 64, F16, F16, "run5"),
    (128, 2, 40, 32, I8, F32, "run0"), (64, 2, 37, 128, I8, F16, "run5"), (256, 2, 21, 16, I8, F32, "holes"),
    (128, 1, 33, 16, F16, F32, "holes"),
])
def test_read(gpu, hd, nkv, T, page, cd, od, where):
    g = rng(T + hd)
    pages = T // page + 3
    c = sta.KvCache(gpu, pages, page, nkv, hd, cd)
    mk = lambda t: t.copy_((torch.randint(-127, 128, t.shape, generator=g) if cd is I8 else torch.randn(t.shape, generator=g)).to(cd))
    mk(c.k), mk(c.v)
    if cd is I8:
        for s in (c.k_scale, c.v_scale):
            s.copy_(torch.rand(s.shape, generator=g) + 0.1)
    slots = torch.randperm(pages * page, generator=g)[:T] if where == "scatter" else torch.arange(T) + page + (5 if where == "run5" else 0)
    bad = torch.zeros(T, dtype=torch.bool)
    if where == "holes":
        slots[0], slots[T - 1], slots[7] = -1, pages * page, -2**31
        bad[[0, 7, T - 1]] = True
    ko, vo = (torch.full((T, nkv, hd), 9.0, dtype=od, device=gpu.device) for _ in range(2))
    sta.kv_read(gpu, c, slots.to(gpu.device, torch.int32), ko, vo)
    ki, vi, si = indices(slots.clamp(0, pages * page - 1), nkv, page, hd)
    for got, raw, at, s in ((ko, c.k, ki, c.k_scale), (vo, c.v, vi, c.v_scale)):
        want = raw.cpu().flatten()[at].float()
        if cd is I8:
            want = want * s.cpu().flatten()[si][..., None]
        want[bad] = 0.0
        assert torch.equal(got.cpu(), want.to(od))


# --------------------------------------------------------------- attention
class Batch:
    """A cache with random tokens of sequences of given (rows, kv_len), pages
    in random order, everything no row may see set to NaN (f16) or to NaN
    scales (int8). wide: the table's rows hold that many tokens at least
    (many rows of f16 queries go to the prompt kernel where what the table
    holds could make a large call)."""

    def __init__(self, gpu, lens, nh, nkv, hd, page, cd, qd, seed=0, gaps=0, q_size=1.5, wide=0):
        g = rng(seed + hd + page)
        self.gpu, self.nh, self.nkv, self.hd = gpu, nh, nkv, hd
        need = [-(-kv // page) for _, kv in lens]
        B, pages = len(lens), sum(need) + 3
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((B, max(max(need) + 1, 2, wide // page)), -1)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        slots = [self.table[b][torch.arange(kv) // page] * page + torch.arange(kv) % page for b, (_, kv) in enumerate(lens)]
        every = torch.cat(slots)
        ks, vs, ss = shapes(pages, nkv, page, hd)
        ki, vi, si = indices(every, nkv, page, hd)
        n = every.numel()
        kt, vt = torch.randn(n, nkv, hd, generator=g), torch.randn(n, nkv, hd, generator=g) + 0.5
        if cd is F16:
            k, v = (torch.full((math.prod(s),), math.nan, dtype=F16) for s in (ks, vs))
            k[ki], v[vi] = kt.half(), vt.half()
            kt, vt = k[ki].double(), v[vi].double()
            self.cache = sta.KvCache.of(k.view(ks).to(gpu.device), v.view(vs).to(gpu.device), page)
        else:
            k, v = (torch.full((math.prod(s),), 99, dtype=I8) for s in (ks, vs))
            s1, s2 = (torch.full((math.prod(ss),), math.nan) for _ in range(2))
            k[ki], v[vi] = ((t * 30).round().clamp(-127, 127).to(I8) for t in (kt, vt))
            s1[si], s2[si] = (torch.rand(n, nkv, generator=g) * 0.05 + 1e-3 for _ in range(2))
            s2[si[: n // 3]] *= 1e-4  # (value scales that differ by much)
            kt, vt = k[ki].double() * s1[si].double()[..., None], v[vi].double() * s2[si].double()[..., None]
            self.cache = sta.KvCache.of(k.view(ks).to(gpu.device), v.view(vs).to(gpu.device), page, s1.view(ss).to(gpu.device),
                                        s2.view(ss).to(gpu.device))
        cut = [sum(kv for _, kv in lens[:b]) for b in range(B + 1)]
        self.k_of, self.v_of = (lambda b, t=t: t[cut[b]:cut[b + 1]] for t in (kt, vt))
        self.q_start, self.spans, r = [], [], 0
        for rows, kv in lens:
            self.q_start.append(r)
            self.spans.append((r, rows, kv))
            r += rows
        self.q_start.append(r)
        T = r + gaps  # rows of no sequence at the end
        self.q = (q_size * torch.randn(T, nh, hd, generator=g)).to(qd)
        self.T, self.one = T, all(rows == 1 for rows, _ in lens) and not gaps
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32)

    def run(self, od=None, gate=None, slopes=None, **kw):
        dev = self.gpu.device
        out = torch.full((self.T, self.nh * self.hd), 7.0, dtype=od or self.q.dtype, device=dev)
        sta.paged_attention(self.gpu, self.cache, self.q.flatten(1).to(dev), out, self.table.to(dev, torch.int32), self.kv_len.to(dev),
                            None if self.one else torch.tensor(self.q_start, dtype=torch.int32, device=dev),
                            gate=None if gate is None else gate.flatten(1).to(dev), slopes=None if slopes is None else slopes.to(dev), **kw)
        return out.cpu().view(self.T, self.nh, self.hd)

    def want(self, scale=None, **kw):
        return attention(self.q, self.k_of, self.v_of, self.spans, scale or 1 / math.sqrt(self.hd), **kw)

    def check(self, got, want):
        outside = want.isnan()
        assert (got[outside] == 7.0).all()
        assert got[~outside].isfinite().all()
        e = rel(got[~outside], want[~outside])
        tol = 1e-5 if got.dtype is F32 else 1e-3
        print(f"rel-L2 {e:.3g}")
        assert e < tol


ATT = [
    # lens, nh, nkv, hd, page, cache, q
    ([(1, 1)], 4, 4, 128, 16, F16, F32),
    ([(1, 0)], 4, 2, 64, 16, F16, F32),
    ([(1, 33)], 8, 2, 128, 16, F16, F32),
    ([(1, 1000)], 8, 1, 256, 32, F16, F32),
    ([(1, 5000)], 14, 2, 64, 64, F16, F32),
    ([(1, 5001)], 16, 2, 128, 256, I8, F32),
    ([(1, 16), (1, 700), (1, 0), (1, 31), (1, 2049)], 8, 2, 128, 16, F16, F32),
    ([(1, 300), (1, 17), (1, 64)], 6, 2, 64, 32, I8, F16),
    ([(1, 64)] * 70, 4, 1, 128, 16, F16, F16),
    ([(3, 40), (0, 5), (1, 900), (8, 8), (2, 1)], 8, 2, 128, 16, F16, F32),
    ([(5, 77), (4, 300)], 4, 4, 256, 64, F16, F32),
    ([(5, 77), (4, 300)], 4, 4, 256, 64, I8, F16),
    ([(2, 130)], 64, 1, 64, 16, F16, F16),
    ([(17, 17), (64, 200)], 4, 2, 128, 16, F16, F16),
    ([(100, 100)], 8, 2, 64, 32, F16, F16),
    ([(257, 300)], 2, 2, 128, 16, F16, F16),
    ([(130, 131), (3, 3), (70, 1000)], 6, 2, 128, 64, I8, F16),
    ([(90, 91), (129, 129)], 4, 1, 256, 32, F16, F16),
    ([(40, 100)], 4, 2, 128, 16, F16, F32),
]


@pytest.mark.parametrize("lens,nh,nkv,hd,page,cd,qd", ATT)
def test_attention(gpu, lens, nh, nkv, hd, page, cd, qd):
    b = Batch(gpu, lens, nh, nkv, hd, page, cd, qd)
    got = b.run()
    b.check(got, b.want())
    for r0, rows, kv in b.spans:
        if kv == 0:
            assert (got[r0:r0 + rows] == 0).all()


def as_prompt(b):
    """Runs the batch; it took the kernel of prompts."""
    launches()
    got = b.run()
    assert launches() == ["prompt_kernel", "prompt_join_kernel"]
    return got


@pytest.mark.parametrize("lens,nh,nkv,hd,page,cd", [
    ([(16, 16)], 2, 1, 128, 16, F16),
    ([(64, 200)], 4, 2, 128, 16, F16),
    ([(100, 100)], 8, 2, 64, 32, I8),
    ([(257, 600)], 2, 2, 128, 16, F16),
    ([(77, 2222)], 6, 2, 128, 64, I8),
    ([(77, 4097)], 8, 2, 128, 64, F16),
    ([(33, 3000)], 8, 1, 256, 16, F16),
    ([(40, 1531)], 4, 1, 64, 16, F16),
    ([(130, 131), (3, 3), (0, 70), (70, 1000)], 6, 2, 128, 64, F16),
    ([(90, 91), (129, 1300)], 4, 1, 256, 32, I8),
])
def test_attention_prompts(gpu, lens, nh, nkv, hd, page, cd):
    b = Batch(gpu, lens, nh, nkv, hd, page, cd, F16, wide=1 << 15, gaps=1)
    b.check(as_prompt(b), b.want())


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("rows,hd,cd,qd,wide", [
    (6, 128, F16, F32, 0), (6, 256, F16, F16, 0), (6, 64, I8, F32, 0), (20, 128, F16, F16, 0),
    (100, 128, F16, F16, 1 << 15), (70, 64, F16, F16, 1 << 15), (70, 256, F16, F16, 1 << 15), (100, 128, I8, F16, 1 << 15)])
def test_attention_values_not_finite(gpu, value, window, rows, hd, cd, qd, wide):
    """A value, key or scale that is not finite is in the rows that see its
    token (a value: in its dim), and nowhere else."""
    kv, nkv, nh, page = rows + 50, 2, 6, 16
    for what in ("value", "key"):
        b = Batch(gpu, [(rows, kv)], nh, nkv, hd, page, cd, qd, wide=wide)
        p, d = kv - rows + rows // 2, 21
        slot = (b.table[0, p // page] * page + p % page).reshape(1)
        ki, vi, si = indices(slot, nkv, page, hd)
        if cd is F16:
            t, at = (b.cache.v, vi[0, 1, d]) if what == "value" else (b.cache.k, ki[0, 1, d])
        else:
            t, at = (b.cache.v_scale if what == "value" else b.cache.k_scale), si[0, 1]
        t.view(-1)[at] = value
        got, want = b.run(window=window), b.want(window=window)
        at_row = torch.arange(rows) + kv - rows
        see = (at_row >= p) & ((at_row < p + window) if window else True)
        assert see.any() and not see.all()
        bad = torch.zeros_like(want, dtype=torch.bool)
        bad[see, nh // 2:, d if cd is F16 and what == "value" else slice(None)] = True
        if what == "value" or math.isnan(value):  # (an infinite key: its score may be the lowest, too)
            assert not got[bad].isfinite().any()
        assert got[~bad].isfinite().all()
        assert rel(got[~bad], want[~bad]) < (1e-5 if qd is F32 else 1e-3)


def test_attention_values_not_finite_long_prompt(gpu):
    """The same in a call whose row blocks fill the GPU, so without chunks: bit
    for bit the call without, but for what sees the value."""
    rows, nkv, nh, hd, page = 4200, 4, 16, 64, 64
    b = Batch(gpu, [(rows, rows)], nh, nkv, hd, page, F16, F16)
    want = as_prompt(b)
    places = [(5, 0, 3), (2100, 2, 63), (4199, 3, 17)]  # token, key head, dim
    bad = torch.zeros_like(want, dtype=torch.bool)
    for p, h, d in places:
        slot = (b.table[0, p // page] * page + p % page).reshape(1)
        b.cache.v.view(-1)[indices(slot, nkv, page, hd)[1][0, h, d]] = -math.inf
        bad[p:, h * nh // nkv:(h + 1) * nh // nkv, d] = True
    got = as_prompt(b)
    assert not got[bad].isfinite().any()
    assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("opts", [dict(cap=5.0), dict(window=1), dict(window=40), dict(window=333, cap=20.0), dict(slopes=True),
                                  dict(slopes=True, window=64, cap=8.0), dict(gate=True), dict(scale=0.05, gate=True)])
@pytest.mark.parametrize("lens,nh,nkv,hd,page,cd,qd", [
    ([(1, 700), (1, 12)], 8, 2, 128, 16, F16, F32),
    ([(4, 500), (2, 40)], 4, 2, 64, 32, I8, F32),
    ([(3, 300)], 4, 1, 256, 16, F16, F16),
    ([(150, 400), (20, 20)], 4, 2, 128, 16, F16, F16),
    ([(140, 500)], 6, 2, 64, 64, I8, F16),
    ([(70, 300)], 4, 2, 256, 16, F16, F16),
])
def test_attention_scores(gpu, lens, nh, nkv, hd, page, cd, qd, opts):
    b = Batch(gpu, lens, nh, nkv, hd, page, cd, qd, seed=5, gaps=2)
    o = dict(opts)
    if o.pop("slopes", False):
        o["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / nh) for i in range(nh)])
    if o.pop("gate", False):
        o["gate"] = torch.randn(b.T, nh, hd, generator=rng(3)).to(qd)
    b.check(b.run(**o), b.want(**o))


def test_attention_gated_rows(gpu):
    """The gate beside each head's query in a wider row."""
    b = Batch(gpu, [(1, 90), (1, 5)], 4, 2, 128, 16, F16, F32)
    row = torch.randn(2, 4 * 256 + 40, generator=rng(9)).to(gpu.device)
    out = torch.empty(2, 512, device=gpu.device)
    dev = gpu.device
    sta.paged_attention(gpu, b.cache, b.q.flatten(1).to(dev), out, b.table.to(dev, torch.int32), b.kv_len.to(dev), gate=row[:, :1024],
                        gated=True)
    gate = row[:, :1024].cpu().view(2, 4, 256)[..., 128:]
    b.check(out.cpu().view(2, 4, 128), b.want(gate=gate))


def test_attention_mixed_types(gpu):
    b = Batch(gpu, [(1, 333), (1, 50)], 4, 2, 128, 16, F16, F16)
    assert rel(b.run(od=F32), b.want()) < 1e-5
    b = Batch(gpu, [(1, 333), (1, 50)], 4, 2, 128, 16, F16, F32)
    assert rel(b.run(od=F16), b.want()) < 1e-3


@pytest.mark.parametrize("qd,rows", [(F32, 1), (F32, 6), (F16, 100)])
def test_attention_peaked_scores(gpu, qd, rows):
    """Scores of up to about 100: one key has all the weight, and most weights are 0."""
    b = Batch(gpu, [(rows, 700)], 4, 2, 128, 16, F16, qd, q_size=20.0)
    got, want = b.run(), b.want()
    assert got.isfinite().all()
    # (a score's own f32 rounding: 100 2^-24 = 6e-6 of a weight)
    assert rel(got, want) < (3e-5 if qd is F32 else 1e-3)


@pytest.mark.parametrize("cd", [F16, I8])
@pytest.mark.parametrize("rows,qd", [(1, F32), (5, F32), (90, F16)])
def test_attention_pages_outside(gpu, cd, rows, qd):
    """Tokens of a page outside the cache are not visible."""
    b = Batch(gpu, [(rows, 400), (rows, 300)], 4, 2, 128, 32, cd, qd)
    b.table[0, 2], b.table[1, 0], b.table[1, 5] = -7, 2**31 - 1, b.cache.num_pages

    def visible(s):
        ok = torch.ones([400, 300][s], dtype=torch.bool)
        for p in ([2], [0, 5])[s]:
            ok[32 * p:32 * p + 32] = False
        return ok

    want = attention(b.q, b.k_of, b.v_of, b.spans, 1 / math.sqrt(128), visible=visible)
    b.check(b.run(), want)


def test_attention_arrays_out_of_range(gpu):
    """kv_len beyond the table, negative, q_start beyond T or decreasing: no
    access out of bounds, and calls after it are right."""
    dev = gpu.device
    b = Batch(gpu, [(1, 100), (1, 64), (1, 30)], 4, 2, 64, 16, F16, F32)
    want = b.run()
    q, table = b.q.flatten(1).to(dev), b.table.to(dev, torch.int32)
    out = torch.empty(3, 256, device=dev)
    for kv in ([100, -5, 2**31 - 1], [10**6, 64, 30]):
        sta.paged_attention(gpu, b.cache, q, out, table, torch.tensor(kv, dtype=torch.int32, device=dev))
    for start in ([0, 1, 2, 99], [-3, 1, 2, 3], [3, 0, 3, 0], [0, 3, 0, 3]):
        sta.paged_attention(gpu, b.cache, q, out, table, b.kv_len.to(dev), torch.tensor(start, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert torch.equal(b.run(), want)


def test_attention_long_cache(gpu):
    """Elements of the cache past 2^32."""
    nkv, hd, page = 8, 128, 256
    pages = 2**32 // (nkv * hd * page) + 40
    dev = gpu.device
    c = sta.KvCache(gpu, pages, page, nkv, hd, I8)
    n = 700
    g = rng(4)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device=dev)
    slots = c.slots(table, torch.arange(n, device=dev)[None])[0]
    kv = torch.randn(2, n, nkv * hd, generator=g).to(dev)
    sta.qk_norm_rope_store(gpu, c, None, kv[0], kv[1], None, slots)
    ko, vo = (torch.empty(n, nkv, hd, device=dev) for _ in range(2))
    sta.kv_read(gpu, c, slots, ko, vo)
    assert rel(ko.flatten(1), kv[0]) < 0.01 and rel(vo.flatten(1), kv[1]) < 0.01
    q = torch.randn(1, 16 * hd, generator=g).to(dev)
    out = torch.empty_like(q)
    sta.paged_attention(gpu, c, q, out, table, torch.tensor([n], dtype=torch.int32, device=dev))
    want = attention(q.cpu().view(1, 16, hd), lambda b: ko.cpu().double(), lambda b: vo.cpu().double(), [(0, 1, n)], 1 / math.sqrt(hd))
    assert rel(out.cpu().view(1, 16, hd), want) < 1e-5


def test_attention_stream_and_repeat(gpu):
    """On another stream than the tensors', and the same bits every time."""
    b = Batch(gpu, [(1, 3000), (1, 200), (1, 900)], 8, 2, 128, 16, F16, F32)
    first = b.run()
    s = torch.cuda.Stream(device=gpu.device)
    s.wait_stream(torch.cuda.current_stream(gpu.device))
    with torch.cuda.stream(s):
        for _ in range(5):
            assert torch.equal(b.run(), first)
    torch.cuda.current_stream(gpu.device).wait_stream(s)


def test_attention_uses_the_kernel(gpu):
    b = Batch(gpu, [(1, 100)], 4, 2, 128, 16, F16, F32)
    launches()
    b.run()
    assert launches() == ["attn_kernel"]


def test_decode_graph_replays(gpu):
    """Captured advance, store and attention, replayed as the sequences grow,
    equal to the same steps run eagerly."""
    nh, nkv, hd, page, B, width = 8, 2, 128, 16, 3, 8 * 256 + 4 * 128
    dev = gpu.device
    cos, sin = (t.to(dev) for t in tables(256, hd))

    class Rows:
        qkv = torch.zeros(B, width, device=dev)
        attn = torch.zeros(B, nh * hd, device=dev)

    def make():
        c = sta.KvCache(gpu, 40, page, nkv, hd)
        table = torch.arange(B * 10, dtype=torch.int32, device=dev).view(B, 10)
        p = sta.PagedAttention(gpu, [c], nh, table, cos, sin, norms=[(torch.ones(hd, device=dev),) * 2], gated=True)
        p.kv_len.copy_(torch.tensor([0, 5, 31]))
        c.k.zero_(), c.v.zero_()
        return p

    def step(p, b):
        p.advance()
        p.attention(0, b)

    eager, p, rows = make(), make(), Rows()
    g = rng(8)
    inputs = [torch.randn(B, width, generator=g).to(dev) for _ in range(40)]
    want = []
    for x in inputs:
        rows.qkv.copy_(x)
        step(eager, rows)
        want.append(rows.attn.clone())
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step(p, rows)  # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(p, rows)
    torch.cuda.current_stream(dev).wait_stream(s)
    p.kv_len.copy_(torch.tensor([0, 5, 31]))
    for x, w in zip(inputs, want):
        rows.qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows.attn, w)


def test_prefill_then_decode(gpu):
    """A prompt stored and attended in one call, then token by token: the
    same rows as one prompt of all tokens."""
    nh, nkv, hd, page, n = 8, 2, 128, 32, 50
    dev = gpu.device
    width = (nh + 2 * nkv) * hd
    cos, sin = (t.to(dev) for t in tables(64, hd))
    g = rng(12)
    qkv = torch.randn(n, width, generator=g).half()
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=dev)

    def make():
        return sta.PagedAttention(gpu, [sta.KvCache(gpu, 3, page, nkv, hd)], nh, table, cos, sin, norms=[(torch.ones(hd, device=dev),) * 2])

    def prompt(p, m):
        pos = torch.arange(m, dtype=torch.int32, device=dev)
        out = torch.empty(m, nh * hd, dtype=F16, device=dev)
        p.prefill(0, qkv[:m].to(dev), out, torch.tensor([0, m], dtype=torch.int32, device=dev), pos, p.cache.slots(table, pos[None])[0],
                  torch.tensor([m], dtype=torch.int32, device=dev))
        return out.float()

    whole = prompt(make(), n)
    p = make()
    prompt(p, n - 5)
    p.kv_len.fill_(n - 5)

    class Rows:
        pass

    b = Rows()
    b.attn = torch.empty(1, nh * hd, device=dev)
    for i in range(n - 5, n):
        p.advance()
        b.qkv = qkv[i:i + 1].float().to(dev)
        p.attention(0, b)
        assert rel(b.attn, whole[i:i + 1]) < 1e-3
