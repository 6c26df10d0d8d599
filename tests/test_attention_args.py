"""Refusals of the cache, attention and log-probability calls (CPU, no GPU):
the Python helpers' with a stand-in for the context, and the C entry points'
own, which look at their arguments before they touch the context or a GPU."""
import ctypes

import pytest
import torch

import shady_thinker_amd as sta
from attn_util import indices, shapes
from shady_thinker_amd._lib import ST_F16, ST_F32, ST_I8, KvCacheStruct, lib

ST_ERR_INVALID, ST_ERR_SHAPE, ST_ERR_ALIGN = 1, 2, 3  # (st_status)
F32, F16, I8, I32 = torch.float32, torch.float16, torch.int8, torch.int32
PAGES, PAGE, NKV, HD, NH, T = 4, 16, 2, 64, 4, 3


class NoGpu:
    handle = None
    device = "cpu"

    def sync_stream(self):
        pass


G = NoGpu()


def cache(dtype=F16):
    return sta.KvCache(G, PAGES, PAGE, NKV, HD, dtype)


def i32(*shape):
    return torch.zeros(*shape, dtype=I32)


# ------------------------------------------------------------ Python helpers
def test_cache_refusals():
    for kw in (dict(page_size=24), dict(head_dim=96), dict(num_pages=0), dict(n_kv_heads=0)):
        a = dict(num_pages=PAGES, page_size=PAGE, n_kv_heads=NKV, head_dim=HD)
        with pytest.raises(ValueError):
            sta.KvCache(G, **{**a, **kw})
    with pytest.raises(TypeError):
        sta.KvCache(G, PAGES, PAGE, NKV, HD, F32)
    c = cache()
    with pytest.raises(TypeError):
        sta.KvCache.of(c.k, c.v.to(I8), PAGE)
    with pytest.raises(ValueError):
        sta.KvCache.of(c.k, c.v, 2 * PAGE)
    with pytest.raises(ValueError):
        sta.KvCache.of(c.k, c.v[:2], PAGE)
    with pytest.raises(ValueError):
        sta.KvCache.of(c.k.repeat(1, 1, 1, 1, 1, 2)[..., ::2], c.v, PAGE)
    with pytest.raises((ValueError, TypeError)):
        sta.KvCache.of(c.k.to(I8), c.v.to(I8), PAGE)  # int8 without scales


def test_layout():
    """Every element of a cache has one place, and the tensors that KvCache
    makes are those that the layout's definition asks for."""
    c = cache(I8)
    assert [tuple(t.shape) for t in (c.k, c.v, c.k_scale)] == [tuple(s) for s in shapes(PAGES, NKV, PAGE, HD)]
    for at, t in zip(indices(torch.arange(PAGES * PAGE), NKV, PAGE, HD), (c.k, c.v, c.k_scale)):
        assert torch.equal(at.flatten().sort().values, torch.arange(t.numel()))


def store(**kw):
    a = dict(q=torch.zeros(T, NH * HD), k=torch.zeros(T, NKV * HD), v=torch.zeros(T, NKV * HD), q_out=torch.zeros(T, NH * HD),
             slots=i32(T), positions=i32(T), cos=torch.zeros(8, 16), sin=torch.zeros(8, 16))
    a.update(kw)
    sta.qk_norm_rope_store(G, cache(), a.pop("q"), a.pop("k"), a.pop("v"), a.pop("q_out"), a.pop("slots"), **a)


@pytest.mark.parametrize("kw", [
    dict(k=torch.zeros(T, NKV * HD, dtype=torch.float64)), dict(v=torch.zeros(T, NKV * HD, dtype=F16)),
    dict(q=torch.zeros(T, NH * HD, dtype=F16)), dict(v=torch.zeros(T, NKV * HD + 8)), dict(q=torch.zeros(T + 1, NH * HD)),
    dict(k=torch.zeros(NKV * HD, T).T), dict(q_out=torch.zeros(T, HD)), dict(q_out=None), dict(q=None), dict(slots=i32(T - 1)),
    dict(slots=torch.zeros(T, dtype=torch.int64)), dict(positions=None), dict(sin=None), dict(cos=None), dict(cos=torch.zeros(16)),
    dict(sin=torch.zeros(4, 16)), dict(q_weight=torch.zeros(HD, dtype=F16)), dict(k_weight=torch.zeros(HD - 1))])
def test_store_refusals(kw):
    with pytest.raises((ValueError, TypeError)):
        store(**kw)


@pytest.mark.parametrize("kw", [
    dict(k_out=torch.zeros(T, NKV, HD, dtype=I8)), dict(v_out=torch.zeros(T, NKV, HD, dtype=F16)), dict(v_out=torch.zeros(T - 1, NKV, HD)),
    dict(k_out=torch.zeros(T, NKV, 2 * HD)[..., ::2]), dict(slots=torch.zeros(T))])
def test_read_refusals(kw):
    a = dict(slots=i32(T), k_out=torch.zeros(T, NKV, HD), v_out=torch.zeros(T, NKV, HD))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        sta.kv_read(G, cache(), **a)


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(T, NH, HD)), dict(q=torch.zeros(T, NH * HD + 8)), dict(q=torch.zeros(T, NH * HD, dtype=torch.bfloat16)),
    dict(q=torch.zeros(T, 2 * NH * HD)[:, ::2]), dict(out=torch.zeros(T - 1, NH * HD)), dict(out=torch.zeros(T, NH * HD, dtype=I32)),
    dict(table=i32(T * 2)), dict(table=torch.zeros(T, 2)), dict(kv_len=i32(T - 1)), dict(q_start=i32(T)), dict(slopes=torch.zeros(NH - 1)),
    dict(gate=torch.zeros(T, NH * HD - 8)), dict(gate=torch.zeros(T, NH * HD), gated=True), dict(gate=torch.zeros(NH * HD, T).T)])
def test_attention_refusals(kw):
    a = dict(q=torch.zeros(T, NH * HD), out=torch.zeros(T, NH * HD), table=i32(T, 2), kv_len=i32(T))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        sta.paged_attention(G, cache(), **a)


@pytest.mark.parametrize("kw", [
    dict(logits=torch.zeros(T * 100)), dict(logits=torch.zeros(T, 100, dtype=torch.bfloat16)), dict(logits=torch.zeros(100, T).T),
    dict(tokens=None), dict(tokens=i32(T - 1)), dict(rank=torch.zeros(T)), dict(logprob=torch.zeros(T, dtype=F16)), dict(top_ids=None),
    dict(top_ids=i32(T - 1, 5)), dict(top_logprobs=torch.zeros(T, 4)), dict(entropy=torch.zeros(T - 1))])
def test_logprobs_refusals(kw):
    a = dict(logits=torch.zeros(T, 100), tokens=i32(T), logprob=torch.zeros(T), entropy=torch.zeros(T), rank=i32(T), top_ids=i32(T, 5),
             top_logprobs=torch.zeros(T, 5))
    a.update(kw)
    with pytest.raises((ValueError, TypeError)):
        sta.token_logprobs(G, **a)


def test_paged_attention_refuses_mixed_caches():
    with pytest.raises(ValueError):
        sta.PagedAttention(G, [cache(), sta.KvCache(G, PAGES, 32, NKV, HD)], NH, i32(1, 2))


# ------------------------------------------------------------- entry points
MEM = (ctypes.c_char * (1 << 16))()
AT = (ctypes.addressof(MEM) + 255) // 256 * 256  # (never read: every call here is refused)


def kv(dtype=ST_F16, k=AT, v=AT, ks=AT, vs=AT, pages=PAGES, page=PAGE, heads=NKV, hd=HD):
    return ctypes.addressof(KEEP.setdefault((dtype, k, v, ks, vs, pages, page, heads, hd), KvCacheStruct(k, v, ks, vs, dtype, pages, page, heads, hd)))


KEEP: dict = {}
BAD_CACHES = [(dict(k=None), ST_ERR_INVALID), (dict(v=None), ST_ERR_INVALID), (dict(dtype=9), ST_ERR_INVALID),
              (dict(dtype=ST_I8, ks=None), ST_ERR_INVALID), (dict(page=24), ST_ERR_SHAPE), (dict(hd=96), ST_ERR_SHAPE),
              (dict(pages=0), ST_ERR_SHAPE), (dict(heads=0), ST_ERR_SHAPE), (dict(k=AT + 8), ST_ERR_ALIGN)]


def c_store(ctx=AT, c=None, q=AT, k=AT, v=AT, dt=ST_F32, qs=NH * HD, ks=NKV * HD, vs=NKV * HD, qh=HD, qw=None, kw=None, eps=1e-6, cos=None,
            sin=None, rot=0, n_pos=0, pos=None, slots=AT, out=AT, od=ST_F32, T=T, heads=NH, flags=0):
    return lib().st_qk_norm_rope_store(ctx, kv() if c is None else c, q, k, v, dt, qs, ks, vs, qh, qw, kw, eps, cos, sin, rot, n_pos, pos,
                                       slots, out, od, T, heads, flags)


def c_read(ctx=AT, c=None, slots=AT, k=AT, v=AT, dt=ST_F32, T=T):
    return lib().st_kv_read(ctx, kv() if c is None else c, slots, k, v, dt, T)


def c_attn(ctx=AT, c=None, q=AT, qd=ST_F32, table=AT, pages=2, kv_len=AT, start=None, scale=0.1, cap=0.0, window=0, slopes=None, gate=None,
           gd=ST_F32, gs=NH * HD, gh=HD, out=AT, od=ST_F32, T=T, B=T, heads=NH):
    return lib().st_paged_attention(ctx, kv() if c is None else c, q, qd, table, pages, kv_len, start, scale, cap, window, slopes, gate, gd, gs,
                                    gh, out, od, T, B, heads)


def c_logprobs(ctx=AT, x=AT, dt=ST_F32, stride=100, tokens=AT, lp=AT, ent=AT, rank=AT, ids=AT, tops=AT, M=T, V=100, top=5):
    return lib().st_token_logprobs(ctx, x, dt, stride, tokens, lp, ent, rank, ids, tops, M, V, top)


@pytest.mark.parametrize("kw,code", BAD_CACHES)
@pytest.mark.parametrize("fn", [c_store, c_read, c_attn])
def test_entry_points_refuse_caches(fn, kw, code):
    assert fn(c=kv(**kw)) == code
    assert lib().st_last_error()


@pytest.mark.parametrize("fn,kw,code", [
    (c_store, dict(ctx=None), ST_ERR_INVALID), (c_store, dict(k=None), ST_ERR_INVALID), (c_store, dict(slots=None), ST_ERR_INVALID),
    (c_store, dict(dt=ST_I8), ST_ERR_INVALID), (c_store, dict(out=None), ST_ERR_INVALID), (c_store, dict(T=0), ST_ERR_SHAPE),
    (c_store, dict(ks=HD), ST_ERR_SHAPE), (c_store, dict(k=AT + 4), ST_ERR_ALIGN),
    (c_store, dict(rot=2 * HD, cos=AT, sin=AT, pos=AT, n_pos=8), ST_ERR_SHAPE),
    (c_read, dict(ctx=None), ST_ERR_INVALID), (c_read, dict(v=None), ST_ERR_INVALID), (c_read, dict(dt=ST_I8), ST_ERR_INVALID),
    (c_read, dict(T=0), ST_ERR_SHAPE), (c_read, dict(k=AT + 4), ST_ERR_ALIGN),
    (c_attn, dict(ctx=None), ST_ERR_INVALID), (c_attn, dict(table=None), ST_ERR_INVALID), (c_attn, dict(qd=ST_I8), ST_ERR_INVALID),
    (c_attn, dict(scale=0.0), ST_ERR_INVALID), (c_attn, dict(scale=float("nan")), ST_ERR_INVALID), (c_attn, dict(cap=-1.0), ST_ERR_INVALID),
    (c_attn, dict(cap=float("nan")), ST_ERR_INVALID), (c_attn, dict(window=-1), ST_ERR_INVALID), (c_attn, dict(B=T - 1), ST_ERR_SHAPE),
    (c_attn, dict(heads=3), ST_ERR_SHAPE), (c_attn, dict(heads=65 * NKV), ST_ERR_SHAPE), (c_attn, dict(pages=0), ST_ERR_SHAPE),
    (c_attn, dict(pages=1 << 28), ST_ERR_SHAPE), (c_attn, dict(q=AT + 8), ST_ERR_ALIGN),
    (c_attn, dict(gate=AT, gs=HD), ST_ERR_SHAPE), (c_attn, dict(gate=AT, gs=NH * HD + 4), ST_ERR_ALIGN),
    (c_logprobs, dict(ctx=None), ST_ERR_INVALID), (c_logprobs, dict(x=None), ST_ERR_INVALID), (c_logprobs, dict(tokens=None), ST_ERR_INVALID),
    (c_logprobs, dict(dt=ST_I8), ST_ERR_INVALID), (c_logprobs, dict(M=0), ST_ERR_SHAPE), (c_logprobs, dict(V=0), ST_ERR_SHAPE),
    (c_logprobs, dict(stride=99), ST_ERR_SHAPE), (c_logprobs, dict(top=33), ST_ERR_SHAPE), (c_logprobs, dict(ids=None), ST_ERR_INVALID)])
def test_entry_points_refuse(fn, kw, code):
    assert fn(**kw) == code
    assert lib().st_last_error()
