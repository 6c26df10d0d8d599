"""Attention where something is not finite, out of all proportion or past an
end: in the rows that see it, and nowhere else, whatever kernel a call takes
and however it is cut.

Tolerances (relative 2-norm) as in test_gpu_attention.py: f16 output and
weights 1e-3, f32 1e-5.
"""
import math

import pytest
import torch

import shady_thinker_amd as sta
from attn_util import attention, indices, rel
from test_gpu_attention import F16, F32, I8, Batch, as_prompt, rng

pytestmark = pytest.mark.gpu


def slot_of(b, p, seq=0):
    page = b.cache.page_size
    return (b.table[seq, p // page] * page + p % page).reshape(1)


# ------------------------------------------------- rows with a NaN, in chunks
@pytest.mark.parametrize("hd,cd", [(128, F16), (64, F16), (256, F16), (128, I8)])
@pytest.mark.parametrize("rows,kv", [(100, 4000), (16, 3000), (100, 100)])
def test_nan_query(gpu, hd, cd, rows, kv):
    """A NaN query's row and head are NaN, over a long cache (chunks) as over
    a short one; the others are what they are without it."""
    b = Batch(gpu, [(rows, kv)], 4, 2, hd, 16, cd, F16, wide=1 << 15)
    r, h = rows // 3, 3
    b.q[r, h, 5] = math.nan
    got, want = as_prompt(b), b.want()
    bad = torch.zeros(want.shape, dtype=torch.bool)
    bad[r, h] = True
    assert got[bad].isnan().all()
    assert rel(got[~bad], want[~bad]) < 1e-3


@pytest.mark.parametrize("rows,kv,hd,cd,qd", [
    (1, 100, 128, F16, F32), (1, 4000, 128, F16, F32), (1, 9000, 256, I8, F32), (5, 4000, 64, F16, F32), (5, 4000, 128, I8, F16),
    (3, 700, 256, F16, F16)])
def test_nan_query_of_few_rows(gpu, rows, kv, hd, cd, qd):
    """The same in calls of one row and of a few."""
    b = Batch(gpu, [(rows, kv)] * 2, 4, 2, hd, 16, cd, qd)
    r, h = rows, 3  # (the second sequence's first row)
    b.q[r, h, 5] = math.nan
    got, want = b.run(), b.want()
    bad = torch.zeros(want.shape, dtype=torch.bool)
    bad[r, h] = True
    assert got[bad].isnan().all()
    assert rel(got[~bad], want[~bad]) < (1e-5 if qd is F32 else 1e-3)


@pytest.mark.parametrize("hd,cd", [(128, F16), (256, F16), (64, I8)])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_key_alone_in_a_chunk(gpu, hd, cd, window):
    """A NaN key (int8: key scale) at a chunk's first place is all that its
    own row sees of the chunk."""
    rows, kv, nkv, nh = 600, 4000, 1, 2
    b = Batch(gpu, [(rows, kv)], nh, nkv, hd, 16, cd, F16, wide=1 << 15)
    p = 3584  # (a multiple of 256 and 512 keys, as the chunks are)
    ki, _, si = indices(slot_of(b, p), nkv, 16, hd)
    t, at = (b.cache.k, ki[0, 0, 7]) if cd is F16 else (b.cache.k_scale, si[0, 0])
    t.view(-1)[at] = math.nan
    got, want = b.run(window=window), b.want(window=window)
    at_row = torch.arange(rows) + kv - rows
    see = (at_row >= p) & ((at_row < p + window) if window else True)
    assert got[see].isnan().all()
    assert got[~see].isfinite().all()
    assert rel(got[~see], want[~see]) < 1e-3


# -------------------------------------------------- the end of a page table
@pytest.mark.parametrize("cd", [F16, I8])
def test_steps_past_the_table(gpu, cd):
    """Captured steps of a batch of which one sequence after the other fills
    its table: it attends to what is stored, and every other sequence's tokens
    stay where they are, bit for bit."""
    nh, nkv, hd, page, B = 4, 2, 64, 16, 3
    dev = gpu.device
    width = (nh + 2 * nkv) * hd
    c = sta.KvCache(gpu, 8, page, nkv, hd, cd)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None:
            t.zero_()
    table = torch.tensor([[3, 6], [5, 0], [2, 7]], dtype=torch.int32, device=dev)
    p = sta.PagedAttention(gpu, [c], nh, table)
    start = torch.tensor([30, 4, 31], dtype=torch.int32)

    class Rows:
        qkv = torch.zeros(B, width, device=dev)
        attn = torch.zeros(B, nh * hd, device=dev)

    def step():
        p.advance()
        p.attention(0, Rows)

    stream = torch.cuda.Stream(device=dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        step()  # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    torch.cuda.current_stream(dev).wait_stream(stream)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None:
            t.zero_()
    p.kv_len.copy_(start)
    g = rng(6)
    every = torch.arange(page * 8, dtype=torch.int32, device=dev)

    def contents():
        ko, vo = (torch.empty(page * 8, nkv, hd, device=dev) for _ in range(2))
        sta.kv_read(gpu, c, every, ko, vo)
        return ko.cpu().double(), vo.cpu().double()

    places = [(table[b].cpu()[torch.arange(32) // page] * page + torch.arange(32) % page).long() for b in range(B)]
    lens, were = start.tolist(), contents()
    for i in range(6):
        x = torch.randn(B, width, generator=g)
        Rows.qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        now = contents()
        touched = [int(places[b][n]) for b, n in enumerate(lens) if n < 32]
        rest = torch.ones(page * 8, dtype=torch.bool)
        rest[touched] = False
        assert all(torch.equal(a[rest], z[rest]) for a, z in zip(were, now))
        lens, were = [min(n + 1, 32) for n in lens], now
        assert p.kv_len.tolist() == lens
        want = attention(x[:, :nh * hd].view(B, nh, hd), lambda b: now[0][places[b][:lens[b]]], lambda b: now[1][places[b][:lens[b]]],
                         [(b, 1, lens[b]) for b in range(B)], 1 / math.sqrt(hd))
        assert rel(Rows.attn.view(B, nh, hd), want) < 1e-5


# ---------------------------------------- several things that are not finite
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,kv,hd,qd,wide", [
    (100, 500, 128, F16, 1 << 15), (100, 4000, 128, F16, 1 << 15), (70, 400, 256, F16, 1 << 15), (300, 3000, 64, F16, 1 << 15),
    (6, 400, 128, F16, 0), (20, 3000, 256, F16, 0)])
def test_infinite_values_of_both_signs(gpu, rows, kv, hd, qd, wide, gated):
    """+inf, which every row sees, and -inf in the same dim, which some see:
    theirs is NaN. A NaN query's row stays NaN where it sees an infinity."""
    nh, nkv, d = 6, 2, 21
    b = Batch(gpu, [(rows, kv)], nh, nkv, hd, 16, F16, qd, wide=wide)
    p = kv - rows + rows // 2
    v = b.cache.v.view(-1)
    for at, value, dim in ((10, math.inf, d), (p, -math.inf, d), (p, math.inf, d + 1)):
        v[indices(slot_of(b, at), nkv, 16, hd)[1][0, 1, dim]] = value
    nan_row = rows - 2
    b.q[nan_row, nh - 1, 3] = math.nan
    gate = torch.randn(rows, nh, hd, generator=rng(2)).to(qd) if gated else None
    got, want = b.run(gate=gate), b.want(gate=gate)
    see = torch.arange(rows) + kv - rows >= p
    special = torch.zeros_like(want, dtype=torch.bool)
    special[:, nh // 2:, d] = True
    special[see, nh // 2:, d + 1] = True
    special[nan_row, nh - 1] = True
    other = slice(nh // 2, nh - 1)
    assert (got[~see, other, d] == math.inf).all() and got[see, other, d].isnan().all()
    assert (got[see, other, d + 1] == math.inf).all()
    assert got[nan_row, nh - 1].isnan().all()
    assert rel(got[~special], want[~special]) < (1e-5 if qd is F32 else 1e-3)


# --------------------------------------- int8: value scales of any proportion
def held(b, seq=0):
    """A sequence's keys and values as the int8 cache holds them, 64 bits."""
    kv = int(b.kv_len[seq])
    page = b.cache.page_size
    at = torch.arange(kv)
    ki, vi, si = indices(b.table[seq][at // page] * page + at % page, b.nkv, page, b.hd)
    c = b.cache
    of = lambda t, i: t.cpu().flatten()[i].double()
    return of(c.k, ki) * of(c.k_scale, si)[..., None], of(c.v, vi) * of(c.v_scale, si)[..., None]


def plain(b, **kw):
    k, v = held(b)
    return attention(b.q, lambda s: k, lambda s: v, b.spans, 1 / math.sqrt(b.hd), **kw)


INT8 = [(100, 150, 128, F16, 1 << 15), (100, 150, 64, F16, 1 << 15), (70, 120, 256, F16, 1 << 15), (100, 3000, 128, F16, 1 << 15),
        (6, 100, 128, F32, 0), (6, 3000, 64, F32, 0), (6, 100, 256, F16, 0)]


def each_row(got, want, tol):
    e = [rel(got[r], want[r]) for r in range(len(want))]
    print("largest row error", max(e))
    assert max(e) < tol


@pytest.mark.parametrize("ratio", [2.0**20, 2.0**45, 2.0**100])
@pytest.mark.parametrize("rows,kv,hd,qd,wide", INT8)
def test_value_scale_of_a_later_token(gpu, rows, kv, hd, qd, wide, ratio):
    """A token whose values are far larger than the others' changes nothing
    for the rows before it, in whose block it is, nor for those whose window
    it has left."""
    b = Batch(gpu, [(rows, kv)], 6, 2, hd, 16, I8, qd, wide=wide)
    p = kv - rows // 2
    si = indices(slot_of(b, p), 2, 16, hd)[2]
    b.cache.v_scale.view(-1)[si[0]] *= ratio
    before = torch.arange(rows) + kv - rows < p
    tol = 1e-5 if qd is F32 else 1e-3
    got, want = b.run(), plain(b)
    each_row(got[before], want[before], tol)
    if qd is F32:
        each_row(got, want, tol)
    got, want = b.run(window=2), plain(b, window=2)
    out = before | (torch.arange(rows) + kv - rows >= p + 2)
    each_row(got[out], want[out], tol)


@pytest.mark.parametrize("ratio", [2.0**24, 2.0**30, 2.0**36])
@pytest.mark.parametrize("rows,kv,hd,qd,wide", INT8 + [(1, 100, 128, F32, 0), (1, 4000, 128, F32, 0)])
def test_value_scale_of_an_unlikely_token(gpu, rows, kv, hd, qd, wide, ratio):
    """A token that every row sees, with values far larger than the others'
    and a weight as much smaller: the others' keep their bits."""
    nh, nkv = 6, 2
    b = Batch(gpu, [(rows, kv)], nh, nkv, hd, 16, I8, qd, wide=wide)
    p = 33
    b.q[:, :, 0] = 3.0
    ki, vi, si = indices(slot_of(b, p), nkv, 16, hd)
    # its key: a score of about -log(ratio) from dim 0 alone
    k = b.cache.k.view(-1)
    k[ki[0].flatten()] = 0
    k[ki[0, :, 0]] = -127
    b.cache.k_scale.view(-1)[si[0]] = math.log(ratio) * math.sqrt(hd) / 3.0 / 127
    b.cache.v_scale.view(-1)[si[0]] *= ratio
    each_row(b.run(), plain(b), 1e-5 if qd is F32 else 1e-3)


# ------------------------------------------------------ caps of any size
@pytest.mark.parametrize("cap", [1e-42, 1e-3, 0.7, 30.0, 1e4, 1e6, 1e12, 3e38, math.inf])
@pytest.mark.parametrize("rows,kv,nh,hd,cd,qd,wide", [
    (100, 300, 4, 128, F16, F16, 1 << 15), (100, 3000, 4, 128, I8, F16, 1 << 15), (70, 200, 4, 256, F16, F16, 1 << 15),
    (70, 200, 4, 64, I8, F16, 1 << 15), (5, 300, 4, 128, F16, F32, 0), (1, 2000, 4, 64, I8, F32, 0), (9, 200, 4, 256, F16, F16, 0)])
def test_cap_of_any_size(gpu, rows, kv, nh, hd, cd, qd, wide, cap):
    """A cap far over the scores leaves them as they are, to f32's bits; a
    tiny one leaves their signs; a score of 0 stays 0."""
    b = Batch(gpu, [(rows, kv)], nh, 2, hd, 16, cd, qd, wide=wide)
    b.q[0] = 0.0
    want = b.want(cap=0.0 if cap == math.inf else cap)
    each_row(b.run(cap=cap), want, 1e-5 if qd is F32 else 1e-3)


@pytest.mark.parametrize("cd", [F16, I8])
@pytest.mark.parametrize("q_size,cap", [(1.0, 5.0), (20.0, 5.0), (20.0, 50.0), (20.0, 200.0), (8.0, 1e5)])
def test_capped_prompt(gpu, cd, q_size, cap):
    """Scores far below, about and far above the cap, in one tile."""
    b = Batch(gpu, [(100, 400)], 4, 2, 128, 16, cd, F16, q_size=q_size, wide=1 << 15)
    b.q[::3] *= 0.02
    each_row(b.run(cap=cap), b.want(cap=cap), 1e-3)
