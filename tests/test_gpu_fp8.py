"""The 8-bit floating point operators on the GPU against 64-bit forms
(tests/fp8_util.py): norms with the residual's addition, quantised rows, their
product with block-scaled weights."""
import math

import pytest
import torch

import shady_thinker_amd as sta
from shady_thinker_amd._lib import launches
from fp8_util import B, F8, U, blocks, check_product, check_rows, rows_of, scales, weight_of

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
DEV = "cuda:0"


def rand(seed, *shape, dtype=F32, chan=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if chan:  # a few large channels
        x = x * (1.0 + 15.0 * (torch.randn(shape[-1], generator=g) > 2.0))
    return x.to(dtype).to(DEV)


def silu64(a):
    return a / (1.0 + torch.exp(-a))


# (f32 silu(a) b: exp(-a) off by 2^-24 (1 + 2 |a|) and the function's own steps,
# then a sum, a quotient and a product of a step each)
def silu_err(a):
    return (8.0 + 2.0 * a.double().cpu().abs()) * 2 * U


@pytest.mark.parametrize("m,k", [(1, 16), (1, 4096), (2, 112), (3, 128), (5, 144), (17, 2752), (33, 2048), (129, 2064), (1, 11008),
                                 (300, 4112)])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("silu", [False, True])
def test_quant(gpu, m, k, dtype, silu):
    x = rand(m + k, m, 2 * k, dtype=dtype, chan=True)
    rows = sta.Fp8Rows(gpu, m, k)
    a, b = x[:, :k], x[:, k:]
    sta.fp8_quant(gpu, a, rows, b if silu else None)
    if silu:
        check_rows(rows.data, rows.scale, silu64(a.double().cpu()) * b.double().cpu(), silu_err(a))
    else:
        check_rows(rows.data, rows.scale, a.double().cpu(), 0.0)


def test_quant_rounds_to_nearest_even(gpu):
    """With scales that are powers of two, every value of e4m3, every tie
    between two and every f32 next to a tie round as torch's conversion does."""
    every = torch.arange(0, 0x7F, dtype=torch.uint8).view(F8).float()
    ties = (every[1:] + every[:-1]) / 2
    near = torch.cat([every, ties, torch.nextafter(ties, ties * 2), torch.nextafter(ties, ties * 0)])
    near = torch.cat([near, -near])
    x = torch.full((blocks(near.numel() * 2), B), 448.0)
    x[:, 1:64] = torch.nn.functional.pad(near, (0, x.shape[0] * 63 - near.numel())).view(-1, 63)
    for p in (0, -20, 9):
        rows = sta.Fp8Rows(gpu, x.shape[0], B)
        sta.fp8_quant(gpu, (x * 2.0**p).to(DEV), rows)
        assert torch.equal(rows.scale.cpu(), torch.full((1, x.shape[0]), 2.0**p))
        assert torch.equal(rows.data.cpu().view(torch.uint8), x.to(F8).view(torch.uint8))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_quant_values_out_of_the_ordinary(gpu, dtype):
    """Zero blocks, the type's smallest and largest values, infinities, NaN:
    each stays in its own block."""
    big = torch.finfo(dtype).max
    x = rand(3, 6, 3 * B, dtype=dtype)
    x[0, :B] = 0
    x[1] = torch.finfo(dtype).smallest_normal / 8  # (a subnormal)
    x[2] = big
    x[2, 7] = -big
    x[3, 5], x[3, 9] = math.inf, -math.inf
    x[4, B + 3] = math.nan
    x[5] = 0
    rows = sta.Fp8Rows(gpu, 6, 3 * B)
    sta.fp8_quant(gpu, x, rows)
    fine = torch.ones(6, dtype=torch.bool)
    fine[3], fine[4] = False, False
    check_rows(rows.data[fine.to(DEV)], rows.scale[:, fine.to(DEV)], x[fine.to(DEV)].double().cpu(), 0.0)
    d, s = rows.data.float().cpu(), rows.scale.cpu()
    assert s[0, 3] == math.inf and d[3, 5] == 448 and d[3, 9] == -448 and (d[3, :B].abs() > 0).sum() == 2
    assert math.isnan(s[1, 4]) and torch.isfinite(s[[0, 2], 4]).all()
    for r, skip in ((3, 0), (4, 1)):
        for b in {0, 1, 2} - {skip}:
            at = slice(b * B, b * B + B)
            check_rows(rows.data[r:r + 1, at], rows.scale[b:b + 1, r:r + 1], x[r:r + 1, at].double().cpu(), 0.0)


def test_silu_ends(gpu):
    """Large magnitudes: silu is a or 0, not NaN."""
    a = torch.tensor([[100.0, -100.0, 1e4, -1e4, 88.0, -88.0, 3e38, -3e38] + [0.0] * 8], device=DEV)
    rows = sta.Fp8Rows(gpu, 1, 16)
    sta.fp8_quant(gpu, a, rows, torch.full_like(a, 1e-30))
    want = silu64(a.double().cpu()) * 1e-30
    got = rows.dequantise().double().cpu()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= want.abs().max() / 448 * 0.5 * 2.0**-9 * (1 + 1e-5) + want.abs() * (2.0**-4 + 1e-5)).all()


# Norms: a thread's 8 P squares in a row, 6 steps in the wave, up to 16 waves,
# the mean, eps, square root, quotient: the sum's error is halved by the root;
# then two products and the weight's sum.
def norm_err(d):
    return ((8 * 4 + 6 + 16 + 3) / 2 + 6) * 2 * U


NORMS = [(1, 4096), (1, 16), (2, 128), (3, 144), (5, 2560), (31, 4112), (77, 8192), (4, 8208), (3, 16400), (2, 32768), (300, 512)]


@pytest.mark.parametrize("m,d", NORMS)
@pytest.mark.parametrize("res,x,y,q", [(F32, F32, None, True), (F32, F32, F32, True), (F16, F16, F16, True), (F16, F16, None, True),
                                       (F32, F16, F32, False), (F16, F32, F16, False), (F32, None, F32, True), (F16, None, None, True)])
def test_norm(gpu, m, d, res, x, y, q):
    r0 = rand(m + d, m, d, dtype=res, chan=True)
    x0 = None if x is None else rand(m + d + 1, m, d, dtype=x)
    one_plus = bool(m % 2)
    w = rand(7, d) * 0.2 + (0.0 if one_plus else 1.0)
    r, out = r0.clone(), None if y is None else torch.empty(m, d, dtype=y, device=DEV)
    rows = sta.Fp8Rows(gpu, m, d) if q else None
    sta.add_rmsnorm(gpu, r, w, x0, out, rows, eps=1e-5, one_plus=one_plus)
    s = r0.double().cpu() + (0 if x is None else x0.double().cpu())
    if x is None:
        assert torch.equal(r, r0)
    else:
        half = torch.finfo(res).eps / 2
        assert ((r.cpu().double() - s).abs() <= s.abs() * (half + U) + 2.0**-25).all()
    want = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5) * (w.double().cpu() + (1.0 if one_plus else 0.0))
    # (the sum r + x may cancel: its rounding is half a step of the sum, so relative to it)
    if y is not None:
        half = torch.finfo(y).eps / 2
        assert ((out.cpu().double() - want).abs() <= want.abs() * (half + norm_err(d)) + 2.0**-25).all()
    if q:
        check_rows(rows.data, rows.scale, want, norm_err(d))


def test_norm_in_place_and_out_of_place(gpu):
    """The same bits into a buffer of its own, into the residual, and with y in
    x's buffer; parts of wider rows; what lies around is left alone."""
    m, d = 9, 2576
    wide = rand(1, m, 3 * d)
    r0, x0, w = wide[:, :d].clone(), wide[:, d:2 * d].clone(), rand(2, d)
    outs = []
    for kind in range(3):
        buf = torch.full((m, 3 * d), 7.0, device=DEV)
        r, x, o = buf[:, :d], buf[:, d:2 * d], buf[:, 2 * d:]
        r.copy_(r0), x.copy_(x0)
        rows = sta.Fp8Rows(gpu, m, d)
        if kind == 0:
            ro = torch.empty(m, d, device=DEV)
            sta.add_rmsnorm(gpu, r, w, x, o, rows, residual_out=ro)
            assert torch.equal(r, r0) and torch.equal(x, x0)
        else:
            ro, o = r, x if kind == 2 else o
            sta.add_rmsnorm(gpu, r, w, x, o, rows)
        outs.append((ro.clone(), o.clone(), rows.data.view(torch.uint8).clone(), rows.scale.clone()))
        if kind == 2:
            assert (buf[:, 2 * d:] == 7.0).all()
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_norm_over_the_residual(gpu, dtype):
    """y in the residual's buffer (no sum goes there): the bits of a buffer of
    its own."""
    m, d = 5, 1040
    r, x, w = rand(1, m, d, dtype=dtype), rand(2, m, d), rand(3, d)
    for add in (None, x):
        ro = None if add is None else torch.empty_like(r)
        want, y = torch.empty_like(r), r.clone()
        sta.add_rmsnorm(gpu, r, w, add, want, residual_out=ro)
        sta.add_rmsnorm(gpu, y, w, add, y, residual_out=ro)
        assert torch.equal(y, want)


def test_norm_rows_keep_to_themselves(gpu):
    """A row of zeros, one with an infinity, one with a NaN, a large one."""
    m, d = 6, 1040
    r0 = rand(1, m, d)
    r0[1], r0[2, 5], r0[3, 700], r0[4] = 0, math.inf, math.nan, r0[4] * 1e15
    r, w = r0.clone(), torch.ones(d, device=DEV)
    y, rows = torch.empty(m, d, device=DEV), sta.Fp8Rows(gpu, m, d)
    sta.add_rmsnorm(gpu, r, w, torch.zeros(m, d, device=DEV), y, rows)
    s = r0.double().cpu()
    want = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6)
    ok = [0, 1, 4, 5]
    assert ((y.cpu().double() - want).abs()[ok] <= want.abs()[ok] * (norm_err(d) + U)).all()
    check_rows(rows.data[ok], rows.scale[:, ok], want[ok], norm_err(d))
    assert torch.isnan(y[3]).all() and torch.isnan(rows.scale[:, 3]).all()
    assert torch.isnan(y[2, 5]) and (y[2, :5] == 0).all() and torch.isnan(rows.scale[0, 2])


GEMMS = [(1, 16, 1), (1, 128, 16), (1, 2560, 2560), (2, 112, 3), (3, 144, 17), (1, 4096, 515), (15, 992, 100), (16, 2752, 131),
         (17, 256, 129), (31, 2752, 260), (32, 1040, 64), (33, 272, 130), (48, 512, 96), (63, 128, 1), (64, 4112, 257), (65, 144, 5),
         (77, 2752, 515), (96, 1040, 128), (127, 256, 129), (128, 2048, 256), (129, 272, 385), (200, 2560, 640), (255, 112, 300),
         (257, 384, 513), (384, 1040, 130), (512, 640, 1028), (1030, 272, 272)]


def gemm_case(seed, m, k, n):
    x8, sx = rows_of(rand(seed, m, k, chan=True))
    w8, sw = weight_of(rand(seed + 1, n, k) * (1 + 3 * torch.rand(n, 1).to(DEV)))
    return x8, sx, w8, sw


@pytest.mark.parametrize("m,k,n", GEMMS)
@pytest.mark.parametrize("dtype", [F32, F16])
def test_gemm(gpu, m, k, n, dtype):
    x8, sx, w8, sw = gemm_case(m + k + n, m, k, n)
    buf = torch.full((m * n + 64,), 7.0, dtype=dtype, device=DEV)
    y = buf[:m * n].view(m, n)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    check_product(y, x8, sx, w8, sw)
    assert (buf[m * n:] == 7.0).all()
    again = torch.empty_like(y)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), again)
    assert torch.equal(y, again)


def tile_cases():
    """(tile, slices, m, k, n, dtype) of every tile that is built for the type."""
    sizes = [(33, 16, 1), (64, 400, 65), (65, 128, 3), (100, 1424, 260), (128, 144, 128), (255, 272, 257), (300, 528, 1000), (513, 2064, 129),
             (1600, 384, 300), (700, 256, 1300), (2300, 400, 2568)]
    for m, k, n in sizes:
        for dtype in (F32, F16):
            for tile in (1, 2, 3, 4, 6) if dtype is F32 or m <= 64 else (1, 2, 3, 4, 5, 7):
                if tile != 7:
                    yield from ((tile, s, m, k, n, dtype) for s in (1, 2, 8))
                elif k > B:  # (the 256 x 256 kernel: two blocks of K at least, no slices)
                    yield tile, 1, m, k, n, dtype


@pytest.mark.parametrize("tile,splits,m,k,n,dtype", tile_cases())
def test_gemm_tiles(gpu, tune, tile, splits, m, k, n, dtype):
    """Every tile, one block of K to many in each slice, at the tiles' edges."""
    tune(FP8_TILE=tile, FP8_SPLITS=splits)
    x8, sx, w8, sw = gemm_case(m + k + n, m, k, n)
    buf = torch.full((m * n + 64,), 7.0, dtype=dtype, device=DEV)
    y = buf[:m * n].view(m, n)
    launches()
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    ran = launches()
    assert ran == ["fp8_wide_kernel" if tile == 7 else "fp8_ring_kernel"] + ["fp8_reduce_kernel"] * (splits > 1 and k > B)
    check_product(y, x8, sx, w8, sw)
    assert (buf[m * n:] == 7.0).all()


@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 32, 33, 48, 49, 64])
@pytest.mark.parametrize("k,n", [(16, 5), (1168, 140), (2560, 1300), (400, 5400), (272, 9000), (144, 11008), (272, 13830), (144, 19456), (16, 28700)])
def test_few_tokens_shapes(gpu, tune, m, k, n):
    """The few tokens' kernel at widths of each of its shapes (16 to 64 columns
    a workgroup: N over its columns' blocks, ends and scales)."""
    tune(FP8_TILE=0)
    x8, sx, w8, sw = gemm_case(m + k + n, m, k, n)
    buf = torch.full((m * n + 64,), 7.0, device=DEV)
    y = buf[:m * n].view(m, n)
    launches()
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    assert launches() == ["fp8_mv_kernel"]
    check_product(y, x8, sx, w8, sw)
    assert (buf[m * n:] == 7.0).all()


@pytest.mark.parametrize("m,k,n", [(3, 131200, 20), (12, 66048, 33), (20, 66048, 40), (40, 66048, 17), (64, 33280, 24), (5, 33280, 8720),
                                   (60, 33280, 8200), (300, 33280, 130)])
def test_gemm_of_many_blocks(gpu, m, k, n):
    """More blocks of K than a wave, or a slice, holds scales of at once."""
    x8, sx = rows_of(rand(1, m, k))
    w8 = rand(2, n, k, dtype=F16).to(F8)
    sw = torch.rand(blocks(n), blocks(k), device=DEV) + 0.5
    y = torch.empty(m, n, device=DEV)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    n0 = (n - 1) // B * B
    check_product(y[:, n0:], x8, sx, w8[n0:], sw[n0 // B:])
    check_product(y[:, :20], x8, sx, w8[:20], sw[:1])


def test_gemm_without_room_for_slices(gpu):
    """Slices whose partial sums do not fit the workspace are not taken (the
    largest K and few tiles, 64 MiB)."""
    m, k, n = 1200, 11008, 3500  # (4 slices: 67 MB, 8: 134)
    x8, sx, w8, sw = gemm_case(3, m, k, n)
    y = torch.empty(m, n, dtype=F16, device=DEV)
    with gpu.tuning(FP8_TILE=4, FP8_SPLITS=8):
        sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    for at in (slice(0, 20), slice(m - 20, m)):
        check_product(y[at], x8[at], sx[:, at], w8, sw, many=True)


@pytest.mark.parametrize("m", [3, 40, 200])
def test_gemm_every_place(gpu, m):
    """One-hot rows return the weight's columns exactly: every k and n has its
    place, and every scale its block."""
    k, n = 400, 300
    w8, sw = weight_of(rand(5, n, k))
    w = w8.double().cpu() * sw.double().cpu().repeat_interleave(B, 0)[:n].repeat_interleave(B, 1)[:, :k]
    for k0 in range(0, k, m):
        cols = [(k0 + i) % k for i in range(m)]
        x = torch.zeros(m, k)
        x[torch.arange(m), cols] = 2.0 ** (torch.arange(m) % 5 - 2).float()
        y = torch.empty(m, n, device=DEV)
        sx = 2.0 ** (torch.arange(blocks(k))[:, None] - torch.arange(m) % 3).float()
        sta.fp8_gemm(gpu, sta.Fp8Rows.of(x.to(F8).to(DEV), sx.to(DEV)), sta.Fp8Weight.of(w8, sw), y)
        f = torch.stack([sx[c // B, i] * x[i, c] for i, c in enumerate(cols)]).double()
        assert torch.equal(y.cpu().double(), (w[:, cols].t() * f[:, None]).float().double())


@pytest.mark.parametrize("m", [1, 13, 64, 130])
def test_gemm_not_finite(gpu, m):
    """NaN rows, scales and weights reach their own row and column alone, also
    from rows and columns past a tile's end."""
    k, n = 272, 150
    x8, sx, w8, sw = gemm_case(11, m, k, n)
    w8.view(torch.uint8)[7, 270] = 0x7F  # NaN in the last block, which ends early
    w8.view(torch.uint8)[8, :8] = 0xFF
    if m > 4:
        x8.view(torch.uint8)[2, 265] = 0x7F
        sx[1, 3] = math.nan
        sx[0, 4] = math.inf
    y = torch.empty(m, n, device=DEV)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), y)
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[:, 7:9] = True
    if m > 4:
        bad[2:4] = True
        assert not torch.isfinite(y[4]).any()
        bad[4] = True
        assert torch.isnan(y[2:4]).all()
    y = y.cpu()
    assert torch.isnan(y[:, 7:9][~bad[:, :2] | True][0]).all() and not torch.isfinite(y[:, 7:9]).any()
    keep_r, keep_n = [i for i in range(m) if m <= 4 or i not in (2, 3, 4)], [i for i in range(n) if i not in (7, 8)]
    blk = [0 if i < B else 1 for i in keep_n]
    want_w = w8.cpu().view(torch.uint8)[keep_n].view(F8)
    xs, ss = x8.cpu().view(torch.uint8)[keep_r].view(F8), sx.cpu()[:, keep_r]
    full = torch.zeros(len(keep_r), len(keep_n), dtype=torch.float64)
    mag = full.clone()
    for b in range(blocks(k)):
        at = slice(b * B, b * B + B)
        f = ss[b].double()[:, None] * sw.cpu()[blk, b].double()
        full += xs[:, at].double() @ want_w[:, at].double().t() * f
        mag += xs[:, at].double().abs() @ want_w[:, at].double().abs().t() * f
    got = y[keep_r][:, keep_n].double()
    assert ((got - full).abs() <= (2 * B + 3 * blocks(k)) * U * mag).all()


@pytest.mark.parametrize("m", [1, 16, 50, 300])
def test_gemm_rows_of_wider_scales(gpu, m):
    """A part of a batch's rows, by slices."""
    k, n, most = 400, 144, m + 9
    x8, sx, w8, sw = gemm_case(21, most, k, n)
    all_rows, w = sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw)
    part = all_rows[5:5 + m]
    y = torch.empty(m, n, device=DEV)
    sta.fp8_gemm(gpu, part, w, y)
    check_product(y, x8[5:5 + m], sx[:, 5:5 + m], w8, sw)
    src = rand(9, m, k)
    sta.fp8_quant(gpu, src, part)
    check_rows(part.data, part.scale, src.double().cpu(), 0.0)
    for at in (slice(0, 5), slice(5 + m, most)):
        assert torch.equal(all_rows.data[at].view(torch.uint8), x8[at].view(torch.uint8)) and torch.equal(all_rows.scale[:, at], sx[:, at])


def test_norm_product_chain(gpu):
    """Norm, product, silu and product as an MLP runs them, against 64 bits
    from what was quantised at each step; a captured graph and another stream
    give the same bits, replay after replay."""
    for m in (1, 20, 150):
        d, inter = 512, 656
        w = rand(1, d) * 0.1 + 1
        wg, wd = weight_of(rand(2, 2 * inter, d) / math.sqrt(d)), weight_of(rand(3, d, inter) / math.sqrt(inter))
        gate_up, down = sta.Fp8Weight.of(*wg), sta.Fp8Weight.of(*wd)
        r, x = rand(4, m, d), rand(5, m, d)
        ro, gu, out = torch.empty(m, d, device=DEV), torch.empty(m, 2 * inter, device=DEV), torch.empty(m, d, device=DEV)
        a, h = sta.Fp8Rows(gpu, m, d), sta.Fp8Rows(gpu, m, inter)

        def mlp():
            sta.add_rmsnorm(gpu, r, w, x, rows=a, residual_out=ro)
            sta.fp8_gemm(gpu, a, gate_up, gu)
            sta.fp8_quant(gpu, gu[:, :inter], h, gu[:, inter:])
            sta.fp8_gemm(gpu, h, down, out)

        mlp()
        torch.cuda.synchronize()
        s = r.double().cpu() + x.double().cpu()
        check_rows(a.data, a.scale, s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * w.double().cpu(), norm_err(d))
        check_product(gu, a.data, a.scale, *wg)
        g, u = gu.double().cpu()[:, :inter], gu.double().cpu()[:, inter:]
        check_rows(h.data, h.scale, silu64(g) * u, silu_err(g))
        check_product(out, h.data, h.scale, *wd)
        want = out.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            out.zero_()
            mlp()
            side.synchronize()
            assert torch.equal(out, want)
            with torch.cuda.graph(graph, stream=side):
                mlp()
        torch.cuda.current_stream().wait_stream(side)
        for i in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            x.mul_(1.0 + 0.5 * (i == 1))  # (new inputs for the last replay)
            if i == 1:
                mlp()
                torch.cuda.synchronize()
                want = out.clone()


def test_graphs_share_the_workspace(gpu):
    """Two captured products in slices of K, whose partial sums meet in the
    context's workspace: replayed in turn, with eager products between them."""
    calls = []
    for seed, (m, k, n, dtype) in enumerate([(130, 2064, 264, F16), (77, 1424, 300, F32), (200, 2064, 130, F16)]):
        case = gemm_case(seed, m, k, n)
        y = torch.empty(m, n, dtype=dtype, device=DEV)
        calls.append((sta.Fp8Rows.of(*case[:2]), sta.Fp8Weight.of(*case[2:]), y))
    with gpu.tuning(FP8_TILE=4, FP8_SPLITS=4):
        for c in calls:
            sta.fp8_gemm(gpu, *c)
        torch.cuda.synchronize()
        want = [y.clone() for _, _, y in calls]
        for (x, w, y), v in zip(calls, want):
            check_product(v, x.data, x.scale, w.w, w.scale, many=v.dtype is F16)
        graphs = []
        for c in calls[:2]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                sta.fp8_gemm(gpu, *c)
        for turn in range(3):
            for _, _, y in calls:
                y.zero_()
            graphs[turn % 2].replay()
            sta.fp8_gemm(gpu, *calls[2])
            graphs[1 - turn % 2].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(y, v) for (_, _, y), v in zip(calls, want))


def test_two_contexts_at_once(gpu):
    """Contexts of their own on streams of their own, products in slices and
    norms in flight on both: each keeps its workspace."""
    other, out = sta.GpuContext(0), []
    for ctx, seed in ((gpu, 1), (other, 2)):
        m, k, n = 100, 2064, 520
        x8, sx, w8, sw = gemm_case(seed, m, k, n)
        r, w = rand(seed, m, k), rand(seed + 5, k)
        out.append((ctx, torch.cuda.Stream(), sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(w8, sw), torch.empty(m, n, dtype=F16, device=DEV), r, w,
                    sta.Fp8Rows(ctx, m, k)))
    torch.cuda.synchronize()
    with gpu.tuning(FP8_TILE=4, FP8_SPLITS=4), other.tuning(FP8_TILE=4, FP8_SPLITS=4):
        for _ in range(10):
            for ctx, stream, x, w, y, r, gain, rows in out:
                with torch.cuda.stream(stream):
                    sta.fp8_gemm(ctx, x, w, y)
                    sta.add_rmsnorm(ctx, r, gain, rows=rows)
        torch.cuda.synchronize()
    for _, _, x, w, y, r, gain, rows in out:
        check_product(y, x.data, x.scale, w.w, w.scale)
        s = r.double().cpu()
        check_rows(rows.data, rows.scale, s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * gain.double().cpu(), norm_err(r.shape[1]))


def test_gemm_past_32_bits(gpu):
    """A weight and rows of more than 2^32 bytes: the last columns and rows."""
    k, n = 32768, 135000
    row = torch.randint(0, 0x7F, (64, k), dtype=torch.uint8, device=DEV) | 0x80 * (torch.rand(64, k, device=DEV) < 0.5).to(torch.uint8)
    big = row.repeat(n // 64 + 1, 1)[:n].view(F8)
    sb = torch.rand(blocks(n), blocks(k), device=DEV) + 0.5
    x8, sx = rows_of(rand(1, 3, k))
    y = torch.empty(3, n, device=DEV)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(x8, sx), sta.Fp8Weight.of(big, sb), y)
    n0 = blocks(n) * B - 2 * B
    check_product(y[:, n0:], x8, sx, big[n0:], sb[n0 // B:])
    check_product(y[:, :100], x8, sx, big[:100], sb[:1])
    w8, sw = weight_of(rand(2, 20, k))
    sx = torch.rand(blocks(k), n, device=DEV)
    y = torch.empty(n, 20, dtype=F16, device=DEV)
    sta.fp8_gemm(gpu, sta.Fp8Rows.of(big, sx * 2.0**-10), sta.Fp8Weight.of(w8, sw), y)
    for at in (slice(0, 40), slice(n - 40, n)):
        check_product(y[at], big[at], sx[:, at] * 2.0**-10, w8, sw, many=True)
    del big, y
    x = rand(3, 50, k, dtype=F16).repeat(n // 50, 1)
    rows = sta.Fp8Rows(gpu, x.shape[0], k)
    sta.fp8_quant(gpu, x, rows)
    check_rows(rows.data[-50:], rows.scale[:, -50:], x[-50:].double().cpu(), 0.0)
    r = torch.empty(2, dtype=F16, device=DEV)
    sta.add_rmsnorm(gpu, x, torch.ones(k, device=DEV), rows=rows)
    s = x[-50:].double().cpu()
    check_rows(rows.data[-50:], rows.scale[:, -50:], s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6), norm_err(k))


def test_linear_takes_the_weight(gpu):
    """sta.linear quantises float rows and calls the product."""
    for m, dtype in ((1, F32), (70, F16)):
        x = rand(m, m, 272, dtype=dtype)
        w8, sw = weight_of(rand(8, 150, 272))
        y, rows = torch.empty(m, 150, device=DEV), sta.Fp8Rows(gpu, m, 272)
        sta.linear(gpu, x, sta.Fp8Weight.of(w8, sw), y)
        sta.fp8_quant(gpu, x, rows)
        check_product(y, rows.data, rows.scale, w8, sw)


def test_scales_helper_agrees(gpu):
    """The 64-bit scales are those of the tests' torch form."""
    y = rand(1, 4, 300)
    assert torch.allclose(scales(y.double().cpu()), rows_of(y)[1].double().cpu(), rtol=2 * U)
