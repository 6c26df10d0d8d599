"""Plain 64-bit forms of the 8-bit floating point operators, on the CPU, and
the bounds that their results are held to."""
import torch

B = 128
F8 = torch.float8_e4m3fn
U = 2.0**-24  # f32's half step


def blocks(n):
    return -(-n // B)


def block_max(y):
    """max |y| of each row's blocks of 128: [blocks, M]."""
    m, k = y.shape
    pad = torch.nn.functional.pad(y.abs(), (0, -k % B))
    return pad.view(m, -1, B).amax(-1).t()


def scales(y):
    return torch.clamp(block_max(y) / 448.0, min=2.0**-126)


def spread(scale, k):
    """[blocks, M] -> [M, k]."""
    return scale.t().repeat_interleave(B, 1)[:, :k]


def check_rows(data, scale, y, err):
    """Quantised rows against y [M, K] in 64 bits, of which they were made with
    a relative error of at most `err` (a number, or one for each element). A
    scale is max |y| times the rounded 1 / 448, rounded: two half steps on top
    of that error. A value v = y / scale is formed with a reciprocal (one step)
    and a product, then rounded to e4m3: half a step, 2^-4 of it, or 2^-10
    below the normal range."""
    data, scale = data.cpu().double(), scale.cpu().double()
    err = torch.as_tensor(err, dtype=torch.float64).expand_as(y)
    want = scales(y)
    most = block_max(err) + 2 * U  # (a block's largest value may be another within the error)
    assert ((scale - want).abs() <= want * most * (1 + 1e-6)).all(), ((scale - want).abs() / want).max()
    v = y / spread(scale, y.shape[1])
    d = err + 4 * U
    off = (data - v).abs() - (torch.clamp(v.abs() * (1 + d) * 2.0**-4, min=2.0**-10) + d * v.abs())
    assert (off <= 0).all(), off.max()


def product(x8, sx, w8, sw):
    """(y, sum of magnitudes) [M, N] in 64 bits."""
    m, k = x8.shape
    n = w8.shape[0]
    y, s = torch.zeros(m, n, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    x, w = x8.cpu().double(), w8.cpu().double()
    sx, sw = sx.cpu().double(), sw.cpu().double()
    for b in range(blocks(k)):
        at = slice(b * B, (b + 1) * B)
        f = sx[b][:, None] * sw[:, b].repeat_interleave(B)[:n]
        y += x[:, at] @ w[:, at].t() * f
        s += x[:, at].abs() @ w[:, at].abs().t() * f.abs()
    return y, s


def eights(x8, sx, w8, sw):
    """The sum over every eight k of the largest product's magnitude [M, N]."""
    m, k = x8.shape
    x, w = (x8.cpu().double() * spread(sx.cpu().double(), k)).abs(), w8.cpu().double().abs()
    w = w * sw.cpu().double().repeat_interleave(B, 0)[:w.shape[0]].repeat_interleave(B, 1)[:, :k]
    tot = torch.zeros(m, w.shape[0], dtype=torch.float64)
    for k0 in range(0, k, 8):
        tot += torch.stack([x[:, i, None] * w[None, :, i] for i in range(k0, k0 + 8)]).amax(0)
    return tot


def check_product(y, x8, sx, w8, sw, many=None):
    """Products are exact; a block's sum of 128 and the FMAs over the blocks
    round each once to f32 (at most a whole step in the matrix unit), the
    block's factor once, the output once. With f16 y and many tokens a product
    is cut below 2^-13 of the power of two of the largest of its eight k: seven
    products (the largest is not cut) by at most that each; many: whether these
    rows were part of such a call."""
    want, s = product(x8, sx, w8, sw)
    m, k = x8.shape
    bound = (2 * min(k, B) + 3 * blocks(k)) * U * s + 2.0**-149
    if y.dtype is torch.float16:
        bound = bound + want.abs() * 2.0**-11 + 2.0**-25
        if m > 64 if many is None else many:
            bound = bound + 7 * 2.0**-13 * eights(x8, sx, w8, sw) * (1 + 2.0**-10)
    off = (y.cpu().double() - want).abs() - bound
    assert (off <= 0).all(), (off.max(), (off > 0).sum())


def rows_of(y):
    """y [M, K] float32 on any device as e4m3 rows, by torch."""
    m, k = y.shape
    pad = torch.nn.functional.pad(y, (0, -k % B)).view(m, -1, B)
    s = (pad.abs().amax(-1) / 448.0).clamp(min=2.0**-126)
    q = (pad / s[..., None]).clamp(-448, 448).to(F8).view(m, -1)[:, :k].contiguous()
    return q, s.t().contiguous()


def weight_of(w):
    """w [N, K] float32 as an e4m3 weight, by torch."""
    n, k = w.shape
    pad = torch.nn.functional.pad(w, (0, -k % B, 0, -n % B)).view(blocks(n), B, blocks(k), B)
    s = (pad.abs().amax((1, 3)) / 448.0).clamp(min=2.0**-126)
    q = (pad / s[:, None, :, None]).clamp(-448, 448).to(F8).view(blocks(n) * B, -1)[:n, :k].contiguous()
    return q, s.contiguous()
