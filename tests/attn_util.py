"""Plain 64-bit forms of the cache and attention operators, and the cache
layout written out from its definition (include/shady_hip.h), on the CPU."""
import math

import torch


_V_HALF = torch.tensor([0, 0, 0, 0, 1, 1, 1, 1] * 2)
_V_PLACE = torch.tensor([0, 1, 2, 3, 0, 1, 2, 3, 4, 5, 6, 7, 4, 5, 6, 7])


def indices(slots, heads, page, hd):
    """Flat elements of [T, heads, hd] in k and v, and of [T, heads] in the scales."""
    s = slots.long()[:, None, None]
    h, d = torch.arange(heads)[None, :, None], torch.arange(hd)[None, None, :]
    p, at = s // page, s % page
    tile = (p * heads + h) * (page // 16) + at // 16
    t = at % 16
    k = (tile * (hd // 8) + d // 8) * 128 + t * 8 + d % 8
    v = ((tile * 2 + _V_HALF[t]) * hd + d) * 8 + _V_PLACE[t]
    return k, v, ((p * heads + h) * page + at)[..., 0]


def shapes(pages, heads, page, hd):
    return (pages, heads, page // 16, hd // 8, 16, 8), (pages, heads, page // 16, 2, hd, 8), (pages, heads, page)


def norm_rope(x, w, eps, plus, cos, sin, pos, pairs):
    """x [T, heads, hd] float64."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() + plus)
    if cos is None:
        return x
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    r = 2 * c.shape[-1]
    y = x.clone()
    j = torch.arange(r // 2)
    a, b = (2 * j, 2 * j + 1) if pairs else (j, j + r // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def attention(q, k_of, v_of, spans, scale, cap=0.0, window=0, slopes=None, gate=None, visible=None):
    """q [T, nh, hd]; spans: (first row, rows, kv_len) of each sequence;
    k_of(b), v_of(b): [kv_len, nkv, hd] float64. Rows outside spans: NaN.
    visible(b): bool [kv_len], keys that may be seen at all."""
    T, nh, hd = q.shape
    out = torch.full((T, nh, hd), math.nan, dtype=torch.float64)
    for b, (r0, n, kv) in enumerate(spans):
        if n == 0:
            continue
        out[r0:r0 + n] = 0.0
        if kv == 0:
            continue
        k, v = k_of(b), v_of(b)
        g = nh // k.shape[1]
        j, p = torch.arange(kv)[None], (torch.arange(n) + kv - n)[:, None]
        see = j <= p
        if window:
            see &= j > p - window
        if visible is not None:
            see &= visible(b)[None]
        for h in range(nh):
            s = q[r0:r0 + n, h].double() @ k[:, h // g].T * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s + slopes[h].double() * (j - p)
            s = torch.where(see, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            w = torch.where(see, torch.exp(s - torch.where(m > -math.inf, m, 0.0)), 0.0)
            tot = w.sum(-1, keepdim=True)
            vv = torch.where(see.any(0)[:, None], v[:, h // g], 0.0)
            out[r0:r0 + n, h] = torch.where(tot > 0, w @ vv / torch.where(tot > 0, tot, 1.0), 0.0)
    if gate is not None:
        out = out / (1.0 + torch.exp(-gate.double()))
    return out


def rel(x, y):
    x, y = x.double().cpu(), y.double().cpu()
    n = torch.linalg.vector_norm(y)
    return (torch.linalg.vector_norm(x - y) / (n if n > 0 else 1.0)).item()
