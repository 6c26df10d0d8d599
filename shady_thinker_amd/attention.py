"""What runs between the quantized linears of a decoder, and on its logits:
the paged key-value cache, the attention that reads it, and log probabilities.

The reference runs these per token in WGSL (src/model.rs:715-726, 540-592:
fused_split_qknorm_kvstore, gqa_attention_head, sigmoid_mul) and samples on
the CPU (:836-968). Here they are entry points of libshady_hip like the
linears, on torch device tensors and torch's current stream:

* `KvCache`: one layer's cache, float16 or int8 (a scale for each token and head);
* `qk_norm_rope_store`: q/k norms, rotation and cache write, one launch;
* `kv_read`: cached tokens back, dequantised;
* `paged_attention`: one token of each sequence, a few drafted ones, prompts;
* `token_logprobs`: log probability and rank of tokens, entropy, top tokens;
* `PagedAttention`: the first three as a DecoderStack's `attention` hook
  (captured in its graph) and for prompts beside `DecoderLinears.prefill`.

Activations are float32 (decode) or float16 (prefill), as the linears'.
Errors raise ValueError / TypeError (arguments) or ShadyHipError (a call).
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from ._lib import ST_F16, ST_F32, ST_FLAG_NORM_PLUS_ONE, ST_FLAG_ROPE_PAIRS, ST_I8, KvCacheStruct, call
from .gpu import ptr
from .model import _need

_F32, _F16, _I32, _I8 = torch.float32, torch.float16, torch.int32, torch.int8
_DT = {_F32: ST_F32, _F16: ST_F16}
_MAX_I32 = 2**31 - 1
TILE = 16  # tokens of a cache tile


def _act(t, name: str) -> int:
    d = _DT.get(t.dtype)
    if d is None:
        raise TypeError(f"{name}: dtype {t.dtype} (need float32 or float16)")
    return d


# As in model.py, what is right in the common case is found by few cheap
# tensor queries (a small call's kernel takes 4 us); a failing check goes on to
# a function that says what is wrong.
def _bad_rows(t, name: str, rows: int, width: int, dtype):
    raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, strides {t.stride()} (need {dtype} [{rows}, {width}], rows of adjacent "
                     "elements)")


def _rows(t, name: str, rows: int, width: int, dtype) -> int:
    """Elements from one row of `t` [rows, width] to the next; a row's
    elements are side by side (a part of a wider row will do)."""
    if t.dtype is not dtype or t.shape != (rows, width):
        _bad_rows(t, name, rows, width, dtype)
    if rows == 1 and t.is_contiguous():
        return width
    s = t.stride()
    if s[1] != 1:
        _bad_rows(t, name, rows, width, dtype)
    return s[0]


def _index(t, name: str, n: int) -> int:
    """Address of a contiguous int32 tensor of at least n."""
    if t.dtype is not _I32 or t.numel() < n or not t.is_contiguous():
        _need(t, name, (_I32,), n)
    return t.data_ptr()


def _f32(t, name: str, n: int) -> int | None:
    """Address of a contiguous float32 tensor of at least n (None: NULL)."""
    if t is None:
        return None
    if t.dtype is not _F32 or t.numel() < n or not t.is_contiguous():
        _need(t, name, (_F32,), n)
    return t.data_ptr()


class KvCache:
    """One layer's paged cache (st_kv_cache). Slot s is place s % page_size of
    page s // page_size; the layout is in tiles of 16 tokens, see the header.
    Token-major tensors go in and out through qk_norm_rope_store and kv_read."""

    def __init__(self, gpu, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=_F16):
        """Allocates the cache on the context's device; what it holds before
        the first write is undefined and never visible to paged_attention."""
        if dtype not in (_F16, _I8):
            raise TypeError(f"KvCache: dtype {dtype} (float16 or int8)")
        if page_size not in (16, 32, 64, 128, 256) or head_dim not in (64, 128, 256) or num_pages < 1 or n_kv_heads < 1:
            raise ValueError(f"KvCache: {num_pages} pages of {page_size} tokens (16, 32, 64, 128 or 256), {n_kv_heads} heads of "
                             f"{head_dim} dims (64, 128 or 256)")
        mk = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device=gpu.device)
        tiles = page_size // TILE
        k = mk(num_pages, n_kv_heads, tiles, head_dim // 8, TILE, 8)
        v = mk(num_pages, n_kv_heads, tiles, 2, head_dim, 8)
        ks = vs = None
        if dtype is _I8:
            ks, vs = (mk(num_pages, n_kv_heads, page_size, dt=_F32) for _ in range(2))
        self._take(k, v, page_size, ks, vs)

    @classmethod
    def of(cls, k, v, page_size: int, k_scale=None, v_scale=None) -> "KvCache":
        """A cache over the caller's tensors, in the layout of st_kv_cache."""
        self = cls.__new__(cls)
        self._take(k, v, page_size, k_scale, v_scale)
        return self

    def _take(self, k, v, page_size, k_scale, v_scale):
        if k.dtype not in (_F16, _I8) or v.dtype is not k.dtype:
            raise TypeError(f"KvCache: dtypes {k.dtype}, {v.dtype} (both float16 or both int8)")
        if k.dim() != 6 or k.shape[2] * TILE != page_size or k.shape[4:] != (TILE, 8):
            raise ValueError(f"KvCache: k {tuple(k.shape)} is not [pages, heads, {page_size} / 16, dim / 8, 16, 8]")
        pages, heads, tiles, d8 = k.shape[:4]
        if tuple(v.shape) != (pages, heads, tiles, 2, d8 * 8, 8):
            raise ValueError(f"KvCache: v {tuple(v.shape)} is not {(pages, heads, tiles, 2, d8 * 8, 8)}")
        if not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("KvCache: k and v must be contiguous")
        if k.dtype is _I8:
            for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                _need(t, name, (_F32,), pages * heads * page_size)
        else:
            k_scale = v_scale = None
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.dtype, self.num_pages, self.page_size, self.n_kv_heads, self.head_dim = k.dtype, pages, page_size, heads, d8 * 8
        self.kv_width = heads * d8 * 8  # a token's keys, or values
        self._struct = KvCacheStruct(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ST_I8 if k.dtype is _I8 else ST_F16, pages, page_size,
                                     heads, d8 * 8)
        self.handle = ctypes.addressof(self._struct)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def slots(self, table, positions):
        """Slots (int32) of `positions` [B] or [B, n] in the sequences whose
        pages are the rows of `table` [B, pages]; torch ops, capturable.
        Positions that the table has no page for, and places of a page outside
        the cache, get a slot outside the cache, which is not written."""
        return self._places(table, positions)[1].to(_I32)

    def _places(self, table, positions):
        """Whether the table has a page for each position; the slots, 64 bits."""
        p = positions.long()
        i = p // self.page_size
        held = i.clamp(0, table.shape[1] - 1)
        page = torch.gather(table, 1, held.view(table.shape[0], -1)).view(p.shape)
        ok = i == held
        slot = torch.add(p, page - i, alpha=self.page_size)  # (64 bits: no product comes round)
        return ok, torch.where(ok, slot, -1).clamp_(-1, _MAX_I32)


def qk_norm_rope_store(gpu, cache: KvCache, q, k, v, q_out, slots, positions=None, cos=None, sin=None, q_weight=None, k_weight=None,
                       eps: float = 1e-6, one_plus: bool = False, pairs: bool = False, gated: bool = False) -> None:
    """Norms (q_weight, k_weight [head_dim] f32; None: no norm) and rotation
    (cos, sin [n_pos, rot / 2] f32 at `positions`; None: no rotation) of the
    new tokens' queries and keys, and the write of keys and values to `slots`
    of the cache (fused_split_qknorm_kvstore, src/model.rs:715-726).

    q [T, heads * head_dim] (gated: twice as wide, each head's query followed
    by its gate), k and v [T, n_kv_heads * head_dim], of one dtype; they may be
    parts of one q|k|v row. q_out [T, heads * head_dim] float32 or float16.
    q and q_out None: keys and values only. one_plus: weights hold w - 1;
    pairs: dims (2j, 2j + 1) rotate together, not (j, j + rot / 2)."""
    hd, kw = cache.head_dim, cache.kv_width
    dtype = k.dtype
    dt = _act(k, "k")
    T = k.shape[0]
    ks, vs = _rows(k, "k", T, kw, dtype), _rows(v, "v", T, kw, dtype)
    heads = qs = qh = qd = rot = n_pos = 0
    qp = op = at = cp = sp = None
    if q is not None:
        if q_out is None:
            raise ValueError("q without q_out")
        qh = 2 * hd if gated else hd
        heads = q.shape[-1] // qh
        qs = _rows(q, "q", T, max(heads, 1) * qh, dtype)
        qd = _act(q_out, "q_out")
        if q_out.numel() < T * heads * hd or not q_out.is_contiguous():
            _need(q_out, "q_out", (_F32, _F16), T * heads * hd)
        qp, op = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    if cos is not None:
        if sin is None or positions is None:
            raise ValueError("cos needs sin and positions")
        if cos.dim() != 2:
            raise ValueError(f"cos {tuple(cos.shape)} (need [n_pos, rot / 2])")
        n_pos, rot = cos.shape
        cp, sp = _f32(cos, "cos", 1), _f32(sin, "sin", n_pos * rot)
        rot *= 2
        at = _index(positions, "positions", T)
    elif sin is not None:
        raise ValueError("sin needs cos")
    qw, kwt = _f32(q_weight, "q_weight", hd), _f32(k_weight, "k_weight", hd)
    slots_at = _index(slots, "slots", T)
    gpu.sync_stream()
    call("st_qk_norm_rope_store", gpu.handle, cache.handle, qp, k.data_ptr(), v.data_ptr(), dt, qs, ks, vs, qh, qw, kwt, eps, cp, sp, rot,
         n_pos, at, slots_at, op, qd, T, heads,
         (ST_FLAG_NORM_PLUS_ONE if one_plus else 0) | (ST_FLAG_ROPE_PAIRS if pairs else 0))


def kv_read(gpu, cache: KvCache, slots, k_out, v_out) -> None:
    """k_out, v_out [T, n_kv_heads, head_dim] (float32 or float16): the cached
    tokens of `slots` [T], dequantised; zeros for a slot outside the cache."""
    T = slots.numel()
    n = T * cache.kv_width
    dtype = k_out.dtype
    dt = _act(k_out, "k_out")
    if v_out.dtype is not dtype or k_out.numel() < n or v_out.numel() < n or not k_out.is_contiguous() or not v_out.is_contiguous():
        _need(k_out, "k_out", (dtype,), n)
        _need(v_out, "v_out", (dtype,), n)
    slots_at = _index(slots, "slots", T)
    gpu.sync_stream()
    call("st_kv_read", gpu.handle, cache.handle, slots_at, k_out.data_ptr(), v_out.data_ptr(), dt, T)


def paged_attention(gpu, cache: KvCache, q, out, table, kv_len, q_start=None, scale: float | None = None, cap: float = 0.0,
                    window: int = 0, slopes=None, gate=None, gated: bool = False) -> None:
    """out = softmax(scale q k^T) v of the new rows over the cache (times
    sigmoid(gate)); gqa_attention_head / gqa_reduce / sigmoid_mul of the
    reference (src/model.rs:540-592).

    q, out [T, heads * head_dim] contiguous, float32 or float16; rows
    q_start[b] .. q_start[b + 1] belong to sequence b (None: one row each),
    the newest of its kv_len[b] cached tokens; table [B, pages] holds each
    sequence's pages. scale None: 1 / sqrt(head_dim). cap > 0: scores capped
    by a tanh; window > 0: the last `window` keys only; slopes [heads] f32:
    slopes * (key - position) added. gate [T, heads * head_dim] (gated: the
    qkv rows' gated q, [T, heads * 2 * head_dim], each head's query followed
    by its gate), rows of adjacent elements."""
    hd = cache.head_dim
    if table.dim() != 2 or q.dim() != 2:
        raise ValueError(f"table {tuple(table.shape)}, q {tuple(q.shape)} (need [B, pages], [T, heads * {hd}])")
    B, pages = table.shape
    T, width = q.shape
    heads = width // hd
    if heads * hd != width or not q.is_contiguous():
        raise ValueError(f"q: shape {tuple(q.shape)} (need contiguous [T, heads * {hd}])")
    qd, od = _act(q, "q"), _act(out, "out")
    if out.numel() < T * width or not out.is_contiguous():
        _need(out, "out", (_F32, _F16), T * width)
    gp, gd, gs, gh = None, 0, 0, 0
    if gate is not None:
        gd = _act(gate, "gate")
        gh = 2 * hd if gated else hd
        gs = _rows(gate, "gate", T, heads * gh, gate.dtype)
        gp = gate.data_ptr()
        if gated:  # (from the first head's gate; the last head's ends the row)
            gp += hd * gate.element_size()
    table_at, len_at = _index(table, "table", B * pages), _index(kv_len, "kv_len", B)
    start_at = None if q_start is None else _index(q_start, "q_start", B + 1)
    slopes_at = _f32(slopes, "slopes", heads)
    gpu.sync_stream()
    call("st_paged_attention", gpu.handle, cache.handle, q.data_ptr(), qd, table_at, pages, len_at, start_at,
         hd ** -0.5 if scale is None else scale, cap, min(window, _MAX_I32), slopes_at, gp, gd, gs, gh, out.data_ptr(), od, T, B, heads)


def token_logprobs(gpu, logits, tokens=None, logprob=None, entropy=None, rank=None, top_ids=None, top_logprobs=None) -> None:
    """Of rows of logits [M, V] (float32 or float16, rows of adjacent
    elements): logprob [M] f32 and rank [M] int32 of `tokens` [M] int32,
    entropy [M] f32, the top tokens top_ids [M, n] int32 and their
    top_logprobs [M, n] f32 (n <= 32). Any of the outputs may be None."""
    if logits.dim() != 2:
        raise ValueError(f"logits: shape {tuple(logits.shape)} (need [M, V])")
    M, V = logits.shape
    dt = _act(logits, "logits")
    stride = _rows(logits, "logits", M, V, logits.dtype)
    if tokens is None and (logprob is not None or rank is not None):
        raise ValueError("logprob and rank need tokens")
    tokens_at = None if tokens is None else _index(tokens, "tokens", M)
    lp, ent = _f32(logprob, "logprob", M), _f32(entropy, "entropy", M)
    rank_at = None if rank is None else _index(rank, "rank", M)
    top, ids, tops = 0, None, None
    if top_ids is not None:
        if top_ids.dim() != 2 or top_ids.shape[0] != M:
            raise ValueError(f"top_ids: shape {tuple(top_ids.shape)} (need [{M}, n])")
        top = top_ids.shape[1]
        if top:
            ids, tops = _index(top_ids, "top_ids", M * top), _f32(top_logprobs, "top_logprobs", M * top)
    elif top_logprobs is not None:
        raise ValueError("top_logprobs needs top_ids")
    gpu.sync_stream()
    call("st_token_logprobs", gpu.handle, logits.data_ptr(), dt, stride, tokens_at, lp, ent, rank_at, ids, tops, M, V, top)


class PagedAttention:
    """The self-attention of a model's layers over paged caches: a
    DecoderStack's `attention` hook for one token of each of B sequences
    (captured in the stack's graph, with `advance` before it), and `prefill`
    for prompts beside DecoderLinears.prefill. Capturing is not a step: the
    lengths and the caches stay as they are (`warm_up`).

    caches: one KvCache per layer (None for layers of another kind). table
    [B, pages] int32, each sequence's pages, the caller's to fill before they
    are needed. norms: per layer (q_weight, k_weight) or None. The remaining
    options are those of qk_norm_rope_store and paged_attention."""

    def __init__(self, gpu, caches, n_heads: int, table, cos=None, sin=None, norms=None, eps: float = 1e-6, one_plus: bool = False,
                 pairs: bool = False, gated: bool = False, **attention):
        self.gpu, self.caches, self.n_heads, self.table = gpu, caches, n_heads, table
        c = next(c for c in caches if c is not None)
        if any(x is not None and (x.page_size, x.n_kv_heads, x.head_dim) != (c.page_size, c.n_kv_heads, c.head_dim) for x in caches):
            raise ValueError("PagedAttention: caches of different pages or heads")
        self.norms = norms or [None] * len(caches)
        self.store = dict(cos=cos, sin=sin, eps=eps, one_plus=one_plus, pairs=pairs, gated=gated)
        self.gated, self.options, self.cache = gated, attention, c
        B = table.shape[0]
        mk = lambda: torch.zeros(B, dtype=_I32, device=gpu.device)
        self.kv_len, self.positions = mk(), mk()
        self.slots, self._nowhere = mk().fill_(-1), mk().fill_(-1)
        self._stores = True
        self.q = torch.empty(B, n_heads * c.head_dim, device=gpu.device)
        self.widths = (n_heads * c.head_dim * (2 if gated else 1), c.n_kv_heads * c.head_dim)

    def advance(self) -> None:
        """Every sequence gets its next place (torch ops on device tensors, so
        a captured step can begin with it): positions = kv_len, then kv_len + 1.
        A sequence that fills its table stays as long as that: its new tokens
        are not stored, and its row attends to those that are."""
        self.positions.copy_(self.kv_len)
        ok, slots = self.cache._places(self.table, self.positions)
        self.slots.copy_(slots)
        self.kv_len += ok

    @contextlib.contextmanager
    def warm_up(self):
        """DecoderStack hook, around the eager step before a capture: it stores
        no token (its place may not be the sequence's yet), and the lengths
        are afterwards what they were."""
        kept, self._stores = self.kv_len.clone(), False
        try:
            yield
        finally:
            self._stores = True
            self.kv_len.copy_(kept)

    def _split(self, qkv):
        w, kw = self.widths
        return qkv[:, :w], qkv[:, w:w + kw], qkv[:, w + kw:w + 2 * kw]

    def _run(self, i, qkv, q_buf, out, slots, positions, table, kv_len, q_start) -> None:
        q, k, v = self._split(qkv)
        qw, kw = self.norms[i] or (None, None)
        qk_norm_rope_store(self.gpu, self.caches[i], q, k, v, q_buf, slots, positions if self.store["cos"] is not None else None,
                           q_weight=qw, k_weight=kw, **self.store)
        paged_attention(self.gpu, self.caches[i], q_buf, out, table, kv_len, q_start, gate=q if self.gated else None, gated=self.gated,
                        **self.options)

    def attention(self, i, b) -> None:
        """DecoderStack hook: b.qkv [B, q|k|v] -> b.attn [B, heads * head_dim]."""
        if self.caches[i] is not None:
            self._run(i, b.qkv, self.q, b.attn, self.slots if self._stores else self._nowhere, self.positions, self.table, self.kv_len, None)

    def prefill(self, i, qkv, out, q_start, positions, slots, kv_len, table=None) -> None:
        """Layer i's attention of prompts: qkv [T, q|k|v] (the output of the
        layer's input projection) -> out [T, heads * head_dim], rows q_start[b]
        .. of sequence b at `positions`, written to `slots`, kv_len [B] with
        these tokens."""
        q_buf = torch.empty(qkv.shape[0], self.n_heads * self.cache.head_dim, dtype=out.dtype, device=qkv.device)
        self._run(i, qkv, q_buf, out, slots, positions, self.table if table is None else table, kv_len, q_start)
