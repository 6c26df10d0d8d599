// Norm, rotation and cache write of new tokens, and the read back of cached
// ones (st_qk_norm_rope_store, st_kv_read). Replaces
// src/shaders/fused_split_qknorm_kvstore.wgsl:1-230.
//
// Both move every byte once; a workgroup takes one head of 16 tokens, a thread
// eight dims ("a piece") of one token. A head's norm and int8 scale are sums
// and maxima over its head_dim / 8 lanes, side by side in one wave; the
// rotation's other dims come from a lane of the same head. Keys are written
// and read in pieces as they are; values lie with eight tokens side by side,
// so a workgroup whose 16 tokens fill a tile turns them in LDS (whole 16-byte
// pieces, lines written by one workgroup); others go element by element.
// 2047 tokens of 32/8 heads of 128, f16: 13.6 us (3.7 TB/s; two heads a
// workgroup 13.8, four 15.4); one token 4.1 us, the launch (events around it; 3.2
// in a kernel trace). The read takes four
// heads a workgroup where there are many (16384 int8 tokens of 8 heads of 128:
// 22.4 us, 4.5 TB/s; with one 28.5).
#include "kvcache.hpp"

#include <algorithm>

namespace {

using namespace st::kv;

struct StoreArgs {
    Cache c;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    int q_head_stride, n_heads;
    const float *q_weight, *k_weight, *cos, *sin;
    float eps, weight_add;
    int rot, n_pos, pairs;
    const int32_t *positions, *slots;
    void *q_out;
    int T, shift;  // shift: groups of 16 tokens start where the first token's tile does
};

template <int P>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
    for (int d = 1; d < P; d *= 2) v += __shfl_xor(v, d);
    return v;
}
// (NaN where any is: an int8 head with a NaN in it reads back as NaN)
template <int P>
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
    for (int d = 1; d < P; d *= 2) {
        const float o = __shfl_xor(v, d);
        v = (v >= o || v != v) ? v : o;
    }
    return v;
}

template <bool F32>
__device__ __forceinline__ void load8(const void *p, int64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const f32x4 *s = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + at);
        const f32x4 a = s[0], b = s[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const half8 a = *reinterpret_cast<const half8 *>(static_cast<const _Float16 *>(p) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    }
}

__device__ __forceinline__ half8 to_half8(const float (&x)[8]) {
    half8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)x[i];
    return r;
}

template <bool F32>
__device__ __forceinline__ void store8(void *p, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        f32x4 *s = reinterpret_cast<f32x4 *>(static_cast<float *>(p) + at);
        s[0] = f32x4{x[0], x[1], x[2], x[3]};
        s[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *reinterpret_cast<half8 *>(static_cast<_Float16 *>(p) + at) = to_half8(x);
    }
}

// Eight values of one head as int8 with the head's scale max|x| / 127.
template <int P>
__device__ __forceinline__ u32x2 quantise(const float (&x)[8], float &scale) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = (m >= fabsf(x[i]) || m != m) ? m : fabsf(x[i]);
    scale = head_max<P>(m) / 127.0f;
    unsigned w[2] = {0, 0};
    if (scale > 0.0f) {  // (a zero head; NaN: its scale says it)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // (an infinity over an infinite scale: 127 of its sign)
            const float r = copysignf(fminf(fabsf(rintf(x[i] / scale)), 127.0f), x[i]);
            w[i / 4] |= ((unsigned)(int)r & 0xFFu) << (8 * (i % 4));
        }
    }
    return u32x2{w[0], w[1]};
}

// (a row of the turned tile: head_dim elements and 16 bytes, so that the
// rows of a wave's tokens start in different banks)
template <int HD, typename E>
constexpr int kTurnRow = HD + 16 / (int)sizeof(E);

// The tile a group of 16 tokens fills in order, or -1 (the whole workgroup
// agrees): tokens t0 .. t0 + 15 exist and their slots are one tile's places.
__device__ __forceinline__ int whole_tile(const Cache &c, const int32_t *slots, int t0, int tok, int T, int slot, bool stored) {
    const bool in = t0 >= 0 && t0 + kTile <= T;
    const int first = in ? slots[t0] : 0;
    const bool mine = in && stored && (first & (kTile - 1)) == 0 && slot == first + tok;
    return __syncthreads_and(mine) ? first >> 4 : -1;
}

template <int HD, bool XF32, bool QF32, bool I8>
__global__ __launch_bounds__(2 * HD) void store_kernel(StoreArgs a) {
    constexpr int P = HD / 8;
    using E = std::conditional_t<I8, signed char, _Float16>;
    using E8 = std::conditional_t<I8, u32x2, half8>;
    const int tid = threadIdx.x, piece = tid % P, tok = tid / P;
    const int unit = blockIdx.y;
    const int nq = a.n_heads, nk = a.c.heads;
    const int t0 = (int)blockIdx.x * kTile - (a.shift ? a.slots[0] & (kTile - 1) : 0);
    const int t = t0 + tok;
    const bool live = t >= 0 && t < a.T;
    const bool is_q = unit < nq, is_v = unit >= nq + nk;
    const int head = is_q ? unit : (unit - nq) % nk;
    const void *src = is_q ? a.q : is_v ? a.v : a.k;
    const int64_t at = live ? (is_q ? t * a.q_stride + (int64_t)head * a.q_head_stride
                                    : t * (is_v ? a.v_stride : a.k_stride) + (int64_t)head * HD) + piece * 8
                            : 0;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int slot = -1, pos = 0;
    if (live) {
        load8<XF32>(src, at, x);
        slot = a.slots[t];
        if (a.cos) pos = a.positions[t];
    }
    const bool placed = !a.cos || (pos >= 0 && pos < a.n_pos);
    if (!is_v) {
        const float *w = is_q ? a.q_weight : a.k_weight;
        if (w) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
            const float r = 1.0f / sqrtf(head_sum<P>(s) * (1.0f / HD) + a.eps);
            float wv[8];
            load8<true>(w, piece * 8, wv);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (wv[i] + a.weight_add);
        }
        if (a.cos) {
            const int half = a.rot / 16;  // pieces of half the rotated dims
            const int64_t row = (int64_t)(placed ? pos : 0) * (a.rot / 2);
            if (a.pairs) {
                if (piece < 2 * half) {
                    const f32x4 c = *reinterpret_cast<const f32x4 *>(a.cos + row + piece * 4);
                    const f32x4 s = *reinterpret_cast<const f32x4 *>(a.sin + row + piece * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float u = x[2 * i], v = x[2 * i + 1];
                        x[2 * i] = u * c[i] - v * s[i];
                        x[2 * i + 1] = v * c[i] + u * s[i];
                    }
                }
            } else {
                const bool low = piece < half;
                const int other = low ? piece + half : piece - half;  // (past the rotated dims: not used)
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __shfl(x[i], (tid & 63) / P * P + (other < P ? other : piece));
                if (piece < 2 * half) {
                    float c[8], s[8];
                    load8<true>(a.cos, row + (low ? piece : other) * 8, c);
                    load8<true>(a.sin, row + (low ? piece : other) * 8, s);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + (low ? -o[i] : o[i]) * s[i];
                }
            }
        }
    }
    if (is_q) {
        if (!live) return;
        if (!placed) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
        }
        store8<QF32>(a.q_out, ((int64_t)t * nq + head) * HD + piece * 8, x);
        return;
    }
    const int page = slot >> a.c.page_shift, place = slot & ((1 << a.c.page_shift) - 1);
    const bool stored = live && placed && slot >= 0 && page < a.c.num_pages;
    E8 e;
    if constexpr (I8) {
        float scale;
        e = quantise<P>(x, scale);
        if (stored && piece == 0) (is_v ? a.c.v_scale : a.c.k_scale)[a.c.scale(page, head, place)] = scale;
    } else {
        e = to_half8(x);
    }
    const int64_t tile = stored ? a.c.tile(page, head, place >> 4) : 0;
    const int in_tile = place & (kTile - 1);
    if (!is_v) {
        if (stored) *reinterpret_cast<E8 *>(static_cast<E *>(a.c.k) + tile * (kTile * HD) + piece * 128 + in_tile * 8) = e;
        return;
    }
    E *const v = static_cast<E *>(a.c.v);
    if (whole_tile(a.c, a.slots, t0, tok, a.T, slot, stored) >= 0) {
        constexpr int kRow = kTurnRow<HD, E>;
        __shared__ __align__(16) E turn[kTile * kRow];
        *reinterpret_cast<E8 *>(&turn[tok * kRow + piece * 8]) = e;
        __syncthreads();
        const int half = tid / HD, d = tid % HD;
        E out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = turn[v_token(half, j) * kRow + d];
        E8 o;
        __builtin_memcpy(&o, out, sizeof o);
        *reinterpret_cast<E8 *>(v + tile * (kTile * HD) + (half * HD + d) * 8) = o;  // (tile: the same for all 16 tokens)
        return;
    }
    if (!stored) return;
    E out[8];
    __builtin_memcpy(out, &e, sizeof e);
    E *const to = v + tile * (kTile * HD) + (v_half(in_tile) * HD + piece * 8) * 8 + v_place(in_tile);
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i * 8] = out[i];
}

struct ReadArgs {
    Cache c;
    const int32_t *slots;
    void *k_out, *v_out;
    int T, shift;
};

// U heads a workgroup, their loads in flight together.
template <int HD, bool OF32, bool I8, int U>
__global__ __launch_bounds__(2 * HD) void read_kernel(ReadArgs a) {
    constexpr int P = HD / 8;
    using E = std::conditional_t<I8, signed char, _Float16>;
    using E8 = std::conditional_t<I8, u32x2, half8>;
    const int tid = threadIdx.x, piece = tid % P, tok = tid / P, head0 = blockIdx.y * U, heads = a.c.heads;
    const bool is_v = blockIdx.z != 0;
    const int t0 = (int)blockIdx.x * kTile - (a.shift ? a.slots[0] & (kTile - 1) : 0);
    const int t = t0 + tok;
    const bool live = t >= 0 && t < a.T;
    const int slot = live ? a.slots[t] : -1;
    const int page = slot >> a.c.page_shift, place = slot & ((1 << a.c.page_shift) - 1);
    const bool held = slot >= 0 && page < a.c.num_pages;
    const int64_t tile = held ? a.c.tile(page, head0, place >> 4) * (kTile * HD) : 0;
    const int64_t next = held ? (int64_t)(kTile * HD) << a.c.tiles_shift() : 0;
    const int in_tile = place & (kTile - 1);
    auto of = [&](int u) { return head0 + u < heads ? u : 0; };  // (past the last head: the first again, not written)
    float scale[U];
    E8 e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        scale[u] = 1.0f;
        e[u] = E8{};
        if constexpr (I8) {
            if (held) scale[u] = (is_v ? a.c.v_scale : a.c.k_scale)[a.c.scale(page, head0 + of(u), place)];
        }
    }
    if (!is_v) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (held) e[u] = *reinterpret_cast<const E8 *>(static_cast<const E *>(a.c.k) + tile + of(u) * next + piece * 128 + in_tile * 8);
    } else {
        const E *const v = static_cast<const E *>(a.c.v) + tile;
        if (whole_tile(a.c, a.slots, t0, tok, a.T, slot, held) >= 0) {
            constexpr int kRow = kTurnRow<HD, E>;
            __shared__ __align__(16) E turn[U][kTile * kRow];
            const int half = tid / HD, d = tid % HD;
            E8 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) o[u] = *reinterpret_cast<const E8 *>(v + of(u) * next + (half * HD + d) * 8);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                E in[8];
                __builtin_memcpy(in, &o[u], sizeof o[u]);
#pragma unroll
                for (int j = 0; j < 8; ++j) turn[u][v_token(half, j) * kRow + d] = in[j];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) e[u] = *reinterpret_cast<const E8 *>(&turn[u][tok * kRow + piece * 8]);
        } else if (held) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const E *const from = v + of(u) * next + (v_half(in_tile) * HD + piece * 8) * 8 + v_place(in_tile);
                E in[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) in[i] = from[i * 8];
                __builtin_memcpy(&e[u], in, sizeof e[u]);
            }
        }
    }
    if (!live) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (head0 + u >= heads) return;
        float x[8];
        if constexpr (I8) {
            const half8 h = i8_to_half8(e[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = held ? (float)h[i] * scale[u] : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)e[u][i];
        }
        store8<OF32>(is_v ? a.v_out : a.k_out, ((int64_t)t * heads + head0 + u) * HD + piece * 8, x);
    }
}

// Groups of 16 tokens; from a group's length of tokens on they start with the
// first token's tile (a prompt that goes on within a page then fills tiles).
bool shifted(int T) { return T >= kTile; }
unsigned groups(int T) { return (unsigned)((T + kTile - 1) / kTile + (shifted(T) ? 1 : 0)); }

template <int HD, bool XF32, bool QF32, bool I8>
void launch_store(st_context *ctx, const StoreArgs &a) {
    // (one head a workgroup at every length: 2047 tokens 13.6 us with one,
    // 13.8 with two, 15.4 with four)
    const dim3 grid(groups(a.T), (unsigned)(a.n_heads + 2 * a.c.heads));
    st::launch(ctx, store_kernel<HD, XF32, QF32, I8>, grid, dim3(2 * HD), 0, a);
}

template <int HD, bool OF32, bool I8>
void launch_read(st_context *ctx, const ReadArgs &a) {
    // Four heads a workgroup where that still leaves every CU some workgroups
    // (16384 int8 tokens of 8 heads: 28.5 us with one, 23.1 with four).
    constexpr int kHeads = 4;
    const int few = (a.c.heads + kHeads - 1) / kHeads;
    const bool several = (int64_t)groups(a.T) * 2 * few >= 4 * (int64_t)ctx->num_cus;
    const dim3 grid(groups(a.T), (unsigned)(several ? few : a.c.heads), 2);
    if (!several)
        st::launch(ctx, read_kernel<HD, OF32, I8, 1>, grid, dim3(2 * HD), 0, a);
    else
        st::launch(ctx, read_kernel<HD, OF32, I8, kHeads>, grid, dim3(2 * HD), 0, a);
}

template <int HD>
void store_by_type(st_context *ctx, const StoreArgs &a, bool xf32, bool qf32, bool i8) {
    if (xf32 && qf32)
        i8 ? launch_store<HD, true, true, true>(ctx, a) : launch_store<HD, true, true, false>(ctx, a);
    else if (xf32)
        i8 ? launch_store<HD, true, false, true>(ctx, a) : launch_store<HD, true, false, false>(ctx, a);
    else if (qf32)
        i8 ? launch_store<HD, false, true, true>(ctx, a) : launch_store<HD, false, true, false>(ctx, a);
    else
        i8 ? launch_store<HD, false, false, true>(ctx, a) : launch_store<HD, false, false, false>(ctx, a);
}

template <int HD>
void read_by_type(st_context *ctx, const ReadArgs &a, bool f32, bool i8) {
    if (f32)
        i8 ? launch_read<HD, true, true>(ctx, a) : launch_read<HD, true, false>(ctx, a);
    else
        i8 ? launch_read<HD, false, true>(ctx, a) : launch_read<HD, false, false>(ctx, a);
}

bool act_dtype(int d) { return d == ST_F32 || d == ST_F16; }
bool whole16(int64_t elements, int dtype) { return elements % (dtype == ST_F32 ? 4 : 8) == 0; }

}  // namespace

extern "C" int st_qk_norm_rope_store(st_context *ctx, const st_kv_cache *cache, const void *q, const void *k, const void *v,
                                     int x_dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                     int q_head_stride, const float *q_weight, const float *k_weight, float eps,
                                     const float *cos, const float *sin, int rot, int n_pos, const int32_t *positions,
                                     const int32_t *slots, void *q_out, int q_dtype, int T, int n_heads, uint32_t flags) {
    const char *const fn = "st_qk_norm_rope_store";
    StoreArgs a{};
    if (!ctx || !k || !v || !slots) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (int rc = check_cache(fn, cache, &a.c)) return rc;
    if ((q == nullptr) != (q_out == nullptr)) return st::fail(ST_ERR_INVALID, "%s: q without q_out, or q_out without q", fn);
    if ((cos == nullptr) != (sin == nullptr)) return st::fail(ST_ERR_INVALID, "%s: cos without sin, or sin without cos", fn);
    if (cos && !positions) return st::fail(ST_ERR_INVALID, "%s: a rotation needs positions", fn);
    if (!act_dtype(x_dtype) || (q && !act_dtype(q_dtype)))
        return st::fail(ST_ERR_INVALID, "%s: x_dtype %d, q_dtype %d (f32 or f16)", fn, x_dtype, q_dtype);
    if (flags & ~(ST_FLAG_NORM_PLUS_ONE | ST_FLAG_ROPE_PAIRS)) return st::fail(ST_ERR_INVALID, "%s: flags 0x%x", fn, flags);
    const int hd = cache->head_dim;
    if (T < 1) return st::fail(ST_ERR_SHAPE, "%s: T=%d", fn, T);
    if (q && (n_heads < 1 || n_heads > 32768)) return st::fail(ST_ERR_SHAPE, "%s: n_heads=%d", fn, n_heads);
    if (cos && (rot < 16 || rot % 16 || rot > hd || n_pos < 1))
        return st::fail(ST_ERR_SHAPE, "%s: rot=%d (a multiple of 16, at most the head dim %d), n_pos=%d", fn, rot, hd, n_pos);
    const int64_t kv = (int64_t)a.c.heads * hd;
    if (k_stride < kv || v_stride < kv) return st::fail(ST_ERR_SHAPE, "%s: a token's keys and values overlap the next one's", fn);
    if (q && (q_head_stride < hd || q_stride < (int64_t)(n_heads - 1) * q_head_stride + hd))
        return st::fail(ST_ERR_SHAPE, "%s: a head's or token's queries overlap the next one's", fn);
    if (!whole16(k_stride, x_dtype) || !whole16(v_stride, x_dtype) ||
        (q && (!whole16(q_stride, x_dtype) || !whole16(q_head_stride, x_dtype))))
        return st::fail(ST_ERR_ALIGN, "%s: strides must be whole 16 bytes", fn);
    if (!st::aligned16(q) || !st::aligned16(k) || !st::aligned16(v) || !st::aligned16(q_out) || !st::aligned16(q_weight) ||
        !st::aligned16(k_weight) || !st::aligned16(cos) || !st::aligned16(sin))
        return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
    a.q = q, a.k = k, a.v = v;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_head_stride = q_head_stride, a.n_heads = q ? n_heads : 0;
    a.q_weight = q_weight, a.k_weight = k_weight, a.cos = cos, a.sin = sin;
    a.eps = eps, a.weight_add = flags & ST_FLAG_NORM_PLUS_ONE ? 1.0f : 0.0f;
    a.rot = rot, a.n_pos = n_pos, a.pairs = (flags & ST_FLAG_ROPE_PAIRS) != 0;
    a.positions = positions, a.slots = slots, a.q_out = q_out;
    a.T = T, a.shift = shifted(T);
    const bool xf32 = x_dtype == ST_F32, qf32 = q_dtype == ST_F32, i8 = cache->dtype == ST_I8;
    if (hd == 64)
        store_by_type<64>(ctx, a, xf32, qf32, i8);
    else if (hd == 128)
        store_by_type<128>(ctx, a, xf32, qf32, i8);
    else
        store_by_type<256>(ctx, a, xf32, qf32, i8);
    return st::launch_check("store_kernel");
}

extern "C" int st_kv_read(st_context *ctx, const st_kv_cache *cache, const int32_t *slots, void *k_out, void *v_out,
                          int out_dtype, int T) {
    const char *const fn = "st_kv_read";
    ReadArgs a{};
    if (!ctx || !slots || !k_out || !v_out) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (int rc = check_cache(fn, cache, &a.c)) return rc;
    if (!act_dtype(out_dtype)) return st::fail(ST_ERR_INVALID, "%s: out_dtype %d (f32 or f16)", fn, out_dtype);
    if (T < 1) return st::fail(ST_ERR_SHAPE, "%s: T=%d", fn, T);
    if (!st::aligned16(k_out) || !st::aligned16(v_out)) return st::fail(ST_ERR_ALIGN, "%s: outputs must be 16-byte aligned", fn);
    a.slots = slots, a.k_out = k_out, a.v_out = v_out, a.T = T, a.shift = shifted(T);
    const bool f32 = out_dtype == ST_F32, i8 = cache->dtype == ST_I8;
    if (cache->head_dim == 64)
        read_by_type<64>(ctx, a, f32, i8);
    else if (cache->head_dim == 128)
        read_by_type<128>(ctx, a, f32, i8);
    else
        read_by_type<256>(ctx, a, f32, i8);
    return st::launch_check("read_kernel");
}
