// Attention of prompts over the paged cache (st_paged_attention, f16 q and
// out, many rows of a sequence). No reference counterpart: it prefills token
// by token (src/inference.rs:93-95).
//
// prompt_kernel: out^T = V^T P^T, P = softmax(K Q^T scale) as attn_kernel
// (attn.hip), on v_mfma_f32_32x32x16_f16: a workgroup takes 128 (row, head)
// pairs of one key head, 32 columns a wave, and goes over the keys once, KT at
// a time.
//  * K and V tiles are double-buffered in LDS, shared by the four waves: f16
//    by the buffer-to-LDS DMA, in the cache's own order, whose 16-byte pieces
//    are the fragments of both products (runs of 256 bytes: no bank
//    conflicts); int8 through registers, converted once.
//  * Scores come as columns, so each lane has one row's maximum, sum and
//    rescaling factor, and the weights are the second product's operand in
//    the registers where they are.
//  * The accumulators are rescaled only when a maximum has grown by 2^8
//    (weights up to 2^8 fit f16, sums are f32).
//  * Weights are rounded to f16 for the second product, which in f32's bits
//    would be two (a high and a low part, as attn_kernel's for f32 results,
//    which a caller may ask for at 10 times the time). The rounding, 2.1e-4
//    rms of each weight, partly averages out and stays below that of the f16
//    result: 4096 rows are 2.13e-4 from the 64-bit form, rounded once they are
//    2.07e-4; the two are 1.5e-4 apart (2.7e-4 and 2.1e-4 at most in draws of
//    all forms).
//  * 4096 rows, f16 cache and int8, in us: 32/8 heads of 128 160-175 (0.79-0.86
//    PFLOP/s) and 208-230, of 64 99 and 131, 16/4 of 256 245 and 303; 128 dims
//    with a cap of 50 215-219 and 263-271, with slopes 217, with a window of
//    512 68. Beyond the products it is the softmax: per score an exp2, and with
//    a cap another and a reciprocal; at 64 dims there are twice as many scores
//    a product; at 256 one wave a SIMD has nothing beside it; int8 tiles are
//    converted again by every workgroup. (int8, 256 dims and a cap or slopes: 7 registers
//    spilled.)
//  * All workgroups of a key head run on one XCD where the head count allows,
//    so a head's K and V are read from HBM once; the last rows, which see
//    most keys, start first.
//  * Few rows over a long cache: chunks of the keys, joined by a second
//    launch.
#include "attn.hpp"

namespace {

using namespace st::attn;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kPairs = 32 * kWaves;
constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit buffer data (gfx9-class)
constexpr int kJoin = 4;                // parts of a join's workgroup
// Tiles of a chunk at least; of a sequence that stays in one chunk. (16 and 32
// rows over 8192 tokens: 19.6 and 21.1 us with 4 tiles at least, 22.5 and 24.4
// with 2, 22.4 and 24.6 with 1; 128 rows: 40.1, 37.3, 37.4; 64 rows over 2048:
// 17.6 with 8 tiles in one chunk, 21.4 with 4.)
constexpr int kLeast = 4, kWhole = 8;
constexpr float kSlack = 8.0f;          // growth of a maximum that is let pass, in powers of two

// (a helper of its own: written inside a kernel template the host pass drops
// the kernel's launch stub)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, _Float16 *lds, unsigned off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, off, 0, 0, 0);
}

// A barrier for LDS alone (__syncthreads also waits for the tile on its way).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float other_half(float v) {  // lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

template <int HD>
constexpr int kKeys = 64;  // keys of a tile (LDS for two of K and V: 64 KiB at 128 dims)

template <int HD, bool I8, bool GEN>
__global__ __launch_bounds__(64 * kWaves, HD == 256 ? 1 : 2) void prompt_kernel(Args a) {
    constexpr int KT = kKeys<HD>, NKT = KT / 32, NS = HD / 16, ND = HD / 32;
    constexpr int kTileE = 16 * HD;                       // elements of a cache tile
    constexpr int kPer = KT * HD / 8 / (64 * kWaves);     // 16-byte pieces of K (and of V) a lane fetches per tile
    __shared__ __align__(16) _Float16 k0s[KT * HD], v0s[KT * HD], k1s[KT * HD], v1s[KT * HD];
    __shared__ __align__(16) float scales[I8 ? 2 : 1][2][I8 ? KT : 1];  // [stage][k, v]
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 31, hf = lane >> 5;
    // (scalars: a division leaves its result in a vector register)
    const int h = scalar((int)blockIdx.x % a.c.heads), item = scalar((int)blockIdx.x / a.c.heads);
    Item it;
    if (!find_item<kPairs, KT, kLeast, kWhole>(a, item, it)) return;
    it = scalars(it);

    // ---- rows: the last block first
    const int block = it.blocks - 1 - it.rb;
    const int npair = it.s.q * a.group, p0 = it.s.kv - it.s.q;
    const int wfirst = block * kPairs + 32 * wave;  // this wave's first pair
    const int pair = wfirst + col;
    const bool real = pair < npair;
    const int tok = real ? pair / a.group : 0, head = h * a.group + (real ? pair - tok * a.group : 0);
    const int pos = real ? p0 + tok : -1;
    const int low = a.window ? max(pos - a.window + 1, 0) : 0;  // keys low .. pos are visible
    // (uniform) positions of the block's and of the wave's first and last rows
    const int bmin = p0 + scalar(block * kPairs / a.group);
    const int bmax = p0 + scalar((min(block * kPairs + kPairs, npair) - 1) / a.group);
    const bool working = wfirst < npair;
    const int wmin = p0 + scalar(wfirst / a.group), wmax = p0 + scalar((min(wfirst + 32, npair) - 1) / a.group);
    const int blow = a.window ? max(bmin - a.window + 1, 0) : 0;    // no row of the block sees keys before this
    const int bhigh = a.window ? bmax - a.window + 1 : 0;           // from here on keys are in every window of the block
    const int wlow = a.window ? max(wmin - a.window + 1, 0) : 0;    // the same for the wave
    const int whigh = a.window ? wmax - a.window + 1 : 0;           // from here on keys are in every window of the wave
    const float slope = GEN && a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    half8 qf[NS];
    {
        const _Float16 *const q = static_cast<const _Float16 *>(a.q) + ((int64_t)(it.s.q0 + tok) * a.n_heads + head) * HD + 8 * hf;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const half8 *>(q + 16 * s);
    }

    // ---- this block's tiles of the chunk
    const int key0 = first_key<KT>(a, it.s);
    int t0 = it.s0, t1 = it.s1;
    t1 = bmax < key0 ? t0 : min(t1, (bmax - key0) / KT + 1);
    if (blow > key0) t0 = max(t0, (blow - key0) / KT);
    t1 = max(t1, t0);

    const int tile0 = key0 / 16, tiles = (it.s.kv + 15) / 16, tsh = a.c.tiles_shift();
    const auto *const pages =
        (const __attribute__((address_space(4))) int32_t *)(a.table + (int64_t)it.b * a.table_stride);
    auto page_of = [&](int t, int p) __attribute__((always_inline)) {  // (-1: none to read)
        return t < tiles && (unsigned)p < (unsigned)a.c.num_pages ? p : -1;
    };
    // A wave fetches kPer pieces a lane, of one cache tile: its tile of the
    // KT / 16, and from which piece on.
    const int my_tile = wave * kPer * 64 * 8 / kTileE, my_piece = wave * kPer * 64 - my_tile * (kTileE / 8);
    // Pages of the tile to fetch, a turn ahead and as they are in the table
    // (as attn_kernel's); a bit of `missing` for each
    // cache tile of the fetched one that is not read (it lands as zeros).
    int page[KT / 16];
    unsigned missing = 0;
    auto look = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < KT / 16; ++j) page[j] = pages[max(min(tile0 + t * (KT / 16) + j, tiles - 1), 0) >> tsh];
    };
    look(t0);
    u32x2 kr[I8 ? kPer : 1], vr[I8 ? kPer : 1];
    float sc = 0.0f;
    auto fetch = [&](_Float16 *ks, _Float16 *vs, int t) __attribute__((always_inline)) {
        int mine = -1;
        missing = 0;
#pragma unroll
        for (int j = 0; j < KT / 16; ++j) {
            const int p = page_of(tile0 + t * (KT / 16) + j, page[j]);
            mine = my_tile == j ? p : mine;
            missing |= p < 0 ? 1u << j : 0u;
        }
        const bool ok = mine >= 0 && t < t1;
        const int ct = tile0 + t * (KT / 16) + my_tile;
        const int64_t e = ok ? a.c.tile(mine, h, ct & ((1 << tsh) - 1)) * kTileE : 0;
        constexpr int size = kTileE * (I8 ? 1 : 2);
        using E = std::conditional_t<I8, signed char, _Float16>;
        const __amdgpu_buffer_rsrc_t rk =
            __builtin_amdgcn_make_buffer_rsrc((void *)(static_cast<E *>(a.c.k) + e), (short)0, ok ? size : 0, kRsrcWord3);
        const __amdgpu_buffer_rsrc_t rv =
            __builtin_amdgcn_make_buffer_rsrc((void *)(static_cast<E *>(a.c.v) + e), (short)0, ok ? size : 0, kRsrcWord3);
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const unsigned off = (my_piece + 64 * i + lane) * 8;
                kr[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, off, 0, 0));
                vr[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, off, 0, 0));
            }
            // lanes 0-15 the key scales of the wave's tile, 16-31 the value scales
            const int64_t at = ok ? a.c.scale(mine, h, (ct * 16) & ((1 << a.c.page_shift) - 1)) : 0;
            const float *const from = ((lane & 16) ? a.c.v_scale : a.c.k_scale) + at;
            sc = from[lane & 15];
            sc = ok ? (lane & 16) ? ldexpf(sc, -8) : sc : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const unsigned off = (my_piece + 64 * i + lane) * 16;
                dma16(rk, ks + (wave * kPer + i) * 64 * 8, off);
                dma16(rv, vs + (wave * kPer + i) * 64 * 8, off);
            }
        }
        look(t + 1);
    };
    auto put = [&](_Float16 *ks, _Float16 *vs, int stage) __attribute__((always_inline)) {  // int8: what fetch brought
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                *reinterpret_cast<half8 *>(ks + ((wave * kPer + i) * 64 + lane) * 8) = i8_to_half8(kr[i]);
                *reinterpret_cast<half8 *>(vs + ((wave * kPer + i) * 64 + lane) * 8) = i8_to_half8(vr[i]);
            }
            if (lane < 32 && my_piece == 0) scales[stage][lane >> 4][my_tile * 16 + (lane & 15)] = sc;
        }
    };

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // m in powers of two; l: this lane's half of the sum
    Held held{0.0f, 0};             // int8
    const float c1 = GEN ? 1.0f : a.scale * kLog2e;

    auto compute = [&](const _Float16 *ks, const _Float16 *vs, int stage, int t, unsigned gone) __attribute__((always_inline)) {
        const int kb = key0 + t * KT;
        if (!working || kb > wmax || kb + KT <= wlow) return;  // (uniform) nothing here for this wave
        f32x16 s[NKT];
#pragma unroll
        for (int n = 0; n < NKT; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
            const _Float16 *const kp = ks + (2 * n + (col >> 4)) * kTileE + hf * 128 + (col & 15) * 8;
#pragma unroll
            for (int j = 0; j < NS; ++j)
                s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(kp + 256 * j), qf[j], s[n], 0, 0, 0);
        }
        // element i of s[n] is key kb + 32 n + 8 (i / 4) + 4 hf + i % 4
        auto key = [&](int n, int i) { return kb + 32 * n + 8 * (i >> 2) + 4 * hf + (i & 3); };
        if constexpr (I8) {
#pragma unroll
            for (int n = 0; n < NKT; ++n)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 f = *reinterpret_cast<const f32x4 *>(&scales[stage][0][32 * n + 8 * g + 4 * hf]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][4 * g + i] *= f[i];
                }
        }
        if constexpr (GEN) {
            const float in = a.cap > 0.0f ? a.scale / a.cap : 0.0f, cap = a.cap * kLog2e, per = a.scale * kLog2e;
            // cap tanh(z) = cap (1 - 2 / (1 + e^(2 z))), z = x scale / cap: to
            // about cap 2^-22, which up to a cap of 64 is a 30th of the weights'
            // own rounding.
            auto by_exp = [&](float x) __attribute__((always_inline)) {
                return cap - 2.0f * cap * __builtin_amdgcn_rcpf(1.0f + exp2_(x * (in * 2.0f * kLog2e)));
            };
            // Over that, scores under a quarter of the cap by tanh's series (its
            // next term is z^10 / 113: 2^-27).
            auto by_series = [&](float x) __attribute__((always_inline)) {
                const float z = x * in, t = z * z;
                const float u = fmaf(t, fmaf(t, fmaf(t, 62.0f / 2835, -17.0f / 315), 2.0f / 15), -1.0f / 3);
                return x * per * fmaf(t, u, 1.0f);
            };
            auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                for (int n = 0; n < NKT; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[n][i] = f(s[n][i]);
            };
            if (a.cap > 64.0f) {
                float far = 0.0f;
#pragma unroll
                for (int n = 0; n < NKT; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) far = fmaxf(far, fabsf(s[n][i]));
                if (__ballot(far * in >= 0.25f))
                    each([&](float x) __attribute__((always_inline)) { return fabsf(x * in) < 0.25f ? by_series(x) : by_exp(x); });
                else
                    each(by_series);
            } else if (a.cap > 0.0f) {
                each(by_exp);
            } else {
                each([&](float x) __attribute__((always_inline)) { return x * per; });
            }
            if (a.slopes) {
#pragma unroll
                for (int n = 0; n < NKT; ++n)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[n][i] = fmaf(slope, (float)(key(n, i) - pos), s[n][i]);
            }
        }
        // (uniform) a key that some row of the wave does not see
        const bool masked = kb + KT - 1 > wmin || kb < whigh || gone;
        if (masked) {
#pragma unroll
            for (int n = 0; n < NKT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int k = key(n, i);
                    s[n][i] = k >= low && k <= pos && !(gone >> (2 * n + (i >> 3)) & 1) ? s[n][i] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NKT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        mx = fmaxf(mx, other_half(mx)) * c1;
        float alpha = 1.0f;
        if (__ballot(mx > m + kSlack)) {  // (m -inf: as soon as anything is visible)
            const float mn = fmaxf(m, mx);
            alpha = mn == -INFINITY ? 1.0f : exp2_(m - mn);
            m = mn;
            l *= alpha;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NKT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[n][i] = exp2_(fmaf(s[n][i], c1, -base));
                sum += s[n][i];
            }
        l += sum;
        if constexpr (I8) {
            // (over 2^8 in LDS, so that no weight overflows)
            auto value_scale = [&](int n, int g) {
                return *reinterpret_cast<const f32x4 *>(&scales[stage][1][32 * n + 8 * g + 4 * hf]);
            };
            if (masked) {  // (those of keys that the row does not see may be anything)
#pragma unroll
                for (int n = 0; n < NKT; ++n)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 f = value_scale(n, g);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[n][4 * g + i] = s[n][4 * g + i] == 0.0f ? 0.0f : s[n][4 * g + i] * f[i];
                    }
            } else {
#pragma unroll
                for (int n = 0; n < NKT; ++n)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 f = value_scale(n, g);
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[n][4 * g + i] *= f[i];
                    }
            }
            float top = 0.0f;
#pragma unroll
            for (int n = 0; n < NKT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[n][i]));
            alpha = held.next(fmaxf(top, other_half(top)), alpha);
            const float down = held.down();
#pragma unroll
            for (int n = 0; n < NKT; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[n][i] *= down;
        }
        if (__ballot(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
#pragma unroll
        for (int n = 0; n < NKT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                half8 p;
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = (_Float16)s[n][8 * u + j];
                const _Float16 *const vp = vs + (2 * n + u) * kTileE + hf * (HD * 8) + col * 8;
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8 *>(vp + 256 * d), p, o[d], 0, 0, 0);
            }
    };
    // f16 values, where some row of the block does not see the tile's every
    // key: 0 times a value that is not finite is a NaN. Those that no row sees
    // may be anything and become zeros; others become zeros too, and the second
    // launch puts them where they are seen. (Without this 4096 rows take 165 us,
    // not 171; 1000 rows over 32000 tokens 720, not 820, though only the last
    // tiles of a block come here.)
    auto clean = [&](_Float16 *vs, int t) __attribute__((always_inline)) {
        const int kb = key0 + t * KT;
        if (I8 || (kb + KT - 1 <= bmin && kb >= bhigh)) return;  // (uniform)
        const bool edge = kb + KT - 1 > bmax || kb < blow;
        for (int i = tid; i < KT * HD / 8; i += 64 * kWaves) {
            const int tile = i / (kTileE / 8), half = i % (kTileE / 8) / HD;
            u32x4 *const at = reinterpret_cast<u32x4 *>(vs + i * 8);
            u32x4 w = *at;
            if (edge) {
                half8 v = __builtin_bit_cast(half8, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = kb + 16 * tile + v_token(half, j);
                    v[j] = k >= blow && k <= bmax ? v[j] : (_Float16)0.0f;
                }
                w = __builtin_bit_cast(u32x4, v);
            }
            unsigned any = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned x = w[j], n = not_finite(x);
                any |= n;
                w[j] = finite(x, n);
            }
            if (edge || any) *at = w;
            if (__builtin_expect(any != 0, 0)) *a.odd = a.call;
        }
        lds_barrier();
    };

    auto turn = [&](_Float16 *ks, _Float16 *vs, _Float16 *kn, _Float16 *vn, int stage, int t) __attribute__((always_inline)) {
        const unsigned gone = missing;
        if constexpr (I8) {
            fetch(kn, vn, t + 1);
            __builtin_amdgcn_sched_barrier(0);
            compute(ks, vs, stage, t, gone);
            put(kn, vn, stage ^ 1);
            __syncthreads();
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // this tile is in LDS, the other free
            fetch(kn, vn, t + 1);
            __builtin_amdgcn_sched_barrier(0);
            clean(vs, t);
            compute(ks, vs, stage, t, gone);
        }
    };
    fetch(k0s, v0s, t0);
    if constexpr (I8) {
        put(k0s, v0s, 0);
        __syncthreads();
    }
    for (int t = t0; t < t1;) {
        turn(k0s, v0s, k1s, v1s, 0, t);
        if (++t >= t1) break;
        turn(k1s, v1s, k0s, v0s, 1, t);
        ++t;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a fetch past the end)

    l += other_half(l);
    if constexpr (I8) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = ldexpf(o[d][i], held.e + 8);
    }
    // ---- the rows, or a chunk's sums to memory, four dims of the block's pairs
    // at a time
    const int row = it.s.q0 + tok, mine = 32 * wave + col;
    const int64_t at = (int64_t)item * a.c.heads + h;
    f32x4 *const part = reinterpret_cast<f32x4 *>(a.part) + at * (HD / 4) * kPairs + mine;
    if (real && it.chunks == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a row that sees nothing is zero)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = {o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv};
                store_out(a, v, row, head, 32 * d + 8 * g + 4 * hf, HD);
            }
    } else if (real) {
        if (t1 > t0) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    part[(8 * d + 2 * g + hf) * kPairs] = f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        }
        // (a row whose scores here are all NaN has no maximum: -inf would say
        // that it sees nothing of the chunk, and the join would pass it over)
        if (hf == 0) reinterpret_cast<f32x2 *>(a.part_ml)[at * kPairs + mine] = f32x2{l != l ? 0.0f : m, l};
    }
}

// Sum of the f16 values of dims 4 d .. 4 d + 3 that are not finite, that keys
// low .. pos have, over the tiles where prompt_kernel left such values out
// (those that some row of the block, at positions bmin .. bmax, does not see).
template <int HD>
__device__ f32x4 odd_values(const Args &a, const Item &it, int h, int d, int bmin, int bmax, int low, int pos) {
    constexpr int KT = kKeys<HD>;
    const int key0 = first_key<KT>(a, it.s), steps = steps_of<KT>(a, it.s), tsh = a.c.tiles_shift();
    const int blow = a.window ? max(bmin - a.window + 1, 0) : 0, bhigh = a.window ? bmax - a.window + 1 : 0;
    f32x4 sum = {};
    for (int t = 0; t < steps; ++t) {
        const int kb = key0 + t * KT;
        if (kb > bmax || kb + KT <= blow || (kb + KT - 1 <= bmin && kb >= bhigh)) continue;
        for (int k = kb; k < kb + KT; k += 4) {  // places of one half of a piece
            if (k > pos || k + 3 < low) continue;
            const int p = a.table[(int64_t)it.b * a.table_stride + (k >> 4 >> tsh)];
            if ((unsigned)p >= (unsigned)a.c.num_pages) continue;
            const int64_t tile = a.c.tile(p, h, (k >> 4) & ((1 << tsh) - 1));
            const _Float16 *const v = static_cast<const _Float16 *>(a.c.v) + tile * (16 * HD) + v_half(k & 15) * (HD * 8) + v_place(k & 15);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const half4 x = *reinterpret_cast<const half4 *>(v + (4 * d + i) * 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float y = (float)x[j];
                    sum[i] += k + j >= low && k + j <= pos && !(fabsf(y) < INFINITY) ? y : 0.0f;
                }
            }
        }
    }
    return sum;
}

// After prompt_kernel: its chunks joined. A launch of its own: the sums of a
// chunk are 64 KiB at 128 dims, which one workgroup (the last to count in) took
// 3 us a chunk to read; here the workgroups of a block's chunks share its dims
// (77 rows over 8192 tokens, 32/8 heads of 128: 35 us with both launches, 82
// with the join in the first). And the values that prompt_kernel left out, if
// it met any: a sum with one is infinite of its sign, or NaN, whatever the
// weight.
template <int HD>
__global__ __launch_bounds__(kJoin * kPairs) void prompt_join_kernel(Args a) {
    constexpr int N = 8;  // chunks asked for at once
    __shared__ __align__(16) f32x4 sums[kJoin - 1][kPairs];
    __shared__ __align__(8) f32x2 tops[kJoin - 1][kPairs];
    const int tid = threadIdx.x, mine = tid % kPairs, part = uniform(tid / kPairs);
    const int h = scalar((int)blockIdx.x % a.c.heads), item = scalar((int)blockIdx.x / a.c.heads);
    Item it;
    const bool odd = uniform(*a.odd) == a.call;  // (a stale one costs time, no more)
    if (!a.split && !odd) return;
    if (!find_item<kPairs, kKeys<HD>, kLeast, kWhole>(a, item, it)) return;
    it = scalars(it);
    if (it.chunks == 1 && !odd) return;
    const int block = it.blocks - 1 - it.rb, pair = block * kPairs + mine;
    const bool real = pair < it.s.q * a.group;
    const int tok = real ? pair / a.group : 0, head = h * a.group + (real ? pair - tok * a.group : 0);
    const int p0 = it.s.kv - it.s.q, npair = it.s.q * a.group, pos = real ? p0 + tok : -1;
    auto odd_sum = [&](int d) {
        return odd_values<HD>(a, it, h, d, p0 + block * kPairs / a.group, p0 + (min(block * kPairs + kPairs, npair) - 1) / a.group,
                              a.window ? max(pos - a.window + 1, 0) : 0, pos);
    };
    if (it.chunks == 1) {
        for (int d = part; d < HD / 4; d += kJoin) {
            const f32x4 sum = odd_sum(d);
            if (!real || (sum[0] == 0.0f && sum[1] == 0.0f && sum[2] == 0.0f && sum[3] == 0.0f)) continue;
            const int row = it.s.q0 + tok;
            const f32x4 v = gated(a, sum, row, head, 4 * d);
            // (added to what is there: that may be a NaN, or infinite by a value
            // that every row of its block sees)
            _Float16 *const to = static_cast<_Float16 *>(a.out) + ((int64_t)row * a.n_heads + head) * HD + 4 * d;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sum[i] != 0.0f) to[i] = (_Float16)((float)to[i] + v[i]);
        }
        return;
    }
    const int share = scalar((HD / 4 + it.chunks - 1) / it.chunks);  // groups of four dims
    const int end = min((it.chunk + 1) * share, HD / 4);
    // many chunks: cut among the parts, else the dims are
    const bool cut = it.chunks > 2 * N;
    const int each = cut ? (it.chunks + kJoin - 1) / kJoin : it.chunks;
    const int first = cut ? part * each : 0, last = min(first + each, it.chunks);
    const int64_t at = (int64_t)it.first * a.c.heads + h, next = (int64_t)it.blocks * a.c.heads;
    const f32x2 *const ml = reinterpret_cast<const f32x2 *>(a.part_ml) + at * kPairs + mine;
    // (the workgroup's turns are the same for all its waves)
    for (int d0 = it.chunk * share; d0 < end; d0 += cut ? 1 : kJoin) {
        const int d = cut ? d0 : min(d0 + part, end - 1);
        const f32x4 *const from = reinterpret_cast<const f32x4 *>(a.part) + (at * (HD / 4) + d) * kPairs + mine;
        float top = -INFINITY, total = 0.0f;
        f32x4 sum = {};
        auto add = [&](const f32x2 *x, const f32x4 *v, int n) __attribute__((always_inline)) {
            float high = top;
#pragma unroll
            for (int i = 0; i < N; ++i) high = fmaxf(high, i < n ? x[i][0] : -INFINITY);
            if (high == -INFINITY) return;  // (chunks that the row does not see hold no sums)
            const float was = exp2_(top - high);
            top = high, total *= was;
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] *= was;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool use = i < n && x[i][0] > -INFINITY;
                const float w = use ? exp2_(x[i][0] - high) : 0.0f;
                total = use ? fmaf(w, x[i][1], total) : total;
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] = use ? fmaf(w, v[i][k], sum[k]) : sum[k];
            }
        };
        for (int c0 = first; c0 < last; c0 += N) {
            f32x2 x[N];
            f32x4 v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = min(c0 + i, last - 1);
                x[i] = ml[c * next * kPairs];
                v[i] = from[c * next * (HD / 4) * kPairs];
            }
            add(x, v, last - c0);
        }
        if (cut) {
            if (part) sums[part - 1][mine] = sum, tops[part - 1][mine] = f32x2{top, total};
            __syncthreads();
            f32x2 x[N];
            f32x4 v[N];
#pragma unroll
            for (int i = 0; i < kJoin - 1; ++i) x[i] = tops[i][mine], v[i] = sums[i][mine];
            __syncthreads();
            if (part) continue;
            add(x, v, kJoin - 1);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        if (odd) {
            const f32x4 more = odd_sum(d);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += more[i];
        }
        if (real && (cut || d0 + part < end))
            store_out(a, f32x4{sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv}, it.s.q0 + tok, head, 4 * d, HD);
    }
}

template <int HD, bool I8, bool GEN>
int launch_prompt(st_context *ctx, Args a) {
    const int heads = a.c.heads;
    // chunks only where the row blocks alone leave CUs without work (at 256 dims
    // a CU holds one workgroup: 77 rows over 8192 tokens, 16 heads of 256, 71 us
    // with as many chunks as fit at once, 80 with twice that)
    const int64_t blocks = ((int64_t)a.T * a.group + kPairs - 1) / kPairs * heads, slots = (HD == 256 ? 1 : 2) * ctx->num_cus;
    if (int rc = plan_cut(ctx, a, kPairs, HD, kKeys<HD>, kLeast, (slots - blocks) / heads)) return rc;
    a.odd = ctx->split_counters + st::kSplitCounters, a.call = ++ctx->calls;
    st::launch(ctx, prompt_kernel<HD, I8, GEN>, dim3((unsigned)(a.G * heads)), dim3(64 * kWaves), 0, a);
    if (int rc = st::launch_check("prompt_kernel"); rc || (I8 && !a.split)) return rc;
    st::launch(ctx, prompt_join_kernel<HD>, dim3((unsigned)(a.G * heads)), dim3(kJoin * kPairs), 0, a);
    return st::launch_check("prompt_join_kernel");
}

template <int HD>
int by_type(st_context *ctx, const Args &a, bool i8) {
    const bool gen = a.cap > 0.0f || a.slopes;
    if (i8) return gen ? launch_prompt<HD, true, true>(ctx, a) : launch_prompt<HD, true, false>(ctx, a);
    return gen ? launch_prompt<HD, false, true>(ctx, a) : launch_prompt<HD, false, false>(ctx, a);
}

}  // namespace

namespace st {
namespace attn {

int prompt_attention(st_context *ctx, const Args &a, bool i8, int hd) {
    return hd == 64 ? by_type<64>(ctx, a, i8) : hd == 128 ? by_type<128>(ctx, a, i8) : by_type<256>(ctx, a, i8);
}

}  // namespace attn
}  // namespace st
