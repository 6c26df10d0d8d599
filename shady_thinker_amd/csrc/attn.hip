// Attention of new rows over the paged cache (st_paged_attention): one token
// of each sequence, a few drafted ones, or prompts. Replaces
// src/shaders/gqa_attention_head.wgsl:1-124 and gqa_reduce.wgsl:1-65 (one
// token over a contiguous f32 cache) and sigmoid_mul.wgsl (the output gate).
//
// attn_kernel: out^T = V^T P^T, P = softmax(K Q^T scale), on
// v_mfma_f32_16x16x32_f16, in one pass over the keys with the running maximum
// and sum of each row.
//  * Columns of the matrices are (row, head) pairs that share a key head, so
//    one read of the cache serves a whole group of heads (and several drafted
//    rows); f32 calls take two columns for a pair, its f16 high and low part
//    (22 bits of q, scaled by a power of two, and of each softmax weight), so
//    that nothing but the cache itself is held in 16 bits.
//  * A wave takes 32 keys (two tiles) of f16 or 64 of int8 at a time. The
//    scores' lanes are the columns and each lane's keys are those whose values
//    one piece of the cache's value tiles holds: the weights go from the first
//    product to the second in the registers where they are, and K and V go
//    from HBM to registers in 16-byte pieces, with no LDS.
//  * Bound by HBM (4 matrix cycles per KiB of the cache are 4% of its time),
//    that is by how many loads are in flight: the next step's are issued
//    before this step's are used. 32/8 heads of 128, f16 cache: 31 sequences
//    of 800 to 8191 tokens 106 us (5.4 TB/s); one of 32000 28 us (4.6 TB/s);
//    int8, the same 31 72 us (4.1 TB/s), one of 65000 35 us (3.9 TB/s, of
//    which 3.5 us join the chunks). 16 sequences of 400 to 4000 tokens, f16
//    and int8: 8 key heads of 128 35 us (4.1 TB/s) and 31, 8 of 64 21 and 24,
//    4 of 256 39 and 34, 32 of 128 (one query head each) 108 (5.3 TB/s) and 72.
//    At 256 dims one step's pieces fill the registers, so loads and products
//    take turns (and int8 spills 2 to 13 of them, f16 with a cap or slopes 3
//    to 7; int8 with either at 128 dims 1 or 2).
//  * f16 queries and results: the weights too are rounded to f16, one column a
//    pair and half the products. The rounding (2.1e-4 rms of each weight,
//    which partly averages out; their sum is of unrounded ones) is below that
//    of the f16 result: 2.2e-4 from the 64-bit form, where results rounded once
//    are 2.1e-4. f32 results keep 22 bits.
//  * A short call is its chain of latencies: 32 keys in 6.2 us, of which 0.6
//    are the item, 1.5 until the loads are out, 0.6 until they are used, 0.3
//    the waves' meeting, 0.5 the store (the rest is the launch).
//  * The cut: every sequence's keys go in chunks of C steps to workgroups of
//    four waves, C the smallest with which all fit the grid (two workgroups a
//    CU), found by each workgroup from the lengths on the device (so that a captured graph stays
//    right, and batches of mixed lengths even, as they grow). The last chunk
//    of a (row block, key head) to count in joins them in order: the counter
//    protocol of the split-K kernels (see qmv_kernel.hpp on its visibility).
#include "attn.hpp"

#include <algorithm>
#include <climits>

namespace {

using namespace st::attn;

constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit buffer data (gfx9-class)
constexpr int kCoherent = 1 | 16;       // sc0 sc1: write through / read past this XCD's L2
constexpr float kShift = 14.0f;         // f16 caches: weights are held times 2^14, f16 keeps them normal down to 2^-28

// Keys of a step of one wave: 32 (two tiles) of f16, 64 of int8 (the same
// bytes; what a step costs beside its products then counts half).
template <bool I8>
constexpr int kStep = I8 ? 64 : 32;
// Steps of a chunk (a multiple of the first), steps that stay in one (a join
// costs 3 to 3.5 us). 16 steps of f16 in one chunk against 32: a sequence of
// 1000 tokens 9.1 and 10.1 us, 16 sequences of up to 4000 of 256 dims 39 and
// 43, batches of 128 dims the same or 3% less; with 8, one of 333 tokens takes
// 8.5, not 6.3. At least 4 steps against 8: 1000 tokens 8.0 and 9.2, but 4
// sequences of up to 2000 13.1 and 11.2.
template <bool I8>
constexpr int kLeast = I8 ? 4 : 8;
template <bool I8>
constexpr int kWhole = I8 ? 8 : 16;

template <int HD, bool I8>
struct Frag {
    static constexpr int SUB = kStep<I8> / 32, NS = HD / 32, ND = HD / 16;
    // 16 bytes a load: a piece of f16; of int8 the pieces of two tokens (k),
    // of two dims (v)
    u32x4 k[I8 ? SUB : 2 * SUB][NS], v[SUB][I8 ? ND / 2 : ND];
    float ks, vs;  // int8: the scales of key `lane` of the step's 64
    unsigned ok;                                       // (uniform) a bit for each tile that is there
};

// Piece `half` of the pair in w (int8), or w (f16).
template <bool I8>
__device__ __forceinline__ half8 piece(u32x4 w, int half) {
    if constexpr (!I8) return __builtin_bit_cast(half8, w);
    const unsigned a = half ? w.z : w.x, b = half ? w.w : w.y;
    return i8_to_half8(u32x2{a, b});
}

template <bool NTL>
__device__ __forceinline__ u32x4 fetch16(const void *p) {
    const u32x4 *const q = static_cast<const u32x4 *>(p);
    return NTL ? __builtin_nontemporal_load(q) : *q;
}

// Over the four lanes of a column (col, col + 16, + 32, + 48).
template <typename Op>
__device__ __forceinline__ float over_q4(float v, Op op) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float max_q4(float v) {
    return over_q4(v, [](float x, float y) { return fmaxf(x, y); });
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float half_turn(float v) { return dpp<0x128>(v); }  // the lane eight columns on

// Two steps' pieces in registers (256 dims: one, two do not fit).
template <int HD>
constexpr bool kTwo = HD <= 128;

// What a call's rows are like.
constexpr int kRows = 0;    // sequences of several rows, perhaps
constexpr int kOne = 1;     // one row each: a block's pairs see the same keys
constexpr int kOneNt = 2;   // the same, and the cache by non-temporal loads

// GEN: capped scores or slopes.
template <int HD, bool I8, bool SPLIT, bool GEN, int MODE, int NW>
__global__ __launch_bounds__(64 * NW, 8 / NW) void attn_kernel(Args a) {
    constexpr int PB = SPLIT ? 8 : 16;  // pairs of a block
    constexpr bool NTL = MODE == kOneNt, ONE = MODE != kRows;
    constexpr int ST = kStep<I8>, SUB = ST / 32, NS = HD / 32, ND = HD / 16, kRow = HD + 4, NT = 64 * NW;
    using F = Frag<HD, I8>;
    using E = std::conditional_t<I8, signed char, _Float16>;
    extern __shared__ __align__(16) float so[];  // [NW][PB][kRow]
    __shared__ float sm[NW][16], sl[NW][16];
    __shared__ float sw[kMaxChunks * PB];
    __shared__ __align__(16) float scales[I8 ? NW : 1][2][I8 ? ST : 1];  // int8: each wave's step's, by key
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.y;
    Item it;
    if (!find_item<PB, ST, kLeast<I8>, kWhole<I8>>(a, (int)blockIdx.x, it)) return;
    it = scalars(it);

    // ---- this lane's column: a (row, head) pair
    const int npair = it.s.q * a.group;
    const int pair = it.rb * PB + (SPLIT ? col & 7 : col);
    const bool real = pair < npair;
    const int tok = real ? row_of_pair(a, pair) : 0, head = h * a.group + (real ? pair - tok * a.group : 0);
    const int p0 = it.s.kv - it.s.q;  // position of the sequence's first row
    const int pos = real ? p0 + tok : -1;
    const int low = a.window ? max(pos - a.window + 1, 0) : 0;  // keys low .. pos are visible
    // (uniform: the block's first and last rows' positions)
    const int pmin = p0 + scalar(row_of_pair(a, it.rb * PB)), pmax = p0 + scalar(row_of_pair(a, min(it.rb * PB + PB, npair) - 1));
    const int wmax = a.window ? pmax - a.window + 1 : 0;  // from here on a key is in every row's window
    const int wmin = a.window ? pmin - a.window + 1 : 0;  // before this it is in none's
    const float slope = GEN && a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    // ---- the queries: loads on their way while the pages are looked up
    half8 qf[NS];
    float qs = a.scale;  // scores are matrix sums times qs
    float x32[SPLIT ? NS : 1][8];
    {
        const int64_t at = ((int64_t)(it.s.q0 + tok) * a.n_heads + head) * HD + q4 * 8;
        if (SPLIT && a.q_f32) {
            const float *const q = static_cast<const float *>(a.q) + at;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const f32x4 u = *reinterpret_cast<const f32x4 *>(q + 32 * s + i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x32[SPLIT ? s : 0][i + j] = u[j];
                }
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const half8 *>(static_cast<const _Float16 *>(a.q) + at + 32 * s);
            if constexpr (SPLIT) {
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x32[s][i] = (float)qf[s][i];
            }
        }
    }

    // ---- the chunk's steps: this wave's are s0 + wave, + NW, ...
    const int key0 = first_key<ST>(a, it.s);
    const int tile0 = key0 / 16, tiles = (it.s.kv + 15) / 16;  // tiles that hold a token
    const int tsh = a.c.tiles_shift();
    // Pages come through the scalar cache a step ahead, as they are in the
    // table and from a place that is in it; whether there is such a tile and
    // page is asked when the step is loaded (asked at once, every step waits for
    // its table entry: 1 us more at one sequence of 1000 tokens).
    const auto *const pages =
        (const __attribute__((address_space(4))) int32_t *)(a.table + (int64_t)it.b * a.table_stride);
    int next[2 * SUB];  // of the step to load
    auto look = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2 * SUB; ++j) next[j] = pages[max(min(tile0 + 2 * SUB * step + j, tiles - 1), 0) >> tsh];
    };
    auto page_of = [&](int t, int p) __attribute__((always_inline)) {  // (-1: none to read)
        return t < tiles && (unsigned)p < (unsigned)a.c.num_pages ? p : -1;
    };
    look(it.s0 + wave);
    // This lane's pieces. Scores: row r = lane % 16 of product `half` is a
    // place of tile r / 8 of two, so that rows 4 q4 .. 4 q4 + 3 of both
    // products, the lane's scores, are the places of V piece q4 % 2 of tile
    // q4 / 2. f16: place r % 8 + 8 half (score i of product `half` goes to
    // place 4 half + i of the piece; runs of 128 bytes a load). int8: place
    // 2 i' + half, i' = r % 8 with its upper two bits swapped (to place
    // 2 i + half), so that one 16-byte load has both products' rows; f16 in
    // that order reads every line twice, by half (32 sequences of 1000: 21 ->
    // 32 us). Values: row r is dim 16 d + r, of int8 32 d + 2 r + half.
    const int in_tile = I8 ? ((col & 1) | (col >> 1 & 2) | (col << 1 & 4)) * 16 : (col & 7) * 8;
    const int k_off = q4 * 128 + in_tile, v_off = ((q4 & 1) * HD + (I8 ? 2 * col : col)) * 8;
    auto load = [&](F &f, int step) __attribute__((always_inline)) {
        const bool in = step < it.s1;
        f.ok = 0;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const int t = tile0 + 2 * (SUB * step + u);
            const int p0 = page_of(t, next[2 * u]), p1 = page_of(t + 1, next[2 * u + 1]);
            const bool ok0 = in && p0 >= 0, ok1 = in && p1 >= 0;
            f.ok |= (ok0 ? 1u : 0u) << (2 * u) | (ok1 ? 1u : 0u) << (2 * u + 1);
            // a tile that is not read: every lane at the cache's first piece
            const int64_t e0 = ok0 ? a.c.tile(p0, h, t & ((1 << tsh) - 1)) * (16 * HD) : 0;
            const int64_t e1 = ok1 ? a.c.tile(p1, h, (t + 1) & ((1 << tsh) - 1)) * (16 * HD) : 0;
            const bool kt = col >= 8, vt = q4 >= 2;
            const E *kp = static_cast<const E *>(a.c.k) + (kt ? e1 : e0) + ((kt ? ok1 : ok0) ? k_off : 0);
            const E *vp = static_cast<const E *>(a.c.v) + (vt ? e1 : e0) + ((vt ? ok1 : ok0) ? v_off : 0);
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int half = 0; half < (I8 ? 1 : 2); ++half)
                    f.k[I8 ? u : 2 * u + half][s] = fetch16<NTL>(kp + 512 * s + 64 * half);
#pragma unroll
            for (int d = 0; d < (I8 ? ND / 2 : ND); ++d) f.v[u][d] = fetch16<NTL>(vp + (I8 ? 256 : 128) * d);
        }
        if constexpr (I8) {
            // (as an array the pages go through scratch memory, every step)
            int p = next[0], n1 = next[1], n2 = next[2], n3 = next[3];
            asm("" : "+s"(n1), "+s"(n2), "+s"(n3));
            p = q4 == 1 ? n1 : p, p = q4 == 2 ? n2 : p, p = q4 == 3 ? n3 : p;
            const int t = tile0 + 4 * step + q4;
            const bool there = in && page_of(t, p) >= 0;
            const int64_t at = there ? a.c.scale(p, h, ((t * 16) & ((1 << a.c.page_shift) - 1)) + col) : 0;
            f.ks = a.c.k_scale[at], f.vs = a.c.v_scale[at];
        }
        look(step + NW);
    };

    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    // int8. (256 dims: in LDS between steps, as the registers are all taken: 16
    // sequences of up to 4000 take 33.7 us, capped 38.5, and in registers 34.9
    // and 43.3; six of 5 drafted rows 38.1 in registers, 39.8 in LDS)
    Held held{0.0f, 0};
    constexpr bool kApart = I8 && !kTwo<HD> && (ONE || GEN);
    __shared__ Held apart[kApart ? NT : 1];
    if constexpr (kApart) apart[tid] = held;
    unsigned odd = 0;  // values that were not finite and not seen by every row

    auto compute = [&](F &f, int step) __attribute__((always_inline)) {
        const int kb = key0 + ST * step;
        // this lane's keys: key(j) for weight j % 8 of product j / 8
        const int kl = kb + 16 * (q4 >> 1) + 4 * (q4 & 1);
        auto key = [&](int j) { return kl + (j & 3) + 8 * (j >> 2 & 1) + 32 * (j >> 3); };
        auto there = [&](int j) { return (f.ok >> (2 * (j >> 3) + (q4 >> 1)) & 1) != 0; };
        float x[8 * SUB];
        float alpha;
        if constexpr (I8) {
            // Scales go by LDS to the lanes that have their keys.
            scales[wave][0][lane] = f.ks, scales[wave][1][lane] = f.vs;
        }
        auto scale_of = [&](int which, int t) {  // of x[4 t] .. x[4 t + 3]
            return *reinterpret_cast<const f32x4 *>(&scales[wave][which][32 * (t >> 1) + 16 * (q4 >> 1) + 4 * (q4 & 1) + 8 * (t & 1)]);
        };
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            f32x4 s4[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                s4[half] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    s4[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(piece<I8>(f.k[I8 ? u : 2 * u + half][s], half), qf[s], s4[half], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v = I8 ? s4[j & 1][j >> 1] : s4[j >> 2][j & 3];
                if constexpr (SPLIT) v += half_turn(v);
                x[8 * u + j] = v * qs;
            }
        }
        if constexpr (I8) {
#pragma unroll
            for (int t = 0; t < 2 * SUB; ++t) {
                const f32x4 ks = scale_of(0, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * t + i] *= ks[i];
            }
        }
        if constexpr (GEN) {
            if (a.cap > 0.0f) {
#pragma unroll
                for (int j = 0; j < 8 * SUB; ++j) x[j] = a.cap * kLog2e * tanhf(x[j] / a.cap);
            }
            if (a.slopes) {
#pragma unroll
                for (int j = 0; j < 8 * SUB; ++j) x[j] = fmaf(slope, (float)(key(j) - pos), x[j]);
            }
        }
        // (uniform) whether every key is there for every row
        const bool full = f.ok == (1u << (2 * SUB)) - 1 && kb + ST - 1 <= pmin && kb >= wmax;
        unsigned seen = (1u << (8 * SUB)) - 1;
        if (!full) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8 * SUB; ++j) {
                const int kj = key(j);
                const bool see = there(j) && kj >= low && kj <= pos;
                seen |= see ? 1u << j : 0u;
                x[j] = see ? x[j] : -INFINITY;
                // values no row of the block sees may be anything
                const bool any = there(j) && kj <= pmax && kj >= wmin;
                if constexpr (!I8) {
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        half8 w = __builtin_bit_cast(half8, f.v[j >> 3][d]);
                        w[j & 7] = any ? w[j & 7] : (_Float16)0.0f;
                        f.v[j >> 3][d] = __builtin_bit_cast(u32x4, w);
                    }
                }
            }
            if constexpr (!I8 && !ONE) {
                // 0 times a value that is not finite is a NaN, also for rows
                // that do not see it: zero too, until the loop is done
                if (pmin != pmax) {
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const unsigned w = f.v[0][d][i], t = not_finite(w);
                            odd |= t;
                            f.v[0][d][i] = finite(w, t);
                        }
                }
            }
        }
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 8 * SUB; ++j) mx = fmaxf(mx, x[j]);
        const float mn = fmaxf(m, max_q4(mx));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float grown = exp2_(m - base);  // (0 before the first visible key)
        alpha = grown;
        m = mn;
        float p[8 * SUB], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8 * SUB; ++j) {
            p[j] = exp2_(x[j] - (I8 ? base : base - kShift));
            sum += p[j];
        }
        l = fmaf(l, grown, sum);
        if constexpr (I8) {
#pragma unroll
            for (int t = 0; t < 2 * SUB; ++t) {
                const f32x4 vs = scale_of(1, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[4 * t + i] *= vs[i];
            }
            if (!full) {  // (a scale that the row does not see may be anything)
#pragma unroll
                for (int j = 0; j < 8 * SUB; ++j) p[j] = seen >> j & 1 ? p[j] : 0.0f;
            }
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8 * SUB; ++j) top = fmaxf(top, fabsf(p[j]));
            volatile Held *const mine = &apart[kApart ? tid : 0];
            if constexpr (kApart) held.top = mine->top, held.e = mine->e;
            alpha = held.next(max_q4(top), grown);
            if constexpr (kApart) mine->top = held.top, mine->e = held.e;
            const float down = held.down();
#pragma unroll
            for (int j = 0; j < 8 * SUB; ++j) p[j] *= down;
        }
        if (__ballot(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            half8 pf;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const _Float16 hi = (_Float16)p[8 * u + j];
                pf[j] = hi;
                if constexpr (SPLIT) pf[j] = col < 8 ? hi : (_Float16)(p[8 * u + j] - (float)hi);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(piece<I8>(f.v[u][I8 ? d / 2 : d], d & 1), pf, o[d], 0, 0, 0);
        }
    };

    auto split_q = [&]() __attribute__((always_inline)) {
        if constexpr (SPLIT) {
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x32[s][i]));
            top = max_q4(top);
            const int e = max((int)((__float_as_uint(top) >> 23) & 255) - 127, -126);
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = ldexpf(x32[s][i], -e);
                    const _Float16 hi = (_Float16)v;
                    qf[s][i] = col < 8 ? hi : (_Float16)(v - (float)hi);
                }
            qs = ldexpf(qs, e);
        }
        if (!real) {
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[s] = half8{0, 0, 0, 0, 0, 0, 0, 0};
        }
        if (!GEN || !(a.cap > 0.0f)) qs *= kLog2e;  // (scores in powers of two)
    };

    if constexpr (kTwo<HD>) {
        // Two steps a turn, one exit: with a break between them the compiler
        // saw a way from there back to the top with the second buffer's loads
        // still in flight, and waited for every load before issuing more.
        int step = it.s0 + wave;
        const int mine = step < it.s1 ? (it.s1 - step + NW - 1) / NW : 0;
        F fa, fb;
        load(fa, step);
        __builtin_amdgcn_sched_barrier(0);  // (or the queries are waited for first)
        split_q();
        for (int i = 0; i < mine / 2; ++i, step += 2 * NW) {
            load(fb, step + NW);
            __builtin_amdgcn_sched_barrier(0);
            compute(fa, step);
            load(fa, step + 2 * NW);
            __builtin_amdgcn_sched_barrier(0);
            compute(fb, step + NW);
        }
        if (mine & 1) compute(fa, step);
    } else {
        F f;
        split_q();
        for (int step = it.s0 + wave; step < it.s1; step += NW) {
            load(f, step);
            compute(f, step);
        }
    }

    if constexpr (!I8 && !ONE) {
        // Such values again, for the rows that see them: their sums are
        // infinite of the value's sign, or NaN, whatever the weight.
        if (__ballot(odd != 0)) {
            look(it.s0 + wave);
            for (int step = it.s0 + wave; step < it.s1; step += NW) {
                F f;
                load(f, step);
                half8 see;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = key0 + ST * step + 16 * (q4 >> 1) + 4 * (q4 & 1) + (j & 3) + 8 * (j >> 2);
                    see[j] = (f.ok >> (q4 >> 1) & 1) && k >= low && k <= pos ? (_Float16)1.0f : (_Float16)0.0f;
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    half8 v = __builtin_bit_cast(half8, f.v[0][d]), up, down;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool bad = !(fabsf((float)v[j]) < INFINITY);
                        up[j] = bad && !(v[j] < (_Float16)0.0f) ? (_Float16)1.0f : (_Float16)0.0f;  // +inf, NaN
                        down[j] = bad && !(v[j] > (_Float16)0.0f) ? (_Float16)1.0f : (_Float16)0.0f;
                    }
                    const f32x4 none = {0, 0, 0, 0};
                    const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_f16(up, see, none, 0, 0, 0);
                    const f32x4 m = __builtin_amdgcn_mfma_f32_16x16x32_f16(down, see, none, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] += (n[i] > 0.0f ? INFINITY : 0.0f) + (m[i] > 0.0f ? -INFINITY : 0.0f);
                }
            }
        }
    }

    // ---- the waves meet in LDS
    l = over_q4(l, [](float x, float y) { return x + y; });
    if constexpr (I8) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] = ldexpf(o[d][i], held.e);
    }
    if constexpr (SPLIT) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] += half_turn(o[d][i]);
    }
    if (col < PB) {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if constexpr (I8) {  // (dims 32 d + 8 q4 .. + 7 in o[2 d] and o[2 d + 1], by turns)
                if (d & 1) continue;
                float *const to = &so[(wave * PB + col) * kRow + d * 16 + q4 * 8];
                *reinterpret_cast<f32x4 *>(to) = f32x4{o[d][0], o[d + 1][0], o[d][1], o[d + 1][1]};
                *reinterpret_cast<f32x4 *>(to + 4) = f32x4{o[d][2], o[d + 1][2], o[d][3], o[d + 1][3]};
            } else {
                *reinterpret_cast<f32x4 *>(&so[(wave * PB + col) * kRow + d * 16 + q4 * 4]) = o[d];
            }
        }
        if (q4 == 0) sm[wave][col] = m, sl[wave][col] = l;
    }
    __syncthreads();
    const int pairs_here = min(PB, npair - it.rb * PB);
    const int quads = pairs_here * (HD / 4);
    const int row_id = (int)blockIdx.x * a.c.heads + h;
    auto weight = [](float mw, float top) { return mw == -INFINITY ? 0.0f : exp2_(mw - top); };
    auto put = [&](f32x4 v, int p, int d) {
        const int g = it.rb * PB + p, t = row_of_pair(a, g);
        store_out(a, v, it.s.q0 + t, h * a.group + g - t * a.group, d, HD);
    };
    const __amdgpu_buffer_rsrc_t rp =
        __builtin_amdgcn_make_buffer_rsrc((void *)a.part, (short)0, a.G * a.c.heads * PB * HD * 4, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rm =
        __builtin_amdgcn_make_buffer_rsrc((void *)a.part_ml, (short)0, a.G * a.c.heads * PB * 8, kRsrcWord3);
    for (int i = tid; i < quads; i += NT) {
        const int p = i / (HD / 4), d = i % (HD / 4) * 4;
        float top = sm[0][p];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, sm[w][p]);
        f32x4 v = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = weight(sm[w][p], top);
            sum = fmaf(f, sl[w][p], sum);
            v += f * *reinterpret_cast<const f32x4 *>(&so[(w * PB + p) * kRow + d]);
        }
        if (it.chunks == 1) {
            put(v * (sum == 0.0f ? 0.0f : 1.0f / sum), p, d);  // (a row that sees nothing is zero)
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rp, ((row_id * PB + p) * HD + d) * 4, 0, kCoherent);
            if (d == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(top), __float_as_uint(sum)}, rm, (row_id * PB + p) * 8, 0,
                                                      kCoherent);
        }
    }
    if (it.chunks == 1) return;

    // ---- the chunks meet: the last one to count in joins them
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's partial results are in memory
    __syncthreads();
    if (tid == 0) {
        unsigned *const cnt = a.cnt + st::spread_counter(it.counter * a.c.heads + h);
        const unsigned done = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        s_last = done == (unsigned)it.chunks - 1;
        if (s_last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
    __syncthreads();
    if (!s_last) return;
    auto row_at = [&](int c) { return (it.first + c * it.blocks) * a.c.heads + h; };
    // Thread (part, quad) takes every parts-th chunk of its quad, so that all
    // chunks' loads are in flight at once; the parts meet in LDS, in order.
    const int parts = max(1, min(NT / quads, (int)(sizeof(float) * NW * PB * kRow / (16 * quads))));
    const int part = tid / quads, i = tid % quads, p = i / (HD / 4), d = i % (HD / 4) * 4;
    constexpr int kFlight = 16;
    u32x4 w8[kFlight];
    auto fetch = [&](int quad, int c0, int by) __attribute__((always_inline)) {
        const int pq = quad / (HD / 4), dq = quad % (HD / 4) * 4;
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const int c = c0 + j * by;
            w8[j] = __builtin_amdgcn_raw_buffer_load_b128(rp, c < it.chunks ? ((row_at(c) * PB + pq) * HD + dq) * 4 : 0x80000000u, 0, kCoherent);
        }
    };
    if (part < parts) fetch(i, part, parts);
    constexpr int TP = 64 / PB * NW;  // threads of a pair (side by side in one wave, or in whole waves' halves)
    constexpr int TW = TP > 64 ? 64 : TP;
    if (tid < PB * TW) {
        const int pp = tid / TW, ii = tid % TW;
        constexpr int kEach = (kMaxChunks + TW - 1) / TW;
        float mv[kEach], lv[kEach];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = ii + j * TW;
            mv[j] = -INFINITY, lv[j] = 0.0f;
            if (c < it.chunks && pp < pairs_here) {
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rm, (row_at(c) * PB + pp) * 8, 0, kCoherent));
                const unsigned w0 = w.x, w1 = w.y;
                mv[j] = __uint_as_float(w0), lv[j] = __uint_as_float(w1);
            }
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) top = fmaxf(top, mv[j]);
#pragma unroll
        for (int x = 1; x < TW; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            mv[j] = weight(mv[j], top);
            sum = fmaf(mv[j], lv[j], sum);
        }
#pragma unroll
        for (int x = 1; x < TW; x *= 2) sum += __shfl_xor(sum, x);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = ii + j * TW;
            if (c < it.chunks) sw[c * PB + pp] = mv[j] * inv;
        }
    }
    __syncthreads();
    auto add = [&](f32x4 &v, int pq, int c0, int by) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const int c = c0 + j * by;
            if (c < it.chunks) v += sw[c * PB + pq] * __builtin_bit_cast(f32x4, w8[j]);
        }
    };
    if (parts > 1) {
        f32x4 v = {0, 0, 0, 0};
        if (part < parts) {
            add(v, p, part, parts);
            for (int c0 = part + kFlight * parts; c0 < it.chunks; c0 += kFlight * parts) {
                fetch(i, c0, parts);
                add(v, p, c0, parts);
            }
            *reinterpret_cast<f32x4 *>(&so[(part * quads + i) * 4]) = v;
        }
        __syncthreads();
        if (part == 0) {
            for (int k = 1; k < parts; ++k) v += *reinterpret_cast<const f32x4 *>(&so[(k * quads + i) * 4]);
            put(v, p, d);
        }
        return;
    }
    for (int q = tid; q < quads; q += NT) {
        const int pq = q / (HD / 4), dq = q % (HD / 4) * 4;
        f32x4 v = {0, 0, 0, 0};
        for (int c0 = 0; c0 < it.chunks; c0 += kFlight) {
            if (q != tid || c0 > 0) fetch(q, c0, 1);
            add(v, pq, c0, 1);
        }
        put(v, pq, dq);
    }
}

template <int HD, bool I8, bool SPLIT, bool GEN, int MODE>
int launch_attn(st_context *ctx, Args a) {
    constexpr int PB = SPLIT ? 8 : 16, NW = 4;
    const int64_t slots = 2 * ctx->num_cus;
    if (int rc = plan_cut(ctx, a, PB, HD, kStep<I8>, kLeast<I8>, slots / a.c.heads)) return rc;
    const size_t lds = (size_t)NW * PB * (HD + 4) * sizeof(float);
    auto kern = attn_kernel<HD, I8, SPLIT, GEN, MODE, NW>;
    if (lds > 32 * 1024)
        ST_HIP(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    st::launch(ctx, kern, dim3((unsigned)a.G, (unsigned)a.c.heads), dim3(64 * NW), lds, a);
    return st::launch_check("attn_kernel");
}

// What the host knows of the lengths is the tables' width. Where that is far
// over them, as while a conversation is young, the next two rules take long
// caches' forms for short ones. With tables for 32768 tokens and with tables of
// the lengths' own width, 32/8 heads of 128, in us: one sequence of 300 tokens 6.7 and
// 6.3, 8 of up to 1000 14.5 and 13.4, a prompt of 77 rows 13.9 and 5.6, one of
// 300 19.5 and 17.4, 16 rows over 600 17.8 and 11.8.
template <int HD, bool I8, bool SPLIT, bool GEN>
int by_size(st_context *ctx, const Args &a) {
    // A cache that no more than one row block reads, and that is larger than
    // what a cache level keeps between calls: non-temporal loads (31 sequences
    // of 8191 tokens at most 114 -> 104 us; in small caches, which the next call
    // finds in L2 again, they cost 1.2 us of 6.2)
    const int64_t bytes = (int64_t)a.B * a.capacity * a.c.heads * HD * (I8 ? 2 : 4);
    const bool once = !a.q_start && a.group <= (SPLIT ? 8 : 16) && bytes >= (int64_t)96 << 20;
    if (once) return launch_attn<HD, I8, SPLIT, GEN, kOneNt>(ctx, a);
    return a.q_start ? launch_attn<HD, I8, SPLIT, GEN, kRows>(ctx, a) : launch_attn<HD, I8, SPLIT, GEN, kOne>(ctx, a);
}

template <int HD, bool I8>
int by_scores(st_context *ctx, const Args &a, bool split) {
    const bool gen = a.cap > 0.0f || a.slopes;
    if (split) return gen ? by_size<HD, I8, true, true>(ctx, a) : by_size<HD, I8, true, false>(ctx, a);
    return gen ? by_size<HD, I8, false, true>(ctx, a) : by_size<HD, I8, false, false>(ctx, a);
}

template <int HD>
int by_type(st_context *ctx, const Args &a, bool i8, bool split) {
    return i8 ? by_scores<HD, true>(ctx, a, split) : by_scores<HD, false>(ctx, a, split);
}

// f16 rows of prompts go to the kernel with 128 pairs a workgroup, where the
// call can be large enough to fill such workgroups and pay for its second
// launch (the host knows what the tables hold at most, not the lengths). Both
// ways, 32/8 heads of 128, in us, this kernel first: 16 rows over 8192 tokens
// 30.6 and 19.6, over 2048 16.5 and 14, over 600 8.9 and 13; 64 rows over 600
// 11.4 and 15; 512 over 512 24 and 24, 4096 over 4096 674 and 167.
bool use_prompt(const st_context *ctx, const Args &a) {
    return (int64_t)a.T * a.group >= 32 * (int64_t)a.B && (int64_t)a.T * a.group * a.capacity >= 1 << 19;
}

bool act_dtype(int d) { return d == ST_F32 || d == ST_F16; }

}  // namespace

namespace st {
namespace attn {

int plan_cut(st_context *ctx, Args &a, int pb, int hd, int step, int least, int64_t extra) {
    const int64_t rows = std::min<int64_t>(a.B, a.T) + (int64_t)a.T * a.group / pb + 1;  // row blocks at most
    if (rows >= kMostRows) return fail(ST_ERR_SHAPE, "st_paged_attention: %d rows", a.T);
    const int heads = a.c.heads;
    const int64_t most_chunks = std::min<int64_t>(kMaxChunks, (a.capacity / step + 1 + least - 1) / least);
    const size_t item = (size_t)heads * pb * (hd + 2) * sizeof(float);
    extra = std::min(extra, rows * (most_chunks - 1));
    extra = std::min(extra, (int64_t)(std::min<size_t>(ctx->ws_bytes, 0x7FFFFFFF) / item) - rows);
    // (more than that are 8 workgroups a CU without a cut; but one sequence much
    // longer than the others then is one workgroup's work in each head: 96
    // sequences over 32 key heads of 64, one of 30000 tokens and the others of
    // 400, take 105 us, 128 of them 211)
    a.split = extra >= 1 && rows * heads <= kSplitCounters;
    a.rows = (int)rows;
    a.G = (int)(rows + (a.split ? extra : 0));
    a.part = ctx->ws;
    a.part_ml = ctx->ws + (size_t)a.G * heads * pb * hd;
    a.cnt = ctx->split_counters;
    return ST_OK;
}

}  // namespace attn
}  // namespace st

extern "C" int st_paged_attention(st_context *ctx, const st_kv_cache *cache, const void *q, int q_dtype, const int32_t *table,
                                  int table_stride, const int32_t *kv_len, const int32_t *q_start, float scale, float cap,
                                  int window, const float *slopes, const void *gate, int gate_dtype, int64_t gate_stride,
                                  int gate_head_stride, void *out, int out_dtype, int T, int B, int n_heads) {
    const char *const fn = "st_paged_attention";
    Args a{};
    if (!ctx || !q || !table || !kv_len || !out) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (int rc = check_cache(fn, cache, &a.c)) return rc;
    if (!act_dtype(q_dtype) || !act_dtype(out_dtype) || (gate && !act_dtype(gate_dtype)))
        return st::fail(ST_ERR_INVALID, "%s: q_dtype %d, out_dtype %d, gate_dtype %d (f32 or f16)", fn, q_dtype, out_dtype, gate_dtype);
    if (T < 1 || B < 1 || B > (1 << 20) || T > (1 << 24)) return st::fail(ST_ERR_SHAPE, "%s: T=%d, B=%d", fn, T, B);
    if (!q_start && T != B) return st::fail(ST_ERR_SHAPE, "%s: without q_start every sequence has one row: T=%d, B=%d", fn, T, B);
    if (n_heads < 1 || n_heads % a.c.heads || n_heads / a.c.heads > 64)
        return st::fail(ST_ERR_SHAPE, "%s: %d heads over %d key heads (a multiple, at most 64 times)", fn, n_heads, a.c.heads);
    if (table_stride < 1 || ((int64_t)table_stride << a.c.page_shift) > 0x7FFFFF00)
        return st::fail(ST_ERR_SHAPE, "%s: table rows of %d pages (positions are 32-bit)", fn, table_stride);
    if (window < 0 || !(cap >= 0.0f) || !(scale > 0.0f)) return st::fail(ST_ERR_INVALID, "%s: scale %g, cap %g, window %d", fn, scale, cap, window);
    const int hd = cache->head_dim;
    if (!st::aligned16(q) || !st::aligned16(out) || !st::aligned16(gate)) return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
    if (gate) {
        if (gate_head_stride < hd || gate_stride < (int64_t)(n_heads - 1) * gate_head_stride + hd)
            return st::fail(ST_ERR_SHAPE, "%s: a head's or token's gates overlap the next one's", fn);
        if (gate_stride % 8 || gate_head_stride % 8) return st::fail(ST_ERR_ALIGN, "%s: gate strides must be multiples of 8", fn);
    }
    a.q = q, a.gate = gate, a.out = out, a.table = table, a.kv_len = kv_len, a.q_start = q_start, a.slopes = slopes;
    a.gate_stride = gate_stride, a.gate_head_stride = gate_head_stride;
    a.table_stride = table_stride, a.capacity = table_stride << a.c.page_shift;
    a.T = T, a.B = B, a.n_heads = n_heads, a.group = n_heads / a.c.heads;
    a.group_shift = (a.group & (a.group - 1)) == 0 ? __builtin_ctz(a.group) : -1;
    a.window = std::min(window, 1 << 30), a.scale = scale;
    // (a cap beyond 2^100 leaves scores as they are; one below f32's normal
    // numbers, whose reciprocal is infinite, is as good as the least of them)
    a.cap = cap > 0x1p100f ? 0.0f : cap > 0.0f ? std::max(cap, 0x1p-126f) : 0.0f;
    a.q_f32 = q_dtype == ST_F32, a.gate_f32 = gate_dtype == ST_F32, a.out_f32 = out_dtype == ST_F32;
    const bool i8 = cache->dtype == ST_I8, split = a.q_f32 || a.out_f32;
    if (!split && use_prompt(ctx, a)) return prompt_attention(ctx, a, i8, hd);
    return hd == 64 ? by_type<64>(ctx, a, i8, split) : hd == 128 ? by_type<128>(ctx, a, i8, split) : by_type<256>(ctx, a, i8, split);
}
