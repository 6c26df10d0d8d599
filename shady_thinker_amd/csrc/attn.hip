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
//  * A wave takes 32 keys (two tiles) at a time. The scores' lanes are the
//    columns and each lane's eight keys are those whose values one piece of
//    the cache's value tiles holds: the weights go from the first product to
//    the second in the registers where they are, and K and V go from HBM to
//    registers in 16-byte (8-byte) pieces, with no LDS.
//  * Bound by HBM (4 matrix cycles per KiB of the cache are 4% of its time),
//    that is by how many loads are in flight: the next step's are issued
//    before this step's are used.
//  * The cut: every sequence's keys go in chunks of C steps to workgroups of
//    four waves, C the smallest with which all fit the grid, found by each
//    workgroup from the lengths on the device (so that a captured graph stays
//    right, and batches of mixed lengths even, as they grow). The last chunk
//    of a (row block, key head) to count in joins them in order: the counter
//    protocol of the split-K kernels (see qmv_kernel.hpp on its visibility).
#include "attn.hpp"

#include <algorithm>
#include <climits>

namespace {

using namespace st::attn;

constexpr int kWaves = 4;
constexpr int kStep = 32;  // keys of a step of one wave
constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit buffer data (gfx9-class)
constexpr int kCoherent = 1 | 16;       // sc0 sc1: write through / read past this XCD's L2
constexpr float kShift = 14.0f;         // weights are held times 2^14: f16 keeps them normal down to 2^-28

template <int HD, bool I8, bool SPLIT>
struct Frag {
    static constexpr int NS = HD / 32, ND = HD / 16;
    using P = std::conditional_t<I8, u32x2, half8>;  // a piece: eight elements
    P k[2][NS], v[ND];
    f32x4 ks[I8 ? 2 : 1], vs[I8 ? 2 : 1];  // the lane's eight keys' scales
};

__device__ __forceinline__ half8 as_half8(half8 v) { return v; }
__device__ __forceinline__ half8 as_half8(u32x2 v) { return i8_to_half8(v); }

__device__ __forceinline__ float max_q4(float v) {  // over the four lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float half_turn(float v) {  // the lane eight columns on
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, true));
}

// Two steps' pieces in registers (256 dims: one, two do not fit).
template <int HD, bool I8>
constexpr bool kTwo = HD <= 128;

template <int HD, bool I8, bool SPLIT>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_kernel(Args a) {
    constexpr int PB = SPLIT ? 8 : 16;  // pairs of a block
    constexpr int NS = HD / 32, ND = HD / 16, kRow = HD + 4;
    using F = Frag<HD, I8, SPLIT>;
    using E = std::conditional_t<I8, signed char, _Float16>;
    extern __shared__ __align__(16) float so[];  // [kWaves][PB][kRow]
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    __shared__ float sw[kMaxChunks * PB];
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int col = lane & 15, q4 = lane >> 4;
    const int h = blockIdx.y;
    Item it;
    if (!find_item<PB, kStep, kWaves>(a, (int)blockIdx.x, it)) return;
    it = scalars(it);

    // ---- this lane's column: a (row, head) pair
    const int npair = it.s.q * a.group;
    const int pair = it.rb * PB + (SPLIT ? col & 7 : col);
    const bool real = pair < npair;
    const int tok = real ? pair / a.group : 0, head = h * a.group + (real ? pair % a.group : 0);
    const int p0 = it.s.kv - it.s.q;  // position of the sequence's first row
    const int pos = real ? p0 + tok : -1;
    const int low = a.window ? max(pos - a.window + 1, 0) : 0;  // keys low .. pos are visible
    // (uniform: the block's first and last rows' positions)
    const int pmin = p0 + scalar(it.rb * PB / a.group), pmax = p0 + scalar((min(it.rb * PB + PB, npair) - 1) / a.group);
    const int wmax = a.window ? pmax - a.window + 1 : 0;  // from here on a key is in every row's window
    const int wmin = a.window ? pmin - a.window + 1 : 0;  // before this it is in none's
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;

    half8 qf[NS];
    float qs = a.scale;  // scores are matrix sums times qs
    {
        float x[NS][8];
        const int64_t at = ((int64_t)(it.s.q0 + tok) * a.n_heads + head) * HD + q4 * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (a.q_f32) {
                const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.q) + at + 32 * s);
                const f32x4 u = p[0], w = p[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[s][i] = u[i], x[s][4 + i] = w[i];
            } else {
                const half8 u = *reinterpret_cast<const half8 *>(static_cast<const _Float16 *>(a.q) + at + 32 * s);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[s][i] = (float)u[i];
            }
        }
        if constexpr (SPLIT) {
            float m = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[s][i]));
            m = max_q4(m);
            int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
            e = max(e, -126);
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = ldexpf(x[s][i], -e);
                    const _Float16 hi = (_Float16)v;
                    qf[s][i] = col < 8 ? hi : (_Float16)(v - (float)hi);
                }
            qs = ldexpf(qs, e);
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) qf[s][i] = (_Float16)x[s][i];
        }
        if (!real) {
#pragma unroll
            for (int s = 0; s < NS; ++s) qf[s] = half8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    }

    // ---- the chunk's steps: this wave's are s0 + wave, + kWaves, ...
    const int key0 = first_key<kStep>(a, it.s);
    const int tile0 = key0 / 16, tiles = (it.s.kv + 15) / 16;  // tiles that hold a token
    const int tsh = a.c.tiles_shift();
    const int32_t *const table = a.table + (int64_t)it.b * a.table_stride;
    // A tile's page (-1: none to read), through the scalar cache: its waits
    // are not those of the pieces in flight.
    const auto *const pages = (const __attribute__((address_space(4))) int32_t *)table;
    auto page_of = [&](int t) __attribute__((always_inline)) {
        const int p = pages[max(min(t, tiles - 1), 0) >> tsh];
        return t < tiles && (unsigned)p < (unsigned)a.c.num_pages ? p : -1;
    };
    int next0 = page_of(tile0 + 2 * (it.s0 + wave)), next1 = page_of(tile0 + 2 * (it.s0 + wave) + 1);  // of the step to load
    // (this lane's pieces: K row r = lane % 16 is place r % 8 (+ 8) of tile
    // r / 8, V piece half q4 % 2 of tile q4 / 2)
    const int k_off = q4 * 128 + (col & 7) * 8, v_off = ((q4 & 1) * HD + col) * 8;
    auto load = [&](F &f, int step, bool &ok0, bool &ok1) __attribute__((always_inline)) {
        const bool in = step < it.s1;
        const int t = tile0 + 2 * step;
        const int p0 = next0, p1 = next1;
        next0 = page_of(t + 2 * kWaves), next1 = page_of(t + 2 * kWaves + 1);
        ok0 = in && p0 >= 0, ok1 = in && p1 >= 0;
        // a tile that is not read: every lane at the cache's first piece
        const int64_t e0 = ok0 ? a.c.tile(p0, h, t & ((1 << tsh) - 1)) * (16 * HD) : 0;
        const int64_t e1 = ok1 ? a.c.tile(p1, h, (t + 1) & ((1 << tsh) - 1)) * (16 * HD) : 0;
        const bool kt = col >= 8, vt = q4 >= 2;
        const E *kp = static_cast<const E *>(a.c.k) + (kt ? e1 : e0) + ((kt ? ok1 : ok0) ? k_off : 0);
        const E *vp = static_cast<const E *>(a.c.v) + (vt ? e1 : e0) + ((vt ? ok1 : ok0) ? v_off : 0);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                f.k[half][s] = *reinterpret_cast<const typename F::P *>(kp + 512 * s + 64 * half);
#pragma unroll
        for (int d = 0; d < ND; ++d) f.v[d] = *reinterpret_cast<const typename F::P *>(vp + 128 * d);
        if constexpr (I8) {
            const int64_t s0 = ok0 ? a.c.scale(p0, h, (t * 16) & ((1 << a.c.page_shift) - 1)) : 0;
            const int64_t s1 = ok1 ? a.c.scale(p1, h, (t * 16 + 16) & ((1 << a.c.page_shift) - 1)) : 0;
            const int64_t at = (vt ? s1 : s0) + (q4 & 1) * 4;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f.ks[half] = *reinterpret_cast<const f32x4 *>(a.c.k_scale + at + 8 * half);
                f.vs[half] = *reinterpret_cast<const f32x4 *>(a.c.v_scale + at + 8 * half);
            }
        }
    };

    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    int ve = -126;  // int8: weights are held times their value scale over 2^ve

    auto compute = [&](F &f, int step, bool ok0, bool ok1) __attribute__((always_inline)) {
        const int kb = key0 + 32 * step;
        f32x4 s4[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            s4[half] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s)
                s4[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(f.k[half][s]), qf[s], s4[half], 0, 0, 0);
        }
        // this lane's keys: key(j) for weight j of the second product
        const int kl = kb + 16 * (q4 >> 1) + 4 * (q4 & 1);
        auto key = [&](int j) { return kl + (j & 3) + 8 * (j >> 2); };
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = s4[j >> 2][j & 3];
            if constexpr (SPLIT) v += half_turn(v);
            if constexpr (I8) v *= f.ks[j >> 2][j & 3];
            x[j] = v * qs;
        }
        if (a.cap > 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = a.cap * tanhf(x[j] / a.cap);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= kLog2e;
        if (a.slopes) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fmaf(slope, (float)(key(j) - pos), x[j]);
        }
        const bool full = ok0 && ok1 && kb + 31 <= pmin && kb >= wmax;  // (uniform) every key for every row
        unsigned seen = 0xFF;
        if (!full) {
            const bool ok = q4 >= 2 ? ok1 : ok0;
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int kj = key(j);
                if (ok && kj >= low && kj <= pos) seen |= 1u << j;
                x[j] = seen >> j & 1 ? x[j] : -INFINITY;
            }
            // values no row of the block sees may be anything
            const bool none0 = !ok;
            if constexpr (!I8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int kj = key(j);
                    const bool any = !none0 && kj <= pmax && kj >= wmin;
#pragma unroll
                    for (int d = 0; d < ND; ++d) f.v[d][j] = any ? f.v[d][j] : (_Float16)0.0f;
                }
            }
        }
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, x[j]);
        const float mn = fmaxf(m, max_q4(mx));
        const float base = mn == -INFINITY ? 0.0f : mn;
        float alpha = exp2_(m - base);  // (0 before the first visible key)
        m = mn;
        float p[8], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = exp2_(x[j] - base + kShift);
            sum += p[j];
        }
        l = fmaf(l, alpha, sum);
        if constexpr (I8) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, seen >> j & 1 ? f.vs[j >> 2][j & 3] : 0.0f);
#pragma unroll
            for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
            const int e = max(ve, (int)((__float_as_uint(top) >> 23) & 255) - 126);  // top / 2^e < 1
            alpha = ldexpf(alpha, ve - e);
            ve = e;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = seen >> j & 1 ? p[j] * ldexpf(f.vs[j >> 2][j & 3], -ve) : 0.0f;
        }
        if (__ballot(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
        half8 pf;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const _Float16 hi = (_Float16)p[j];
            pf[j] = hi;
            if constexpr (SPLIT) pf[j] = col < 8 ? hi : (_Float16)(p[j] - (float)hi);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(f.v[d]), pf, o[d], 0, 0, 0);
    };

    if constexpr (kTwo<HD, I8>) {
        int step = it.s0 + wave;
        F fa, fb;
        bool a0, a1, b0, b1;
        load(fa, step, a0, a1);
        while (step < it.s1) {
            load(fb, step + kWaves, b0, b1);
            __builtin_amdgcn_sched_barrier(0);
            compute(fa, step, a0, a1);
            step += kWaves;
            if (step >= it.s1) break;
            load(fa, step + kWaves, a0, a1);
            __builtin_amdgcn_sched_barrier(0);
            compute(fb, step, b0, b1);
            step += kWaves;
        }
    } else {
        F f;
        bool ok0, ok1;
        for (int step = it.s0 + wave; step < it.s1; step += kWaves) {
            load(f, step, ok0, ok1);
            compute(f, step, ok0, ok1);
        }
    }

    // ---- the four waves meet in LDS
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (I8) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] = ldexpf(o[d][i], ve);
    }
    if constexpr (SPLIT) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] += half_turn(o[d][i]);
    }
    if (col < PB) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *reinterpret_cast<f32x4 *>(&so[(wave * PB + col) * kRow + d * 16 + q4 * 4]) = o[d];
        if (q4 == 0) sm[wave][col] = m, sl[wave][col] = l;
    }
    __syncthreads();
    constexpr int kQuads = PB * HD / 4;
    const int pairs_here = min(PB, npair - it.rb * PB);
    const int row_id = (int)blockIdx.x * a.c.heads + h;
    auto weight = [](float mw, float top) { return mw == -INFINITY ? 0.0f : exp2_(mw - top); };
    auto row_of = [&](int p, int &row, int &hd) {
        const int g = it.rb * PB + p;
        row = it.s.q0 + g / a.group, hd = h * a.group + g % a.group;
    };
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void *)a.part, (short)0, a.G * a.c.heads * PB * HD * 4, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rm = __builtin_amdgcn_make_buffer_rsrc((void *)a.part_ml, (short)0, a.G * a.c.heads * PB * 8, kRsrcWord3);
    for (int i = tid; i < kQuads; i += 64 * kWaves) {
        const int p = i / (HD / 4), d = i % (HD / 4) * 4;
        if (p >= pairs_here) continue;
        float top = sm[0][p];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][p]);
        f32x4 v = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = weight(sm[w][p], top);
            sum = fmaf(f, sl[w][p], sum);
            v += f * *reinterpret_cast<const f32x4 *>(&so[(w * PB + p) * kRow + d]);
        }
        if (it.chunks == 1) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (a row that sees nothing is zero)
            int row, hd;
            row_of(p, row, hd);
            store_out(a, v * inv, row, hd, d, HD);
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rp, ((row_id * PB + p) * HD + d) * 4, 0, kCoherent);
            if (d == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(top), __float_as_uint(sum)}, rm, (row_id * PB + p) * 8, 0,
                                                      kCoherent);
        }
    }
    if (it.chunks == 1) return;

    // ---- the chunks meet: the last one to count in joins them in order
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
    constexpr int TP = 64 * kWaves / PB;  // threads of a pair (of one wave)
    {
        const int p = tid / TP, i = tid % TP;
        constexpr int kEach = (kMaxChunks + TP - 1) / TP;
        float mv[kEach], lv[kEach];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = i + j * TP;
            mv[j] = -INFINITY, lv[j] = 0.0f;
            if (c < it.chunks && p < pairs_here) {
                const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rm, (row_at(c) * PB + p) * 8, 0, kCoherent));
                const unsigned w0 = w.x, w1 = w.y;
                mv[j] = __uint_as_float(w0), lv[j] = __uint_as_float(w1);
            }
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) top = fmaxf(top, mv[j]);
#pragma unroll
        for (int d = 1; d < TP; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            mv[j] = weight(mv[j], top);
            sum = fmaf(mv[j], lv[j], sum);
        }
#pragma unroll
        for (int d = 1; d < TP; d *= 2) sum += __shfl_xor(sum, d);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int c = i + j * TP;
            if (c < it.chunks) sw[c * PB + p] = mv[j] * inv;
        }
    }
    __syncthreads();
    for (int i = tid; i < kQuads; i += 64 * kWaves) {
        const int p = i / (HD / 4), d = i % (HD / 4) * 4;
        if (p >= pairs_here) continue;
        f32x4 v = {0, 0, 0, 0};
        for (int c0 = 0; c0 < it.chunks; c0 += 8) {
            u32x4 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = __builtin_amdgcn_raw_buffer_load_b128(rp, c0 + j < it.chunks ? ((row_at(c0 + j) * PB + p) * HD + d) * 4 : 0x80000000u, 0,
                                                             kCoherent);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < it.chunks) v += sw[(c0 + j) * PB + p] * __builtin_bit_cast(f32x4, w[j]);
        }
        int row, hd;
        row_of(p, row, hd);
        store_out(a, v, row, hd, d, HD);
    }
}

template <int HD, bool I8, bool SPLIT>
int launch_attn(st_context *ctx, Args a) {
    constexpr int PB = SPLIT ? 8 : 16;
    if (int rc = plan_cut(ctx, a, PB, HD, kStep, kWaves, 2 * ctx->num_cus / a.c.heads)) return rc;
    const int heads = a.c.heads;
    const size_t lds = (size_t)kWaves * PB * (HD + 4) * sizeof(float);
    auto kern = attn_kernel<HD, I8, SPLIT>;
    if (lds > 48 * 1024)
        ST_HIP(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    st::launch(ctx, kern, dim3((unsigned)a.G, (unsigned)heads), dim3(64 * kWaves), lds, a);
    return st::launch_check("attn_kernel");
}

template <int HD>
int by_type(st_context *ctx, const Args &a, bool i8, bool split) {
    if (i8) return split ? launch_attn<HD, true, true>(ctx, a) : launch_attn<HD, true, false>(ctx, a);
    return split ? launch_attn<HD, false, true>(ctx, a) : launch_attn<HD, false, false>(ctx, a);
}

// f16 rows of prompts go to the kernel with 128 pairs a workgroup.
bool use_prompt(const st_context *ctx, const Args &a) {
    return (int64_t)a.T * a.group >= 32 * (int64_t)a.B;
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
    a.window = std::min(window, 1 << 30), a.scale = scale, a.cap = cap;
    a.q_f32 = q_dtype == ST_F32, a.gate_f32 = gate_dtype == ST_F32, a.out_f32 = out_dtype == ST_F32;
    const bool i8 = cache->dtype == ST_I8, split = a.q_f32 || a.out_f32;
    if (!split && use_prompt(ctx, a)) return prompt_attention(ctx, a, i8, hd);
    return hd == 64 ? by_type<64>(ctx, a, i8, split) : hd == 128 ? by_type<128>(ctx, a, i8, split) : by_type<256>(ctx, a, i8, split);
}
