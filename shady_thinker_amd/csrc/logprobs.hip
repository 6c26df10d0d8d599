// Log probabilities of given tokens, with their rank, the entropy and the top
// alternatives of rows of logits (st_token_logprobs), in one pass. The
// reference reads the logits back and samples on the CPU (src/model.rs:836-968).
//
// Of a row x with maximum m and S = sum exp(x - m) over all but one maximum:
//   log p_j = (x_j - m) - log1p(S),   H = log1p(S) - T / (1 + S),
//   T = sum exp(x - m) (x - m)
// (leaving the maximum's own 1 out of the sum keeps a likely token's small
// -log p exact to f32's last bits, not to 2^-24).
// Bound by HBM (each logit once). A workgroup takes a chunk of a row into
// registers; each wave has (m, S, T) of its own and they meet in LDS. The top
// tokens: the k-th of the threads' largest logits is a lower bound of the
// chunk's k-th largest, so only logits from there on (k and a few more) are
// candidates; these are ranked among each other by value, then index. The
// last chunk of a row to count in joins the chunks (the counter protocol of the
// split-K kernels, see qmv_kernel.hpp), its top tokens found in the same way
// among the chunks'.
// 512 rows of 151936 f32, top 5: 72 us (4.3 TB/s; 56 without top tokens, 5.5
// TB/s; f16 logits 71 and 50); one row, top 20: 12.4 us (top 1 8.6, none 5.8: a
// selection's three barriers and ranking are 3 us, in the chunks and again in
// the join). Rows of which all but 1000 logits are -inf: chunks with nothing
// else are one round a token (below), one row, top 20, 30 us, top 32 38; 512
// rows, top 5, 100, top 32 160.
#include "common.hpp"

#include <algorithm>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTop = 32;
constexpr int kMergeEach = 17;                        // of the joined chunks' top tokens, per thread
constexpr int kMaxChunks = kMergeEach * kThreads / kMaxTop;  // of a row: 2^20 logits in chunks of 8192, and one for its start
constexpr int kCandidates = 512;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit buffer data (gfx9-class)
constexpr int kNt = 2;                  // non-temporal: a logit is read once
constexpr int kCoherent = 1 | 16;       // sc0 sc1: write through / read past this XCD's L2

struct Args {
    const void *x;
    int64_t stride;
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float *top_logprobs;
    int V, top, chunks;
    float *part;       // [row][chunk] of part_words(top)
    unsigned *cnt;     // spread_counter(row)
};

// A chunk's partial result: m, S, T, rank, then `top` keys of two words.
__host__ __device__ constexpr int part_words(int top) { return 4 + 2 * top; }

// Order of (value, index) as an unsigned: larger value first, then lower
// index. Equal zeros of both signs.
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __float_as_uint(v + 0.0f);
    return (int)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float((int)o < 0 ? o & 0x7FFFFFFFu : ~o); }

struct Sums {
    float m, s, t;  // t in units of log 2
};

// The sums of two disjoint parts (m -inf: nothing in it).
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    if (b.m > a.m) {
        const Sums c = a;
        a = b, b = c;
    }
    if (b.m == -INFINITY) return a;
    const float d = (b.m - a.m) * kLog2e, f = __builtin_amdgcn_exp2f(d), w = f * (1.0f + b.s);
    a.s += w;
    a.t += f * b.t + (w > 0.0f ? w * d : 0.0f);
    return a;
}

// Reductions over a wave: the four rows of 16 lanes by DPP, then their first
// lanes as scalars (every lane gets the result).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float lane_of(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0x121>(v)), v = fmaxf(v, dpp<0x122>(v)), v = fmaxf(v, dpp<0x124>(v)), v = fmaxf(v, dpp<0x128>(v));
    return fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0x121>(v), v += dpp<0x122>(v), v += dpp<0x124>(v), v += dpp<0x128>(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// The top `k` of a workgroup's elements (value x[j], not NaN, index idx(j),
// present where idx(j) >= 0, -inf where not) as keys in order in `out`; fewer
// than k present: keys 0 after them. `mine` is the largest x[j] of the thread.
// lists: threads 32 c .. 32 c + k - 1 hold ordered lists' first .. k-th elements
// (the k-th of any is a bound that k threads reach).
struct TopShared {
    unsigned long long cand[kCandidates];
    unsigned long long best[kWaves];
    unsigned mine[kThreads];
    unsigned bound;
    int n;
};
template <int E, typename Idx>
__device__ __forceinline__ void top_of_block(const float (&x)[E], float mine, Idx idx, int k, TopShared &sh, unsigned long long *out,
                                             bool lists) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    sh.mine[tid] = order_of(mine);
    if (tid == 0) sh.n = 0;
    if (tid < k) out[tid] = 0;
    __syncthreads();
    if (wave == 0) {
        // bisection between the smallest and the largest, until k threads
        // reach the bound and few more (bit by bit took three times as many
        // turns, of 60-100 cycles each)
        const u32x4 o = *reinterpret_cast<const u32x4 *>(&sh.mine[4 * lane]);
        unsigned bound = min(min(o.x, o.y), min(o.z, o.w)), over = max(max(o.x, o.y), max(o.z, o.w));
        if (lists) bound = sh.mine[32 * (lane & 7) + k - 1];
        bound = lists ? order_of(wave_max(value_of(bound))) : order_of(-wave_max(-value_of(bound)));
        over = order_of(wave_max(value_of(over)));
        if (__popcll(__ballot(o.x >= over)) + __popcll(__ballot(o.y >= over)) + __popcll(__ballot(o.z >= over)) +
                __popcll(__ballot(o.w >= over)) >=
            k)
            bound = over;
#pragma unroll 1
        while (over - bound > 1) {
            const unsigned b = bound + (over - bound) / 2;
            const int n = __popcll(__ballot(o.x >= b)) + __popcll(__ballot(o.y >= b)) + __popcll(__ballot(o.z >= b)) +
                          __popcll(__ballot(o.w >= b));
            if (n >= k) {
                bound = b;
                if (n <= k + k / 4 + 2) break;
            } else {
                over = b;
            }
        }
        if (lane == 0) sh.bound = bound;
    }
    __syncthreads();
    const unsigned bound = sh.bound;
    const float least = bound <= order_of(-INFINITY) ? -INFINITY : value_of(bound);
    if (__ballot(mine >= least)) {
        int hits = 0;  // (one LDS atomic's wait, not one for each j)
#pragma unroll
        for (int j = 0; j < E; ++j) hits += x[j] >= least;
        int at = hits ? atomicAdd(&sh.n, hits) : 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (x[j] >= least) {
                const int i = idx(j);
                if (at < kCandidates) sh.cand[at] = i >= 0 ? (unsigned long long)order_of(x[j]) << 32 | ~(unsigned)i : 0ull;
                ++at;
            }
        }
    }
    __syncthreads();
    const int n = sh.n;
    if (n <= kCandidates) {
        for (int c = tid; c < n; c += kThreads) {
            const unsigned long long key = sh.cand[c];
            int r = 0, i = 0;
            for (; i + 8 <= n; i += 8) {
#pragma unroll
                for (int u = 0; u < 8; ++u) r += sh.cand[i + u] > key;
            }
            for (; i < n; ++i) r += sh.cand[i] > key;
            if (r < k && key) out[r] = key;
        }
        __syncthreads();
        return;
    }
    // very many equal values (rows of few distinct logits): one at a time
    unsigned long long last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < k; ++r) {
        unsigned long long best = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int i = idx(j);
            const unsigned long long key = i >= 0 ? (unsigned long long)order_of(x[j]) << 32 | ~(unsigned)i : 0ull;
            if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const unsigned long long o = __shfl_xor(best, d);
            best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) sh.best[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        if (tid == 0) out[r] = best;
        last = best;
    }
    __syncthreads();
}

template <bool F16, int E>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
    constexpr int VEC = F16 ? 8 : 4, NL = E / VEC;
    using X = std::conditional_t<F16, _Float16, float>;
    __shared__ __align__(16) TopShared sh;
    __shared__ Sums s_sums[kWaves];
    __shared__ int s_rank[kWaves];
    __shared__ unsigned long long s_top[kMaxTop];
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = blockIdx.y, chunk = blockIdx.x;
    const X *const xr = static_cast<const X *>(a.x) + row * a.stride;
    // (an f16 row that starts inside a dword: from that dword on)
    const int skew = F16 ? (int)(reinterpret_cast<uintptr_t>(xr) >> 1 & 1) : 0;
    const int begin = chunk * (kThreads * E) - skew;  // index of the chunk's first element
    const int first = begin + tid * VEC;
    const bool whole = begin >= 0 && begin + kThreads * E <= a.V;  // (uniform)
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool known = token >= 0 && token < a.V;
    float x[E];
    // The dwords that hold the row; past them nothing is read.
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void *)(xr - skew), (short)0,
                                                                        (int)((a.V + skew) * sizeof(X) + 3) & ~3, kRsrcWord3);
    u32x4 raw[NL];
#pragma unroll
    for (int l = 0; l < NL; ++l)
        raw[l] = __builtin_amdgcn_raw_buffer_load_b128(rx, (chunk * (kThreads * E) + (l * kThreads + tid) * VEC) * (int)sizeof(X), 0, kNt);
#pragma unroll
    for (int l = 0; l < NL; ++l) {
        if constexpr (F16) {
            const half8 v = __builtin_bit_cast(half8, raw[l]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[l * VEC + i] = (float)v[i];
        } else {
            const f32x4 v = __builtin_bit_cast(f32x4, raw[l]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[l * VEC + i] = v[i];
        }
    }
    if (!whole) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int i = first + j / VEC * (kThreads * VEC) + j % VEC;
            x[j] = i >= 0 && i < a.V ? x[j] : -INFINITY;
        }
    }
    const float xt = known ? (float)xr[token] : 0.0f;
    auto idx = [&](int j) {
        const int i = first + j / VEC * (kThreads * VEC) + j % VEC;
        return i < a.V ? i : -1;
    };

    // ---- this wave's sums
    auto largest = [&]() {
        float m = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) m = fmaxf(m, x[j]);
        return m;
    };
    float mine = largest();
    Sums w{wave_max(mine), 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = (x[j] - w.m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
        w.s += e;
        w.t = fmaf(e, d, w.t);
    }
    w.s = wave_sum(w.s), w.t = wave_sum(w.t);
    if (w.s >= 2.0f && w.s < INFINITY && w.t > -INFINITY) {
        w.s -= 1.0f;
    } else {
        // A maximum that outweighs the rest (its 1 stays out of the sum), a
        // -inf or absent element (0 times -inf above), an infinity, a NaN
        // (which orders as +inf: the row's results are NaN either way).
        int equal = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = x[j] != x[j] ? INFINITY : x[j];
        mine = largest();
        w = Sums{wave_max(mine), 0.0f, 0.0f};
        const float base = w.m == -INFINITY ? 0.0f : w.m;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool top = x[j] == w.m;
            equal += __popcll(__ballot(top));
            const float d = fmaxf((x[j] - base) * kLog2e, -300.0f), e = top ? 0.0f : __builtin_amdgcn_exp2f(d);
            w.s += e;
            w.t = fmaf(e, d, w.t);
        }
        w.s = wave_sum(w.s) + (float)(equal - 1), w.t = wave_sum(w.t);
    }
    int ahead = 0;
    if (a.rank && known) {
        const float xk = xt != xt ? INFINITY : xt;
        if (whole && token >= begin + kThreads * E) {  // (uniform: as the next)
#pragma unroll
            for (int j = 0; j < E; ++j) ahead += __popcll(__ballot(x[j] >= xk));
        } else if (whole && token < begin) {
#pragma unroll
            for (int j = 0; j < E; ++j) ahead += __popcll(__ballot(x[j] > xk));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int i = idx(j);
                ahead += __popcll(__ballot(i >= 0 && (x[j] > xk || (x[j] == xk && i < token))));
            }
        }
    }
    if (lane == 0) s_sums[wave] = w, s_rank[wave] = ahead;
    if (a.top > 0)
        top_of_block(x, mine, idx, a.top, sh, s_top, false);
    else
        __syncthreads();
    Sums sum = s_sums[0];
    ahead = s_rank[0];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) sum = join(sum, s_sums[k]), ahead += s_rank[k];

    // ---- the row's chunks meet
    if (a.chunks > 1) {
        const int words = part_words(a.top);
        const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(
            (void *)(a.part + (size_t)row * a.chunks * words), (short)0, a.chunks * words * 4, kRsrcWord3);
        const int at = chunk * words * 4;
        if (tid == 0)
            __builtin_amdgcn_raw_buffer_store_b128(
                u32x4{__float_as_uint(sum.m), __float_as_uint(sum.s), __float_as_uint(sum.t), (unsigned)ahead}, rp, at, 0, kCoherent);
        if (tid < a.top)
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{(unsigned)s_top[tid], (unsigned)(s_top[tid] >> 32)}, rp, at + 16 + tid * 8, 0,
                                                  kCoherent);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part is in memory
        __syncthreads();
        if (tid == 0) {
            unsigned *const cnt = a.cnt + st::spread_counter(row);
            const unsigned done = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
            s_last = done == (unsigned)a.chunks - 1;
            if (s_last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        }
        __syncthreads();
        if (!s_last) return;
        // thread (p, c): key p of chunks c, c + 8, ... and the sums of chunks
        // tid (at most kMaxChunks < 256)
        constexpr unsigned kNone = 0x80000000u;  // past the buffer: reads 0
        const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      rp, tid < a.chunks ? (unsigned)(tid * words * 4) : kNone, 0, kCoherent));
        u32x2 kv[kMergeEach];
#pragma unroll
        for (int j = 0; j < kMergeEach; ++j) {
            const int c = (tid >> 5) + 8 * j, p = tid & 31;
            kv[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                  rp, c < a.chunks && p < a.top ? (unsigned)((c * words + 4 + 2 * p) * 4) : kNone, 0, kCoherent));
        }
        const unsigned v0 = v.x, v1 = v.y, v2 = v.z, v3 = v.w;
        Sums g{tid < a.chunks ? __uint_as_float(v0) : -INFINITY, __uint_as_float(v1), __uint_as_float(v2)};
        int r = (int)v3;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            g = join(g, Sums{__shfl_xor(g.m, d), __shfl_xor(g.s, d), __shfl_xor(g.t, d)});
            r += __shfl_xor(r, d);
        }
        __syncthreads();
        if (lane == 0) s_sums[wave] = g, s_rank[wave] = r;
        float kx[kMergeEach];
        int ki[kMergeEach];
        mine = -INFINITY;
#pragma unroll
        for (int j = 0; j < kMergeEach; ++j) {
            const unsigned lo = kv[j].x, hi = kv[j].y;
            kx[j] = hi ? value_of(hi) : -INFINITY;
            ki[j] = hi ? (int)~lo : -1;
            mine = fmaxf(mine, kx[j]);
        }
        if (a.top > 0)
            top_of_block(kx, mine, [&](int j) { return ki[j]; }, a.top, sh, s_top, true);
        else
            __syncthreads();
        sum = s_sums[0], ahead = s_rank[0];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) sum = join(sum, s_sums[k]), ahead += s_rank[k];
    }

    // ---- the row's results
    const bool finite = fabsf(sum.m) < INFINITY;  // (an infinity, a NaN, or nothing but -inf: no distribution)
    const float base = finite ? sum.m : __builtin_nanf(""), logs = log1pf(sum.s);
    if (tid == 0) {
        if (a.logprob) a.logprob[row] = known ? (xt - base) - logs : __builtin_nanf("");
        if (a.rank) a.rank[row] = known ? ahead : -1;
        if (a.entropy) a.entropy[row] = finite ? logs - sum.t * kLn2 / (1.0f + sum.s) : __builtin_nanf("");
    }
    if (tid < a.top) {
        const unsigned long long key = s_top[tid];
        a.top_ids[(int64_t)row * a.top + tid] = (int32_t)~(unsigned)key;
        if (a.top_logprobs) a.top_logprobs[(int64_t)row * a.top + tid] = (value_of((unsigned)(key >> 32)) - base) - logs;
    }
}

template <bool F16, int E>
int launch_rows(st_context *ctx, Args a, int M) {
    a.chunks = (a.V + (F16 ? 1 : 0) + kThreads * E - 1) / (kThreads * E);  // (an f16 row may start inside a dword)
    const size_t row = (size_t)a.chunks * part_words(a.top) * sizeof(float);
    const int most = a.chunks == 1 ? 65535 : (int)std::min<size_t>(st::kSplitCounters, ctx->ws_bytes / row);
    if (most < 1) return st::fail(ST_ERR_WORKSPACE, "st_token_logprobs: a row of %d logits needs %zu bytes of workspace", a.V, row);
    a.part = ctx->ws;
    a.cnt = ctx->split_counters;
    const int size = F16 ? 2 : 4;
    for (int m = 0; m < M; m += most) {
        Args b = a;
        const int n = std::min(most, M - m);
        b.x = static_cast<const char *>(a.x) + (int64_t)m * a.stride * size;
        if (a.tokens) b.tokens = a.tokens + m;
        if (a.logprob) b.logprob = a.logprob + m;
        if (a.entropy) b.entropy = a.entropy + m;
        if (a.rank) b.rank = a.rank + m;
        if (a.top_ids) b.top_ids = a.top_ids + (int64_t)m * a.top;
        if (a.top_logprobs) b.top_logprobs = a.top_logprobs + (int64_t)m * a.top;
        st::launch(ctx, logprobs_kernel<F16, E>, dim3((unsigned)a.chunks, (unsigned)n), dim3(kThreads), 0, b);
        if (int rc = st::launch_check("logprobs_kernel")) return rc;
    }
    return ST_OK;
}

template <bool F16>
int by_size(st_context *ctx, const Args &a, int M) {
    // Few rows: small chunks, so that every CU has some (one row of 151936: 75
    // workgroups); many: large ones, whose fixed cost is a quarter per logit.
    const bool large = (int64_t)M * ((a.V + 8191) / 8192) >= 2 * ctx->num_cus || a.V + 1 > 2048 * kMaxChunks;
    return large ? launch_rows<F16, 32>(ctx, a, M) : launch_rows<F16, 8>(ctx, a, M);
}

}  // namespace

extern "C" int st_token_logprobs(st_context *ctx, const void *logits, int dtype, int64_t stride, const int32_t *tokens,
                                 float *logprob, float *entropy, int32_t *rank, int32_t *top_ids, float *top_logprobs, int M,
                                 int V, int top) {
    const char *const fn = "st_token_logprobs";
    if (!ctx || !logits) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (dtype != ST_F32 && dtype != ST_F16) return st::fail(ST_ERR_INVALID, "%s: dtype %d (f32 or f16)", fn, dtype);
    if (!tokens && (logprob || rank)) return st::fail(ST_ERR_INVALID, "%s: logprob and rank need tokens", fn);
    if (top < 0 || top > kMaxTop) return st::fail(ST_ERR_SHAPE, "%s: top=%d (at most %d)", fn, top, kMaxTop);
    if (top > 0 && !top_ids) return st::fail(ST_ERR_INVALID, "%s: top=%d without top_ids", fn, top);
    if (top == 0 && (top_ids || top_logprobs)) top_ids = nullptr, top_logprobs = nullptr;
    if (M < 1 || V < 1 || V > (1 << 20) || top > V || stride < V)
        return st::fail(ST_ERR_SHAPE, "%s: M=%d, V=%d (at most 2^20), stride %lld, top=%d", fn, M, V, (long long)stride, top);
    if ((reinterpret_cast<uintptr_t>(logits) & (dtype == ST_F32 ? 3 : 1)) != 0)
        return st::fail(ST_ERR_ALIGN, "%s: logits not aligned to their type", fn);
    Args a{logits, stride, tokens, logprob, entropy, rank, top_ids, top_logprobs, V, top, 0, nullptr, nullptr};
    return dtype == ST_F16 ? by_size<true>(ctx, a, M) : by_size<false>(ctx, a, M);
}
