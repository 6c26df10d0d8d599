// What the attention kernels share: arguments, the cut of a call into items,
// the epilogue.
#pragma once

#include "kvcache.hpp"

#include <climits>

namespace st {
namespace attn {

using namespace st::kv;

constexpr int kMaxChunks = 256;      // chunks of one sequence at most
constexpr float kLog2e = 1.44269504088896340736f;

struct Args {
    Cache c;
    const void *q, *gate;
    void *out;
    const int32_t *table, *kv_len, *q_start;
    const float *slopes;
    int64_t gate_stride;
    int gate_head_stride;
    int table_stride, capacity;  // pages of a table row, tokens they hold
    int T, B, n_heads, group;    // group: query heads of a key head
    int group_shift;             // its logarithm, -1: not a power of two
    int window;                  // 0: none
    float scale, cap;            // cap 0: none
    bool q_f32, gate_f32, out_f32;
    // cut: grid.x items, whose chunks' partial results meet in `part`
    // (G * heads rows of PB * HD, then PB (max, sum) pairs) through `cnt`
    int G, split, rows;  // rows: row blocks at most
    float *part, *part_ml;
    unsigned *cnt;
    // prompts: *odd becomes call where a block left out values (odd_values)
    unsigned *odd, call;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The same, certainly in a scalar register: the compiler drops the builtin for
// a value that it knows to be uniform and then computes it in a vector one
// where it came out of a division. Inside inline asm the wait states are the
// writer's: one between a vector write and v_readfirstlane of it, five between
// that write of a scalar and a vector load that reads it.
__device__ __forceinline__ int scalar(int v) {
    int r;
    asm("s_nop 1\n\tv_readfirstlane_b32 %0, %1\n\ts_nop 4" : "=s"(r) : "v"(v));
    return r;
}
// A pair's row.
__device__ __forceinline__ int row_of_pair(const Args &a, int pair) {
    return a.group_shift >= 0 ? pair >> a.group_shift : pair / a.group;
}
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// Sequence b's rows [q0, q0 + q) and tokens kv (with the rows'), within bounds
// whatever the arrays hold.
struct Seq {
    int q0, q, kv;
};
__device__ __forceinline__ Seq seq_of(const Args &a, int b) {
    Seq s;
    int q0 = b, q1 = b + 1;
    if (a.q_start) q0 = a.q_start[b], q1 = a.q_start[b + 1];
    q0 = min(max(q0, 0), a.T), q1 = min(max(q1, 0), a.T);
    s.q0 = q0;
    s.q = max(q1 - q0, 0);
    s.kv = min(max(a.kv_len[b], 0), a.capacity);
    return s;
}

// First key that any of a sequence's rows sees, at a step's start.
template <int STEP>
__device__ __forceinline__ int first_key(const Args &a, const Seq &s) {
    if (!a.window) return 0;
    const int lo = s.kv - s.q + 1 - a.window;  // (kv below 2^31, q at most 2^24, window at most 2^30)
    return max(lo, 0) & ~(STEP - 1);
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// One workgroup's share: row block rb of sequence b, chunk `chunk` of its
// `chunks`, steps [s0, s1) of the sequence's keys; item ids of the chunks are
// first + chunk * blocks.
struct Item {
    Seq s;
    int b, rb, blocks, chunk, chunks, s0, s1, first, counter;
};

constexpr int kMostRows = 1 << 24;   // row blocks of one call
constexpr int kMostSteps = 1 << 27;  // steps of a sequence (of 16 keys at least)

template <int PB>
__device__ __forceinline__ int blocks_of(const Args &a, const Seq &s) {
    return (int)((unsigned)(s.q * a.group + PB - 1) / PB);
}
template <int STEP>
__device__ __forceinline__ int steps_of(const Args &a, const Seq &s) {
    return (s.kv - first_key<STEP>(a, s) + STEP - 1) / STEP;
}

// C: chunks of C steps so that all items fit the grid: sum over blocks of
// ceil(steps / C) <= work / C + blocks <= G. A multiple of LEAST.
template <int LEAST, int WHOLE>
__device__ __forceinline__ int chunk_steps(const Args &a, unsigned long long work, int blocks, int longest) {
    if (!a.split || longest <= WHOLE) return kMostSteps;
    const unsigned room = (unsigned)max(a.G - blocks, 1);
    const unsigned long long up = work + room - 1;
    unsigned long long c = up >> 32 ? up / room : (unsigned)up / room;
    c = max(c, (unsigned long long)((longest + kMaxChunks - 1) / kMaxChunks));
    c = max((c + LEAST - 1) / LEAST * LEAST, (unsigned long long)LEAST);
    return c > kMostSteps ? kMostSteps : (int)c;
}

// A sequence of up to WHOLE steps stays in one chunk: joining chunks costs
// more than that many steps.
template <int WHOLE>
__device__ __forceinline__ int chunks_of(int steps, int C) {
    return steps <= max(C, WHOLE) ? 1 : (steps + C - 1) / C;
}

// Item w of the call (the same for every wave), or false: there is none.
template <int PB, int STEP, int LEAST, int WHOLE>
__device__ __forceinline__ bool find_item(const Args &a, int w, Item &it) {
    const int lane = threadIdx.x & 63;
    if (a.B == 1) {
        it.s = seq_of(a, 0);
        it.s = Seq{uniform(it.s.q0), uniform(it.s.q), uniform(it.s.kv)};
        it.b = 0;
        it.blocks = blocks_of<PB>(a, it.s);
        if (!it.blocks) return false;
        const int steps = steps_of<STEP>(a, it.s), C = chunk_steps<LEAST, WHOLE>(a, (unsigned long long)it.blocks * steps, it.blocks, steps);
        it.chunks = chunks_of<WHOLE>(steps, C);
        if (w >= it.blocks * it.chunks) return false;
        it.chunk = it.blocks == 1 ? w : w / it.blocks, it.rb = w - it.chunk * it.blocks;
        it.first = it.rb, it.counter = it.rb;
        it.s0 = min(it.chunk * C, steps), it.s1 = it.chunks == 1 ? steps : min(it.s0 + C, steps);
        return true;
    }
    unsigned long long work = 0;
    int blocks = 0, longest = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        if (b < a.B) {
            const Seq s = seq_of(a, b);
            const int n = blocks_of<PB>(a, s), steps = steps_of<STEP>(a, s);
            work += (unsigned long long)n * steps;
            blocks = min(blocks + min(n, kMostRows), kMostRows);
            longest = max(longest, n ? steps : 0);
        }
    }
    work = wave_sum(work);
    blocks = wave_sum(blocks);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) longest = max(longest, __shfl_xor(longest, d));
    // (more row blocks than T rows have: q_start decreases somewhere. The
    // counters and the grid are made for a.rows, so nothing is computed)
    if (uniform(blocks) > a.rows) return false;
    const int C = chunk_steps<LEAST, WHOLE>(a, work, uniform(blocks), uniform(longest));
    int items = 0, rows = 0;  // before this turn's sequences
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        Seq s{0, 0, 0};
        int n = 0, chunks = 1, steps = 0;
        if (b < a.B) {
            s = seq_of(a, b);
            n = blocks_of<PB>(a, s), steps = steps_of<STEP>(a, s);
            chunks = chunks_of<WHOLE>(steps, C);
        }
        int upto = n * chunks, rows_upto = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int i = __shfl_up(upto, d), r = __shfl_up(rows_upto, d);
            if (lane >= d) upto += i, rows_upto += r;
        }
        const unsigned long long mine = __ballot(items + upto > w);
        if (mine) {
            const int l = __builtin_ctzll(mine);
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            it.b = b0 + l;
            it.s = Seq{of(s.q0), of(s.q), of(s.kv)};
            it.blocks = of(n), it.chunks = of(chunks);
            const int begin = items + of(upto) - it.blocks * it.chunks, idx = w - begin;
            it.chunk = it.blocks == 1 ? idx : idx / it.blocks, it.rb = idx - it.chunk * it.blocks;
            it.first = begin + it.rb;
            it.counter = rows + of(rows_upto) - it.blocks + it.rb;
            const int st = of(steps);
            it.s0 = min(it.chunk * C, st), it.s1 = it.chunks == 1 ? st : min(it.s0 + C, st);
            return true;
        }
        items += __builtin_amdgcn_readlane(upto, 63), rows += __builtin_amdgcn_readlane(rows_upto, 63);
    }
    return false;
}

// An item's fields as scalars (once it is known that there is one): what is
// derived from them (page loads, loop bounds) has to be, or the compiler takes
// vector loads and waits for them among the pieces in flight.
__device__ __forceinline__ Item scalars(const Item &it) {
    return Item{Seq{scalar(it.s.q0), scalar(it.s.q), scalar(it.s.kv)}, scalar(it.b), scalar(it.rb), scalar(it.blocks),
                scalar(it.chunk), scalar(it.chunks), scalar(it.s0), scalar(it.s1), scalar(it.first), scalar(it.counter)};
}

// Sign bits set where a half of w is an infinity or a NaN; w with zeros there.
__device__ __forceinline__ unsigned not_finite(unsigned w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ unsigned finite(unsigned w, unsigned odd) { return w & ~((odd - (odd >> 15)) | odd); }
__device__ __forceinline__ unsigned not_finite(half8 v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    return not_finite(w.x) | not_finite(w.y) | not_finite(w.z) | not_finite(w.w);
}

// int8 caches: how a row's weights, softmax weight times value scale, are held
// in f16: over 2^e, with e such that the largest so far (`top`, in units of the
// row's present maximum) is held between 2^3 and 2^15. Value scales may be of
// any proportion to each other: what counts is a weight's proportion to the
// row's largest, and only tokens that the row sees count. (e by the largest
// scale that any row of the block sees, and never lower again: a later token
// with values 2^20 times as large cost the rows before it 17% of their result.)
struct Held {
    float top;
    int e;

    // The next tile's largest weight; the maximum has grown, so that earlier
    // weights count `grown` times what they did. Returns what the sums so far,
    // held as before, have to be multiplied by.
    __device__ __forceinline__ float next(float largest, float grown) {
        top = fmaxf(top * grown, largest);
        const int t = (int)(__float_as_uint(top) >> 23) - 126, was = e;  // top < 2^t (0, an infinity: -126, 129)
        if (top > 0.0f && (unsigned)(t - e - 4) > 11u) e = max(t - 11, -126);
        return was == e ? grown : ldexpf(grown, was - e);
    }
    __device__ __forceinline__ float down() const { return ldexpf(1.0f, -e); }
};

// Where the output's eight or four values go: times sigmoid(gate) where there
// is one.
__device__ __forceinline__ f32x4 gated(const Args &a, f32x4 o, int row, int head, int d) {
    if (!a.gate) return o;
    const int64_t at = row * a.gate_stride + (int64_t)head * a.gate_head_stride + d;
    f32x4 g;
    if (a.gate_f32) {
        g = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.gate) + at);
    } else {
        const half4 h = *reinterpret_cast<const half4 *>(static_cast<const _Float16 *>(a.gate) + at);
        g = f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] / (1.0f + expf(-g[i]));
    return o;
}

__device__ __forceinline__ void store_out(const Args &a, f32x4 o, int row, int head, int d, int hd) {
    o = gated(a, o, row, head, d);
    const int64_t at = ((int64_t)row * a.n_heads + head) * hd + d;
    if (a.out_f32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + at) = o;
    } else {
        *reinterpret_cast<half4 *>(static_cast<_Float16 *>(a.out) + at) =
            half4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
    }
}

// The cut of a call into row blocks of pb pairs and chunks of steps: a.G and
// what goes with it; `extra` chunks more than row blocks at most.
int plan_cut(st_context *ctx, Args &a, int pb, int hd, int step, int least, int64_t extra);

// prompt.hip: f16 q and out, checked by the caller.
int prompt_attention(st_context *ctx, const Args &a, bool i8, int hd);

}  // namespace attn
}  // namespace st
