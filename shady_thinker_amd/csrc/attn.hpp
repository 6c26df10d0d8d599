// What the attention kernels share: arguments, the cut of a call into items,
// the epilogue.
#pragma once

#include "kvcache.hpp"

namespace st {
namespace attn {

using namespace st::kv;

constexpr int kStep = 32;            // keys of a step of one wave
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
    int window;                  // 0: none
    float scale, cap;            // cap 0: none
    bool q_f32, gate_f32, out_f32;
    // cut: grid.x items, whose chunks' partial results meet in `part`
    // (G * heads rows of PB * HD, then PB (max, sum) pairs) through `cnt`
    int G, split, rows;  // rows: row blocks at most
    float *part, *part_ml;
    unsigned *cnt;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
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
__device__ __forceinline__ int first_key(const Args &a, const Seq &s) {
    if (!a.window) return 0;
    const int64_t lo = (int64_t)s.kv - s.q + 1 - a.window;
    return lo > 0 ? (int)lo & ~(kStep - 1) : 0;
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

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

}  // namespace attn
}  // namespace st
