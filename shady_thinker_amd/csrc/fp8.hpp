// Rows and weights in 8-bit floating point (OCP e4m3: finite, at most 448)
// with float32 scales of blocks of 128, on the device, and the argument checks
// their entry points share.
#pragma once

#include <initializer_list>

#include "common.hpp"

namespace st {
namespace f8 {

constexpr int kBlock = 128;       // elements of a row, rows of a weight, under one scale
constexpr float kMost = 448.0f;   // e4m3's largest value
constexpr float kLeast = 0x1p-126f;  // the least scale: its reciprocal is finite too

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Eight adjacent elements as they are stored, and as floats.
template <bool F32>
struct Raw8;
template <>
struct Raw8<true> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const void *p, int64_t at) {
        const f32x4 *s = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + at);
        a = s[0], b = s[1];
    }
    __device__ __forceinline__ void to(float (&x)[8]) const {
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
};
template <>
struct Raw8<false> {
    half8 a;
    __device__ __forceinline__ void load(const void *p, int64_t at) {
        a = *reinterpret_cast<const half8 *>(static_cast<const _Float16 *>(p) + at);
    }
    __device__ __forceinline__ void to(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    }
};

template <bool F32>
__device__ __forceinline__ void store8(void *p, int64_t at, const float (&x)[8]) {
    if constexpr (F32) {
        f32x4 *s = reinterpret_cast<f32x4 *>(static_cast<float *>(p) + at);
        s[0] = f32x4{x[0], x[1], x[2], x[3]};
        s[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        half8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = (_Float16)x[i];
        *reinterpret_cast<half8 *>(static_cast<_Float16 *>(p) + at) = r;
    }
}

// Over 16 lanes side by side (a row of the DPP), the row turned by 8, 4, 2 and
// 1 lanes: every lane gets the largest, or the sum (each lane's in an order of
// its own: one lane's is taken).
template <int N>
__device__ __forceinline__ unsigned turned(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x120 + N, 0xF, 0xF, false);
}
template <int N>
__device__ __forceinline__ unsigned max_turned(unsigned v) {
    const unsigned o = turned<N>(v);
    return v > o ? v : o;
}
template <int N>
__device__ __forceinline__ float add_turned(float v) {
    return v + __uint_as_float(turned<N>(__float_as_uint(v)));
}
__device__ __forceinline__ float row_sum(float v) { return add_turned<1>(add_turned<2>(add_turned<4>(add_turned<8>(v)))); }

// The scale of a block whose 128 values lie in 16 lanes side by side, eight in
// each: max |x| times the f32 nearest to 1 / 448, at least 2^-126. Magnitudes
// compare as their bits do, with NaN above infinity, so that a NaN in a block
// makes its scale NaN.
__device__ __forceinline__ float block_scale(const float (&x)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned b = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    m = max_turned<1>(max_turned<2>(max_turned<4>(max_turned<8>(m))));
    const float s = __uint_as_float(m) * (1.0f / kMost);
    return s < kLeast ? kLeast : s;
}

// Eight values over their block's scale, each quotient rounded to f32 and then to
// e4m3 (to nearest, even). A product with the reciprocal alone may be a step off,
// which takes a quotient at the middle of two e4m3 values to either (16 of a
// million f16 values); its remainder, exact in an FMA, corrects it (0 keeps its
// sign: -0 is added to it). 4096 f16 rows of silu of 11008 43.5 -> 43.8 us, without
// silu 28.4, f32 77.7 and 43.4 as before. The largest is 448 within two steps, which rounds to
// 448. Where the scale is not finite: 448 of its sign for an infinity (0 times
// infinity, so the smaller of NaN and 448), 0 beside it, and 448 beside a NaN.
__device__ __forceinline__ u32x2 to_e4m3(const float (&x)[8], float scale) {
    float inv = __builtin_amdgcn_rcpf(scale);
    inv = fmaf(-fmaf(scale, inv, -1.0f), inv, inv);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = x[i] * inv;
        v[i] = fmaf(-fmaf(scale, q, -x[i]), inv, q);
    }
    if (!(scale < __builtin_inff())) {
        inv = __builtin_amdgcn_rcpf(scale);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = copysignf(fminf(fabsf(x[i] * inv), kMost), x[i]);
    }
    u32x2 r;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    r.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    r.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], w, true);
    return r;
}

inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
inline bool one_of(const void *p, std::initializer_list<const void *> others) {
    for (const void *o : others)
        if (p && p == o) return true;
    return false;
}
inline int blocks(int n) { return (n + kBlock - 1) / kBlock; }
inline bool act_dtype(int d) { return d == ST_F32 || d == ST_F16; }
inline bool whole16(int64_t elements, int dtype) { return elements % (dtype == ST_F32 ? 4 : 8) == 0; }

}  // namespace f8

// A call's launches go to the context's device, whichever is current.
struct OnDevice {
    int before = -1;
    hipError_t error;
    explicit OnDevice(const st_context *ctx) {
        error = hipGetDevice(&before);
        if (error == hipSuccess && before != ctx->device) error = hipSetDevice(ctx->device);
        if (before == ctx->device) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

}  // namespace st
