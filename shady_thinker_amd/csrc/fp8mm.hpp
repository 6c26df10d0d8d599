// What the kernels of st_fp8_gemm share (fp8mv.hip: few tokens, fp8mm.hip:
// many): arguments, fragments, loads to LDS, stores.
#pragma once

#include "fp8.hpp"

namespace st {
namespace f8 {

constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit data
constexpr int kOutside = 0x7FFFFFF0;    // an offset past every resource: the load gives zeros

struct MmArgs {
    const uint8_t *x, *w;
    const float *sx, *sw;
    void *y;
    int64_t sx_stride;
    int M, K, N;
    int f32;  // y's type
};

// A lane's 32 elements of a fragment (16 rows x 128 k), as the matrix
// instruction takes them: 16-byte chunks c and c + 4 (c = lane / 16) of row
// lane % 16. Which k that is does not matter, it is the same for both operands.
template <bool EXACT>
struct Frag;
template <>
struct Frag<false> {
    i32x8 v;
    __device__ __forceinline__ void set(i32x4 a, i32x4 b) { v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <>
struct Frag<true> {
    half8 v[4];
    static __device__ __forceinline__ half8 eight(int lo, int hi) {
        const half2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        const half2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
        return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    }
    __device__ __forceinline__ void set(i32x4 a, i32x4 b) {
        v[0] = eight(a.x, a.y), v[1] = eight(a.z, a.w), v[2] = eight(b.x, b.y), v[3] = eight(b.z, b.w);
    }
};
__device__ __forceinline__ f32x4 mfma(const Frag<false> &a, const Frag<false> &b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(const Frag<true> &a, const Frag<true> &b) {
    f32x4 p = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[j], b.v[j], p, 0, 0, 0);
    return p;
}

// A buffer resource (uniform) and loads from it to LDS, at `lds` + 16 (or 4)
// lane. Eight lanes take a row's 128 bytes: loads to registers in the fragments'
// order (neighbouring lanes in different rows) went one lane at a time, 64 cycles
// an instruction (16 tokens x 4096 x 22016: 24.9 us; through LDS 20.1). By
// assembly: of the builtin's loads in flight the compiler does not know which
// part of LDS each fills, so before reads of any it waits for more than it must.
// Nothing is written to registers; wait_loads says when they have come, and a
// loop with these has no other vector loads (whose waits would count them) and
// no other use of m0. A resource that may come out of the vector unit (a lane it
// was kept in) needs five wait states before it is read: settle(). That every
// scalar operand has them, the offset too, is checked in the assembly that the
// compiler wrote (tests/test_fp8_wait_states.py); five states in each DMA instead
// cost 4 % (4096 x 4096 x 22016: 333 -> 347 us).
typedef i32x4 Rsrc;
__device__ __forceinline__ Rsrc scalar(Rsrc r) {
    return Rsrc{__builtin_amdgcn_readfirstlane(r.x), __builtin_amdgcn_readfirstlane(r.y), __builtin_amdgcn_readfirstlane(r.z), kRsrcWord3};
}
__device__ __forceinline__ Rsrc rsrc(const void *p, unsigned bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return scalar(Rsrc{(int)(unsigned)at, (int)(unsigned)((at >> 32) & 0xFFFF), (int)bytes, kRsrcWord3});
}
__device__ __forceinline__ unsigned lds_at(const void *p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
__device__ __forceinline__ void settle(Rsrc &a, Rsrc &b) {
    a = scalar(a), b = scalar(b);
    asm volatile("s_nop 4" : "+s"(a), "+s"(b));
}
__device__ __forceinline__ void lds16(Rsrc r, unsigned lds, unsigned voff, int soff) {  // (r settled)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff), "s"(r), "s"(soff) : "memory");
}
__device__ __forceinline__ void lds4(Rsrc r, unsigned lds, int voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(scalar(r)) : "memory");
}

// s_waitcnt: at most n vector loads in flight (LDS reads too: none).
template <int N, bool LDS>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "six bits");
    __builtin_amdgcn_s_waitcnt((LDS ? 0x0070 : 0x0F70) + (N & 15) + (N >> 4 << 14));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}

// Four neighbouring n of token m.
__device__ __forceinline__ void store_n4(void *y, bool f32, int m, int n, int N, f32x4 v) {
    const int64_t at = (int64_t)m * N + n;
    if (n + 4 <= N && (N & 3) == 0) {
        if (f32)
            *reinterpret_cast<f32x4 *>(static_cast<float *>(y) + at) = v;
        else
            *reinterpret_cast<half4 *>(static_cast<_Float16 *>(y) + at) = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < N) {
            if (f32)
                static_cast<float *>(y)[at + i] = v[i];
            else
                static_cast<_Float16 *>(y)[at + i] = (_Float16)v[i];
        }
}

// Few tokens (fp8mv.hip): the estimated time (us) of at most 64, and the call.
double mv_us(const st_context *ctx, const MmArgs &a);
int mv(st_context *ctx, const MmArgs &a);

}  // namespace f8
}  // namespace st
