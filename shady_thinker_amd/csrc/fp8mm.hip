// Product of e4m3 rows with an e4m3 weight, float32 scales of 128 x 128
// blocks of the weight and of each token's 128 dims (st_fp8_gemm; no reference
// counterpart, as INT8):
//   y[m][n] = sum_b sx[b][m] sw[n / 128][b] sum_{k in b} x[m][k] w[n][k]
// Two ways to sum a block's 128 products:
//  * v_mfma_f32_16x16x128_f8f6f4 takes the block whole. In each eight k it keeps
//    a product to 2^-13 of the largest one's power of two (measured: a product
//    of 2^-14 beside one of 1 is lost, in another eight it counts to 2^-23), so
//    the sum is off by some 2^-15 of its magnitude: for f16 y, whose own
//    rounding is 2^-12 at the mean.
//  * f32 y: e4m3 is exact in f16, and so are the products of
//    v_mfma_f32_16x16x32_f16 in its f32 sums. Half the rate; also for few
//    tokens, where the weight's bytes bound the call.
// One FMA with the block's factor adds its sum to the accumulator. The weight
// is the A operand, so that a lane holds four neighbouring n of one token,
// whose factor is then one register.
#include "fp8.hpp"

#include <algorithm>

#include "xcd.hpp"

namespace {

using namespace st::f8;

constexpr int kRsrcWord3 = 0x00020000;  // raw 32-bit data
constexpr int kOutside = 0x7FFFFFF0;    // an offset past every resource: the load gives zeros

struct MmArgs {
    const uint8_t *x, *w;
    const float *sx, *sw;
    void *y;
    int64_t sx_stride;
    int M, K, N;
};

// A lane's 32 elements of a fragment (16 rows x 128 k), as the matrix
// instruction takes them.
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

// Four neighbouring n of token m.
template <bool F32>
__device__ __forceinline__ void store_n4(void *y, int m, int n, int N, f32x4 v) {
    const int64_t at = (int64_t)m * N + n;
    if (n + 4 <= N && (N & 3) == 0) {
        if constexpr (F32)
            *reinterpret_cast<f32x4 *>(static_cast<float *>(y) + at) = v;
        else
            *reinterpret_cast<half4 *>(static_cast<_Float16 *>(y) + at) = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < N) {
            if constexpr (F32)
                static_cast<float *>(y)[at + i] = v[i];
            else
                static_cast<_Float16 *>(y)[at + i] = (_Float16)v[i];
        }
}

// Up to 16 MT tokens: a workgroup takes 16 columns, its waves every W-th block
// of k; operands go from memory to registers. A lane's fragment is 16-byte
// chunks c and c + 4 of a row's 128 bytes (c = lane / 16): which k that is does
// not matter, it is the same for both operands.
template <int MT, int W, bool F32>
__global__ __launch_bounds__(64 * W) void mv_kernel(MmArgs a) {
    __shared__ f32x4 part[W][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int KB = (a.K + kBlock - 1) / kBlock;
    const __amdgpu_buffer_rsrc_t rw =
        __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + (int64_t)n0 * a.K), (short)0, min(16, a.N - n0) * a.K, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void *)a.x, (short)0, a.M * a.K, kRsrcWord3);
    const float *const sw = a.sw + (int64_t)(n0 / kBlock) * KB;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0, 0, 0, 0};
    for (int b = wave; b < KB; b += W) {
        const int k0 = b * kBlock + c * 16;
        const bool in0 = k0 < a.K, in1 = k0 + 64 < a.K;  // (K ends inside the last block)
        const i32x4 w0 = __builtin_amdgcn_raw_buffer_load_b128(rw, in0 ? r * a.K + k0 : kOutside, 0, 0);
        const i32x4 w1 = __builtin_amdgcn_raw_buffer_load_b128(rw, in1 ? r * a.K + k0 + 64 : kOutside, 0, 0);
        const float s = sw[b];
        Frag<true> w;
        w.set(w0, w1);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int at = (16 * t + r) * a.K + k0;
            const i32x4 x0 = __builtin_amdgcn_raw_buffer_load_b128(rx, in0 ? at : kOutside, 0, 0);
            const i32x4 x1 = __builtin_amdgcn_raw_buffer_load_b128(rx, in1 ? at + 64 : kOutside, 0, 0);
            const float f = a.sx[b * a.sx_stride + min(16 * t + r, a.M - 1)] * s;
            Frag<true> x;
            x.set(x0, x1);
            acc[t] += mfma(w, x) * f;
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 64; i += 64 * W) {
        const int t = i >> 6, l = i & 63;
        f32x4 v = part[0][t][l];
#pragma unroll
        for (int w = 1; w < W; ++w) v += part[w][t][l];
        const int m = 16 * t + (l & 15);
        if (m < a.M) store_n4<F32>(a.y, m, n0 + 4 * (l >> 4), a.N, v);
    }
}

// 16 bytes for each lane from a resource to LDS, at `lds` + 16 lane.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t *lds, int voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, voff, soff, 0, 0);
}

// Many tokens: a workgroup takes BM tokens x BN columns, its WM x WN waves
// equal parts of them. A block of 128 k of both operands is in LDS while the
// next one's comes by DMA; a row's 128 bytes are eight 16-byte chunks, chunk j
// of row r at j ^ (r % 8), so that fragment reads hit every bank once.
template <int BM, int BN, int WM, int WN, bool F32>
__global__ __launch_bounds__(64 * WM * WN) void mm_kernel(MmArgs a) {
    constexpr int W = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
    constexpr int DX = BM / 8 / W, DW = BN / 8 / W;  // DMAs (8 rows) of a wave
    static_assert(DX * 8 * W == BM && DW * 8 * W == BN, "whole DMAs a wave");
    __shared__ __align__(1024) uint8_t s0[(BM + BN) * kBlock], s1[(BM + BN) * kBlock];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int KB = (a.K + kBlock - 1) / kBlock;
    const int tm = (a.M + BM - 1) / BM;
    const int id = st::xcd_order(blockIdx.x, gridDim.x);
    const int m0 = id % tm * BM, n0 = id / tm * BN;
    const int wm0 = wave % WM * (BM / WM), wn0 = wave / WM * (BN / WN);
    const int rows_x = min(BM, a.M - m0), rows_w = min(BN, a.N - n0);
    const __amdgpu_buffer_rsrc_t rx =
        __builtin_amdgcn_make_buffer_rsrc((void *)(a.x + (int64_t)m0 * a.K), (short)0, rows_x * a.K, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rw =
        __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + (int64_t)n0 * a.K), (short)0, rows_w * a.K, kRsrcWord3);
    // lane i of a DMA fills position i % 8 of its row i / 8
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    int vx[DX], vw[DW];
#pragma unroll
    for (int j = 0; j < DX; ++j) vx[j] = min((wave * DX + j) * 8 + (lane >> 3), rows_x - 1) * a.K + chunk;
#pragma unroll
    for (int j = 0; j < DW; ++j) vw[j] = min((wave * DW + j) * 8 + (lane >> 3), rows_w - 1) * a.K + chunk;
    auto load = [&](uint8_t *s, int b) {
        const bool in = b * kBlock + chunk < a.K;
#pragma unroll
        for (int j = 0; j < DX; ++j) dma16(rx, s + (wave * DX + j) * 1024, in ? vx[j] : kOutside, b * kBlock);
#pragma unroll
        for (int j = 0; j < DW; ++j) dma16(rw, s + BM * kBlock + (wave * DW + j) * 1024, in ? vw[j] : kOutside, b * kBlock);
    };
    const float *const sw = a.sw + (int64_t)((n0 + wn0) / kBlock) * KB;
    const bool alive = n0 + wn0 < a.N;
    float f[MT], fn[MT], g, gn;
    auto load_scales = [&](float(&to)[MT], float &w, int b) {
#pragma unroll
        for (int t = 0; t < MT; ++t) to[t] = a.sx[b * a.sx_stride + min(m0 + wm0 + 16 * t + r, a.M - 1)];
        w = alive ? sw[b] : 0.0f;
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0, 0, 0, 0};
    const int pos = (c ^ (r & 7)) * 16;
    auto frag = [&](const uint8_t *s, int row) {
        const uint8_t *p = s + (row + r) * kBlock;
        Frag<F32> v;
        v.set(*reinterpret_cast<const i32x4 *>(p + pos), *reinterpret_cast<const i32x4 *>(p + (pos ^ 64)));
        return v;
    };
    auto step = [&](uint8_t *s, uint8_t *next, int b) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's DMAs of block b, and its scales
        __syncthreads();                     // everyone's; and everyone has read `next`'s last block
#pragma unroll
        for (int t = 0; t < MT; ++t) f[t] = fn[t];
        g = gn;
        if (b + 1 < KB) {
            load_scales(fn, gn, b + 1);
            load(next, b + 1);
        }
        Frag<F32> wf[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) wf[u] = frag(s + BM * kBlock, wn0 + 16 * u);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const Frag<F32> xf = frag(s, wm0 + 16 * t);
            const float fs = f[t] * g;
#pragma unroll
            for (int u = 0; u < NT; ++u) acc[t][u] += mfma(wf[u], xf) * fs;
        }
    };
    load_scales(fn, gn, 0);
    load(s0, 0);
    for (int b = 0; b < KB; b += 2) {
        step(s0, s1, b);
        if (b + 1 < KB) step(s1, s0, b + 1);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = m0 + wm0 + 16 * t + r;
#pragma unroll
        for (int u = 0; u < NT; ++u)
            if (m < a.M) store_n4<F32>(a.y, m, n0 + wn0 + 16 * u + 4 * c, a.N, acc[t][u]);
    }
}

template <int MT>
void launch_mv(st_context *ctx, const MmArgs &a, bool f32) {
    constexpr int W = 8;
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(64 * W);
    f32 ? st::launch(ctx, mv_kernel<MT, W, true>, grid, block, 0, a) : st::launch(ctx, mv_kernel<MT, W, false>, grid, block, 0, a);
}

template <int BM, int BN, int WM, int WN>
void launch_mm(st_context *ctx, const MmArgs &a, bool f32) {
    const dim3 grid((unsigned)((a.M + BM - 1) / BM * ((a.N + BN - 1) / BN))), block(64 * WM * WN);
    f32 ? st::launch(ctx, mm_kernel<BM, BN, WM, WN, true>, grid, block, 0, a)
        : st::launch(ctx, mm_kernel<BM, BN, WM, WN, false>, grid, block, 0, a);
}

}  // namespace

extern "C" int st_fp8_gemm(st_context *ctx, const uint8_t *x, const float *x_scale, int64_t scale_stride, const uint8_t *w,
                           const float *w_scale, void *y, int y_dtype, int M, int K, int N) {
    const char *const fn = "st_fp8_gemm";
    if (!ctx || !x || !x_scale || !w || !w_scale || !y) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (!act_dtype(y_dtype)) return st::fail(ST_ERR_INVALID, "%s: y_dtype %d (f32 or f16)", fn, y_dtype);
    if (M < 1 || N < 1 || K < 16 || K % 16 || K > (1 << 22))
        return st::fail(ST_ERR_SHAPE, "%s: M=%d, K=%d (a multiple of 16, at most 2^22), N=%d", fn, M, K, N);
    if (scale_stride < M) return st::fail(ST_ERR_SHAPE, "%s: a block's scales overlap the next one's", fn);
    if ((int64_t)blocks(M) * blocks(N) > (1 << 28)) return st::fail(ST_ERR_SHAPE, "%s: M=%d, N=%d", fn, M, N);
    if (!st::aligned16(x) || !st::aligned16(w) || !st::aligned16(y) || !aligned4(x_scale) || !aligned4(w_scale))
        return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned (scales: 4)", fn);
    const MmArgs a{x, w, x_scale, w_scale, y, scale_stride, M, K, N};
    const st::OnDevice on(ctx);
    if (on.error != hipSuccess) return st::hip_fail(on.error, fn);
    const bool f32 = y_dtype == ST_F32;
    if (M <= 64) {
        M <= 16 ? launch_mv<1>(ctx, a, f32) : M <= 32 ? launch_mv<2>(ctx, a, f32) : launch_mv<4>(ctx, a, f32);
        return st::launch_check("mv_kernel");
    }
    launch_mm<128, 128, 2, 2>(ctx, a, f32);
    return st::launch_check("mm_kernel");
}
