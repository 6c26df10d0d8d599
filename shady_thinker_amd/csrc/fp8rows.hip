// Rows of activations as e4m3 with a scale for each token and 128 dims:
// st_add_rmsnorm (the residual's addition and the norm before a linear; the
// reference's rmsnorm.wgsl / add_rmsnorm.wgsl, src/model.rs:685-691, 799, 820)
// and st_fp8_quant (rows, or silu(a) b, before the output and down projections).
//   r = residual + x,  y = r (mean r^2 + eps)^-1/2 (weight + 0 or 1)
//   s_b = max |y_k| / 448 over the block b,  q_k = e4m3(y_k / s_b)
// Bound by HBM: every value is read and written once, in registers between. 4096
// rows: norms of 4096 dims, f32 43.2 us (5.05 TB/s), f16 25.4 (4.6), of 8192 f32
// 81.1 (5.4), silu of f16 11008 44.5 (5.1); a copy of 1 GiB runs at 5.1. A row is a
// workgroup of the norm (its sum goes through LDS once), 256 threads of 2048 dims
// one of the quantising. Few rows are a launch and a chain of latencies: one row
// of 4096 3.2 us, one of silu of 11008 2.4. f32 arithmetic; a value is rounded
// once to e4m3 (2^-4), the residual once to its type.
#include "fp8.hpp"

#include <algorithm>

namespace {

using namespace st::f8;

struct NormArgs {
    const void *res, *x;
    void *res_out;
    const float *weight;
    void *y;
    uint8_t *y8;
    float *scale;
    int64_t res_stride, x_stride, out_stride, y_stride, scale_stride;
    float eps, weight_add, per_d;
    int pieces;  // of a row: D / 8
    int y_f32;
};

// One workgroup a row; a thread holds pieces of eight dims, blockDim.x apart,
// from their load to the last store.
template <bool RF32, bool XF32, int P>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
    __shared__ f32x4 sums[16];  // of each wave's four rows of lanes
    const int tid = threadIdx.x, waves = blockDim.x >> 6;
    const int64_t t = blockIdx.x;
    float r[P][8];
    float sum = 0.0f;
    Raw8<RF32> rr[P];
    Raw8<XF32> rx[P];
    f32x4 w[P][2];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int piece = tid + p * (int)blockDim.x;
        if (piece < a.pieces) {
            rr[p].load(a.res, t * a.res_stride + piece * 8);
            if (a.x) rx[p].load(a.x, t * a.x_stride + piece * 8);
            const f32x4 *s = reinterpret_cast<const f32x4 *>(a.weight) + piece * 2;
            w[p][0] = s[0], w[p][1] = s[1];
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int piece = tid + p * (int)blockDim.x;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[p][i] = 0.0f;
        if (piece < a.pieces) {
            rr[p].to(r[p]);
            if (a.x) {
                float x[8];
                rx[p].to(x);
#pragma unroll
                for (int i = 0; i < 8; ++i) r[p][i] += x[i];
                if (a.res_out) store8<RF32>(a.res_out, t * a.out_stride + piece * 8, r[p]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += r[p][i] * r[p][i];
    }
    sum = row_sum(sum);
    if ((tid & 15) == 0) reinterpret_cast<float *>(sums)[tid >> 4] = sum;
    __syncthreads();
    f32x4 all = sums[0];
#pragma unroll
    for (int i = 1; i < 16; ++i)
        if (i < waves) all += sums[i];
    sum = (all.x + all.y) + (all.z + all.w);
    const float norm = __builtin_amdgcn_rsqf(sum * a.per_d + a.eps);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int piece = tid + p * (int)blockDim.x;
        const bool live = piece < a.pieces;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = live ? r[p][i] * norm * (w[p][i / 4][i % 4] + a.weight_add) : 0.0f;
        if (a.y && live) {
            if (a.y_f32)
                store8<true>(a.y, t * a.y_stride + piece * 8, y);
            else
                store8<false>(a.y, t * a.y_stride + piece * 8, y);
        }
        if (a.y8) {
            const float s = block_scale(y);
            const u32x2 q = to_e4m3(y, s);
            if (live) {
                *reinterpret_cast<u32x2 *>(a.y8 + t * a.pieces * 8 + piece * 8) = q;
                if (piece % 16 == 0) a.scale[piece / 16 * a.scale_stride + t] = s;
            }
        }
    }
}

struct QuantArgs {
    const void *a, *b;
    int64_t a_stride, b_stride, scale_stride;
    uint8_t *y8;
    float *scale;
    int pieces, units;  // pieces of a row; workgroups a row
};

// 16 lanes a block of 128, a thread eight dims.
template <bool F32, bool SILU>
__global__ __launch_bounds__(256) void quant_kernel(QuantArgs a) {
    const int64_t t = blockIdx.x / a.units;
    const int piece = (blockIdx.x % a.units) * 256 + threadIdx.x;
    const bool live = piece < a.pieces;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live) {
        Raw8<F32> ra, rb;
        ra.load(a.a, t * a.a_stride + piece * 8);
        if constexpr (SILU) rb.load(a.b, t * a.b_stride + piece * 8);
        ra.to(x);
        if constexpr (SILU) {
            float y[8];
            rb.to(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i] * -1.44269504f)) * y[i];
        }
    }
    const float s = block_scale(x);
    const u32x2 q = to_e4m3(x, s);
    if (live) {
        *reinterpret_cast<u32x2 *>(a.y8 + t * a.pieces * 8 + piece * 8) = q;
        if (piece % 16 == 0) a.scale[piece / 16 * a.scale_stride + t] = s;
    }
}

template <bool RF32, bool XF32>
void launch_norm(st_context *ctx, const NormArgs &a, int M) {
    // One piece a thread up to 8192 dims (4095 rows of 4096, f32: 42.2 us; two 43.3, four 46.2; one row 2.9, 3.1, 3.7), but two
    // of many f16 rows whose workgroups are large for what they load (4095 rows, us of two and one: of 4112 27.3, 28.1; 4608
    // 28.8, 29.6; 5120 31.8, 33.8; 6144 37.4, 37.2; 7168 42.5, 44.2; 8192 46.7, 47.7; 256 to 1024 rows 0 to 10 % less or equal)
    const bool two = !RF32 && a.pieces > 512 && M >= ctx->num_cus;
    const int per = a.pieces <= 1024 ? 1 + two : a.pieces <= 2048 ? 2 : 4;
    const dim3 block((unsigned)(((a.pieces + per - 1) / per + 63) / 64 * 64));
    if (per == 1)
        st::launch(ctx, norm_kernel<RF32, XF32, 1>, dim3((unsigned)M), block, 0, a);
    else if (per == 2)
        st::launch(ctx, norm_kernel<RF32, XF32, 2>, dim3((unsigned)M), block, 0, a);
    else
        st::launch(ctx, norm_kernel<RF32, XF32, 4>, dim3((unsigned)M), block, 0, a);
}

}  // namespace

extern "C" int st_add_rmsnorm(st_context *ctx, const void *residual, int res_dtype, int64_t res_stride, const void *x, int x_dtype,
                              int64_t x_stride, void *residual_out, int64_t out_stride, const float *weight, float eps, void *y,
                              int y_dtype, int64_t y_stride, uint8_t *y8, float *y_scale, int64_t scale_stride, int M, int D,
                              uint32_t flags) {
    const char *const fn = "st_add_rmsnorm";
    if (!ctx || !residual || !weight) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if ((x == nullptr) != (residual_out == nullptr))
        return st::fail(ST_ERR_INVALID, "%s: x without residual_out, or residual_out without x", fn);
    if ((y8 == nullptr) != (y_scale == nullptr)) return st::fail(ST_ERR_INVALID, "%s: y8 without y_scale, or y_scale without y8", fn);
    if (!y && !y8) return st::fail(ST_ERR_INVALID, "%s: neither y nor y8", fn);
    if (!act_dtype(res_dtype) || (x && !act_dtype(x_dtype)) || (y && !act_dtype(y_dtype)))
        return st::fail(ST_ERR_INVALID, "%s: dtypes %d, %d, %d (f32 or f16)", fn, res_dtype, x_dtype, y_dtype);
    if (flags & ~ST_FLAG_NORM_PLUS_ONE) return st::fail(ST_ERR_INVALID, "%s: flags 0x%x", fn, flags);
    if (M < 1 || D < 16 || D % 16 || D > 32768)
        return st::fail(ST_ERR_SHAPE, "%s: M=%d, D=%d (a multiple of 16, at most 32768)", fn, M, D);
    if (res_stride < D || (x && (x_stride < D || out_stride < D)) || (y && y_stride < D) || (y8 && scale_stride < M))
        return st::fail(ST_ERR_SHAPE, "%s: a row overlaps the next one", fn);
    if (!whole16(res_stride, res_dtype) || (x && (!whole16(x_stride, x_dtype) || !whole16(out_stride, res_dtype))) ||
        (y && !whole16(y_stride, y_dtype)))
        return st::fail(ST_ERR_ALIGN, "%s: strides must be whole 16 bytes", fn);
    if (!st::aligned16(residual) || !st::aligned16(x) || !st::aligned16(residual_out) || !st::aligned16(weight) || !st::aligned16(y) ||
        !st::aligned16(y8) || !aligned4(y_scale))
        return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned (y_scale: 4)", fn);
    // (a row's outputs may be written before another's inputs are read: in one buffer they are the same row's)
    if (y && ((y == x && (y_dtype != x_dtype || y_stride != x_stride)) ||
              (y == residual && (y_dtype != res_dtype || y_stride != res_stride))))
        return st::fail(ST_ERR_INVALID, "%s: y in an input's buffer with another type or stride", fn);
    if (x && residual_out == residual && out_stride != res_stride)
        return st::fail(ST_ERR_INVALID, "%s: residual_out in residual's buffer with another stride", fn);
    if (y && y == residual_out) return st::fail(ST_ERR_INVALID, "%s: y in residual_out's buffer", fn);
    if ((int64_t)M * 1024 > 0xFFFFFFFF) return st::fail(ST_ERR_SHAPE, "%s: M=%d (fewer than 2^22)", fn, M);
    if (x && residual_out == x && (res_dtype != x_dtype || out_stride != x_stride))
        return st::fail(ST_ERR_INVALID, "%s: residual_out in x's buffer with another type or stride", fn);
    if (weight == y || weight == residual_out || one_of(y8, {residual, x, residual_out, weight, y}) ||
        one_of(y_scale, {residual, x, residual_out, weight, y, y8}))
        return st::fail(ST_ERR_INVALID, "%s: an output in another argument's buffer", fn);
    NormArgs a{};
    a.res = residual, a.x = x, a.res_out = residual_out, a.weight = weight, a.y = y, a.y8 = y8, a.scale = y_scale;
    a.res_stride = res_stride, a.x_stride = x_stride, a.out_stride = out_stride, a.y_stride = y_stride, a.scale_stride = scale_stride;
    a.eps = eps, a.weight_add = flags & ST_FLAG_NORM_PLUS_ONE ? 1.0f : 0.0f, a.per_d = 1.0f / D;
    a.pieces = D / 8, a.y_f32 = y_dtype == ST_F32;
    const st::OnDevice on(ctx);
    if (on.error != hipSuccess) return st::hip_fail(on.error, fn);
    const bool rf32 = res_dtype == ST_F32, xf32 = x ? x_dtype == ST_F32 : rf32;
    if (rf32)
        xf32 ? launch_norm<true, true>(ctx, a, M) : launch_norm<true, false>(ctx, a, M);
    else
        xf32 ? launch_norm<false, true>(ctx, a, M) : launch_norm<false, false>(ctx, a, M);
    return st::launch_check("norm_kernel");
}

extern "C" int st_fp8_quant(st_context *ctx, const void *a, const void *b, int dtype, int64_t a_stride, int64_t b_stride, uint8_t *y8,
                            float *y_scale, int64_t scale_stride, int M, int K) {
    const char *const fn = "st_fp8_quant";
    if (!ctx || !a || !y8 || !y_scale) return st::fail(ST_ERR_INVALID, "%s: NULL argument", fn);
    if (!act_dtype(dtype)) return st::fail(ST_ERR_INVALID, "%s: dtype %d (f32 or f16)", fn, dtype);
    if (M < 1 || K < 16 || K % 16 || K > (1 << 22)) return st::fail(ST_ERR_SHAPE, "%s: M=%d, K=%d (a multiple of 16, at most 2^22)", fn, M, K);
    if (a_stride < K || (b && b_stride < K) || scale_stride < M) return st::fail(ST_ERR_SHAPE, "%s: a row overlaps the next one", fn);
    if (!whole16(a_stride, dtype) || (b && !whole16(b_stride, dtype))) return st::fail(ST_ERR_ALIGN, "%s: strides must be whole 16 bytes", fn);
    if (!st::aligned16(a) || !st::aligned16(b) || !st::aligned16(y8) || !aligned4(y_scale))
        return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned (y_scale: 4)", fn);
    QuantArgs q{};
    q.a = a, q.b = b, q.a_stride = a_stride, q.b_stride = b_stride, q.scale_stride = scale_stride;
    q.y8 = y8, q.scale = y_scale, q.pieces = K / 8, q.units = (K / 8 + 255) / 256;
    if ((int64_t)M * q.units * 256 > 0xFFFFFFFF) return st::fail(ST_ERR_SHAPE, "%s: M=%d rows of %d are too many", fn, M, K);
    if (one_of(y8, {a, b}) || one_of(y_scale, {a, b, y8})) return st::fail(ST_ERR_INVALID, "%s: an output in another argument's buffer", fn);
    const st::OnDevice on(ctx);
    if (on.error != hipSuccess) return st::hip_fail(on.error, fn);
    const dim3 grid((unsigned)(M * q.units)), block(256);
    const bool f32 = dtype == ST_F32;
    if (b)
        f32 ? st::launch(ctx, quant_kernel<true, true>, grid, block, 0, q) : st::launch(ctx, quant_kernel<false, true>, grid, block, 0, q);
    else
        f32 ? st::launch(ctx, quant_kernel<true, false>, grid, block, 0, q) : st::launch(ctx, quant_kernel<false, false>, grid, block, 0, q);
    return st::launch_check("quant_kernel");
}
