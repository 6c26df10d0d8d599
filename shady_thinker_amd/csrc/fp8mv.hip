// e4m3 rows times an e4m3 weight (st_fp8_gemm), up to 64 tokens: bound by the
// weight's bytes.
//
// A workgroup takes 16 NT columns, its W waves every W-th block of 128 k. A
// wave brings its blocks of both operands to LDS by DMA, S of them ahead, in
// slots of its own: it waits for its own loads only, and the waves meet once,
// when their sums are added in order. A row's 128 bytes are eight 16-byte
// chunks, chunk j of row r at j ^ (r % 8), so that fragment reads hit every
// bank once. e4m3 goes to f16 exactly and f16 products are exact in the matrix
// instruction's f32 sums (the 8-bit instruction's are not, see fp8mm.hip).
//
// Sizes of columns and waves (MI355X, cold weights; us of (NT, W)):
//   16 columns, 16 or 8 waves: up to a tile a CU (one token 4096 x 4096: (1, 16) 5.9, (1, 8) 7.1, (2, 8) 6.9, (2, 4) 8.3)
//   16 columns, fewer waves, several workgroups a CU: up to 1.2
//   32 columns, 8 waves: up to 2 (4096 x 8192: (2, 8) 9.6, (1, 8) 10.9, (2, 4) 10.1)
//   then four waves and 32, 48 or 64 columns, whichever leaves the fullest CU
//   the fewest (4096 x 22016: 48 20.2, 32 20.7, 64 21.1; 28672: 64 24.4, 32 26.3, 48 28.2)
#include "fp8mm.hpp"

#include <algorithm>

namespace {

using namespace st::f8;

constexpr int S = 2;  // slots of a wave (three: 4096 x 22016, 48 columns 15.8 -> 18.2 us: fewer workgroups a CU)

// X8: at most eight tokens, one DMA of x for a block.
template <int MT, bool X8, int NT, int W>
__global__ __launch_bounds__(64 * W) void mv_kernel(MmArgs a) {
    constexpr int XD = X8 ? 1 : 2 * MT, ND = 2 * NT + XD;  // DMAs of a slot, eight rows each
    constexpr int SLOT = ND * 1024;
    static_assert(!X8 || MT == 1, "eight tokens are one fragment");
    static_assert(SLOT >= MT * NT * 1024, "the waves' sums fit the first slots");
    __shared__ __align__(1024) uint8_t s0[W * SLOT], s1[W * SLOT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int KB = (a.K + kBlock - 1) / kBlock;
    const int rows_w = min(16 * NT, a.N - n0);
    const __amdgpu_buffer_rsrc_t rw =
        __builtin_amdgcn_make_buffer_rsrc((void *)(a.w + (int64_t)n0 * a.K), (short)0, rows_w * a.K, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void *)a.x, (short)0, a.M * a.K, kRsrcWord3);
    // (the columns' blocks: two where 48 columns lie across a border)
    const int nb = n0 / kBlock, nb_last = (a.N - 1) / kBlock, cross = (nb + 1) * kBlock - n0;  // columns before the border
    const float *const sw0 = a.sw + (int64_t)nb * KB, *const sw1 = a.sw + (int64_t)min(nb + 1, nb_last) * KB;
    // lane i of a DMA fills position i % 8 of its row i / 8; rows past the last repeat it
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    int vw[2 * NT], vx[XD];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) vw[j] = min(8 * j + (lane >> 3), rows_w - 1) * a.K + chunk;
#pragma unroll
    for (int j = 0; j < XD; ++j) vx[j] = min(8 * j + (lane >> 3), a.M - 1) * a.K + chunk;
    struct Scales {
        float x[MT], w0, w1;
    } f0, f1;
    auto load = [&](uint8_t *s, Scales &f, int b) {
        uint8_t *const at = s + wave * SLOT;
        const bool in = b * kBlock + chunk < a.K;  // (K ends inside the last block; past it: zeros)
        const int bs = min(b, KB - 1), so = bs * kBlock;
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) dma16(rw, at + j * 1024, in ? vw[j] : kOutside, so);
#pragma unroll
        for (int j = 0; j < XD; ++j) dma16(rx, at + (2 * NT + j) * 1024, in ? vx[j] : kOutside, so);
#pragma unroll
        for (int t = 0; t < MT; ++t) f.x[t] = a.sx[bs * a.sx_stride + min(16 * t + r, a.M - 1)];
        f.w0 = sw0[bs];
        if constexpr (NT == 3) f.w1 = sw1[bs];
    };
    const int pos = r * kBlock + (c ^ (r & 7)) * 16;
    const int xpos = (X8 ? r & 7 : r) * kBlock + (c ^ (r & 7)) * 16;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0, 0, 0, 0};
    auto frag = [&](const uint8_t *at, int p) {
        Frag<true> v;
        v.set(*reinterpret_cast<const i32x4 *>(at + p), *reinterpret_cast<const i32x4 *>(at + (p ^ 64)));
        return v;
    };
    auto step = [&](uint8_t *s, Scales &f, int b) {
        const uint8_t *const at = s + wave * SLOT;
        wait_loads<(S - 1) * ND, false>();  // (the other slot's may be in flight)
        Frag<true> w[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) w[u] = frag(at + u * 2048, pos);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const Frag<true> x = frag(at + (2 * NT + 2 * t) * 1024, xpos);
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float g = NT == 3 && 16 * u >= cross ? f.w1 : f.w0;
                acc[t][u] += mfma(w[u], x) * (f.x[t] * g);
            }
        }
        wait_lds();  // (the fragments are read: the slot may be filled)
        load(s, f, b + S * W);
    };
    load(s0, f0, wave);
    load(s1, f1, wave + W);
    for (int b = wave; b < KB; b += S * W) {
        step(s0, f0, b);
        if (b + W < KB) step(s1, f1, b + W);
    }
    wait_loads<0, true>();
    __syncthreads();
    f32x4 *const part = reinterpret_cast<f32x4 *>(s0);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) part[(wave * MT * NT + t * NT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * NT * 64; i += 64 * W) {
        const int q = i >> 6, l = i & 63;
        f32x4 v = part[i];
#pragma unroll
        for (int w = 1; w < W; ++w) v += part[w * MT * NT * 64 + i];
        const int m = 16 * (q / NT) + (l & 15);
        if (m < a.M) store_n4(a.y, a.f32, m, n0 + 16 * (q % NT) + 4 * (l >> 4), a.N, v);
    }
}

struct Shape {
    int nt, w;
};

Shape shape(const st_context *ctx, const MmArgs &a) {
    const int tiles = (a.N + 15) / 16, cus = ctx->num_cus, KB = blocks(a.K);
    if (tiles <= cus) {
        // 16 waves where they share the blocks evenly (of 2560, 20 blocks: 8 waves 4.3 us, 16 4.4; of 4096: 7.1, 5.9)
        const bool even = 10 * ((KB + 15) / 16 * 16) <= 11 * KB;
        return {1, a.M <= 16 && even ? 16 : 8};
    }
    if (a.M > 32) return {2, 4};
    if (5 * tiles <= 6 * cus) return {1, a.M <= 16 ? 8 : 4};  // (several workgroups a CU: no second round for a few)
    if (tiles <= 2 * cus) return {2, 8};
    Shape best{2, 4};
    int least = 1 << 30;
    for (int nt = 2; nt <= (a.M <= 16 ? 4 : 3); ++nt) {
        const int cost = ((tiles + nt - 1) / nt + cus - 1) / cus * nt;  // tiles of the fullest CU
        if (cost <= least) least = cost, best.nt = nt;
    }
    return best;
}

template <int MT, bool X8, int NT, int W>
void run(st_context *ctx, const MmArgs &a) {
    st::launch(ctx, mv_kernel<MT, X8, NT, W>, dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT))), dim3(64 * W), 0, a);
}

template <int MT, bool X8>
void by_shape(st_context *ctx, const MmArgs &a, Shape s) {
    if constexpr (MT > 2) {
        s.nt == 1 ? run<MT, X8, 1, 8>(ctx, a) : run<MT, X8, 2, 4>(ctx, a);
    } else {
        if constexpr (MT == 1) {
            if (s.nt == 1 && s.w == 16) return run<MT, X8, 1, 16>(ctx, a);
            if (s.nt == 4) return run<MT, X8, 4, 4>(ctx, a);
        }
        if constexpr (MT == 2)
            if (s.nt == 1 && s.w == 4) return run<MT, X8, 1, 4>(ctx, a);
        if (s.nt == 1) return run<MT, X8, 1, 8>(ctx, a);
        if (s.nt == 2) return s.w == 8 ? run<MT, X8, 2, 8>(ctx, a) : run<MT, X8, 2, 4>(ctx, a);
        run<MT, X8, 3, 4>(ctx, a);
    }
}

}  // namespace

namespace st {
namespace f8 {

// Of 33 to 64 tokens (fewer always come here): a start, and the fullest CUs'
// blocks, which come faster where CUs are idle (fitted at K 1024 to 14336, N 1024
// to 22016).
double mv_us(const st_context *ctx, const MmArgs &a) {
    const Shape s = shape(ctx, a);
    const double each = s.nt == 1 ? (a.M <= 48 ? 0.165 : 0.21) : (a.M <= 48 ? 0.28 : 0.41);
    return 2.6 + std::max(0.6, (double)((a.N + 15) / 16) / s.nt / ctx->num_cus) * blocks(a.K) * each;
}

int mv(st_context *ctx, const MmArgs &a) {
    const Shape s = shape(ctx, a);
    if (a.M <= 8)
        by_shape<1, true>(ctx, a, s);
    else if (a.M <= 16)
        by_shape<1, false>(ctx, a, s);
    else if (a.M <= 32)
        by_shape<2, false>(ctx, a, s);
    else if (a.M <= 48)
        by_shape<3, false>(ctx, a, s);
    else
        by_shape<4, false>(ctx, a, s);
    return st::launch_check("fp8_mv_kernel");
}

}  // namespace f8
}  // namespace st
