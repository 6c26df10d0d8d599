// Product of e4m3 rows with an e4m3 weight, float32 scales of 128 x 128
// blocks of the weight and of each token's 128 dims (st_fp8_gemm; no reference
// counterpart, as INT8):
//   y[m][n] = sum_b sx[b][m] sw[n / 128][b] sum_{k in b} x[m][k] w[n][k]
// Up to 48 tokens: fp8mv.hip; up to 64 whichever is estimated faster. Here,
// two ways to sum a block's 128 products:
//  * v_mfma_f32_16x16x128_f8f6f4 takes the block whole. In each eight k it keeps
//    a product to 2^-13 of the largest one's power of two (measured: a product
//    of 2^-14 beside one of 1 is lost, in another eight it counts to 2^-23), so
//    the sum is off by some 2^-15 of its magnitude (rel-L2 1.4e-5 on normal
//    values, 6.8e-5 where one channel is 1000 times the rest): for f16 y, whose
//    own rounding is 2.1e-4, of more than 64 tokens, unless the context asks for
//    exact products (ST_TUNE_FP8_EXACT; 77 x 5120 x 13824 18 -> 30 us, 512 x 11008
//    x 4096 35 -> 55, 4096 x 4096 x 22016 329 -> 648).
//  * otherwise e4m3 goes to f16, exactly, and the products of
//    v_mfma_f32_16x16x32_f16 are exact in its f32 sums. Half the rate.
// One FMA with the block's factor adds its sum to the accumulator: 4 FMAs beside
// an instruction of 32 cycles, which fit under it but draw power (8192^3, a
// workgroup a tile: 454 us, without them 425; instructions alone on random
// operands 3.9 PFLOP/s, with them 3.6). The weight is the A operand, so that a lane holds four
// neighbouring n of one token, whose factor is then one register.
//
// Both kernels keep a block of both operands in LDS, brought by DMA while the
// ones before it are multiplied. A row's 128 bytes are eight 16-byte chunks,
// chunk j of row r at j ^ (r % 8), so that fragment reads hit every bank once.
// Within a block the order is written out (sched_barrier): an instruction, the
// FMAs of the one D before, now and then a DMA (all at once the waves queue for
// the address unit: 16 cycles each). The next block's first fragments are read
// before this one's last instructions.
#include "fp8mm.hpp"

#include <algorithm>

#include "xcd.hpp"

namespace {

using namespace st::f8;

constexpr int kMostRows = 1 << 28;
constexpr int D = 3;      // instructions between one and its FMAs
constexpr int kPanel = 6; // tiles along the tokens that run side by side: an XCD's 32 CUs then
                          // share 6 strips of x and 5 of w in its L2 (4096 x 4096 x 22016 in 128 x 256: all 387 us, 8 381, 6 370, 4 384; in 256 x 256: 348, 343, 338, 338)

struct Place {
    int m0, n0, split;
};
template <int BM, int BN>
__device__ __forceinline__ Place place(const MmArgs &a, int splits) {
    const int id = st::xcd_order(blockIdx.x, gridDim.x);
    const int tiles = gridDim.x / splits, tm = (a.M + BM - 1) / BM, tn = tiles / tm;
    const int split = id / tiles, tile = id - split * tiles;
    const int panel = tile / (kPanel * tn), at = tile - panel * kPanel * tn, wide = min(kPanel, tm - panel * kPanel);
    return {(panel * kPanel + at % wide) * BM, at / wide * BN, split};
}

// 16 tokens' sums (16 NT columns of a wave) to y, turned in LDS R tokens at a
// time, so that neighbouring lanes write a row's 16-byte chunks; as the lanes
// hold them, four neighbours each, a store went one lane at a time (4096 x 4096 x
// 22016 in tiles of 128 x 256: 387 -> 366 us). Chunk j of row r is at j ^ (r %
// chunks). (N a multiple of 16 bytes.)
template <typename T, int R, int NT>
__device__ __forceinline__ void turned(i32x4 *s, const f32x4 (&v)[NT], T *y, int m, int rows, int n, int N) {
    constexpr int PER = 16 / sizeof(T), CHUNKS = 16 * NT / PER, ROWS = 64 / CHUNKS;
    static_assert(CHUNKS <= 64 && R % ROWS == 0, "whole rows");
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // (its addresses do not wait in registers through the blocks)
    const int r = lane & 15, c = lane >> 4, j = lane % CHUNKS;
#pragma unroll
    for (int h = 0; h < 16; h += R) {
        if (r / R * R == h) {
            const int row = r - h;
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                if constexpr (sizeof(T) == 4)
                    reinterpret_cast<f32x4 *>(s)[row * CHUNKS + ((4 * u + c) ^ (row % CHUNKS))] = v[u];
                else
                    reinterpret_cast<half4 *>(s + row * CHUNKS + ((2 * u + c / 2) ^ (row % CHUNKS)))[c & 1] =
                        half4{(_Float16)v[u].x, (_Float16)v[u].y, (_Float16)v[u].z, (_Float16)v[u].w};
            }
        }
        wait_lds();
#pragma unroll
        for (int i = 0; i < R; i += ROWS) {
            const int row = i + lane / CHUNKS;
            const i32x4 w = s[row * CHUNKS + (j ^ (row % CHUNKS))];
            if (h + row < rows && n + j * PER < N) *reinterpret_cast<i32x4 *>(y + (int64_t)(m + h + row) * N + n + j * PER) = w;
        }
        wait_lds();
    }
}

// ------------------------------------------------------------------ a ring
// BM x BN of y by WM x WN waves, S stages of LDS, K in slices where the tiles
// alone leave CUs idle (f32 partial sums in the workspace, added in order by
// reduce_kernel). Block b + S - 1 comes while b is multiplied. What bounds it is
// its loads: without the products and their reads it took 80 % of its time. DMAs
// alone reach 14 to 17 TB/s from the L2s; the tiles bring 9 to 12 (512 x 11008 x
// 4096 in 128 x 256, four slices: 270 MB in 30 us; 77 x 5120 x 13824 in 64 x 128:
// 212 MB in 17.5, an eighth of it rows past the last), and why not more is open.
template <int BM, int BN, int WM, int WN, int S, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, WM * WN >= 8 ? 2 : 1) void ring_kernel(MmArgs a, float *part, int splits) {
    constexpr int W = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16, STEPS = MT * NT;
    constexpr int DX = BM / 8 / W, DW = BN / 8 / W, ND = DX + DW;  // DMAs (8 rows) of a wave
    static_assert(DX * 8 * W == BM && DW * 8 * W == BN && NT % 2 == 0 && BN / WN <= kBlock, "whole DMAs, one scale a wave");
    constexpr int STAGE = (BM + BN) * kBlock;
    __shared__ __align__(1024) uint8_t lds[S * STAGE];
    __shared__ __align__(16) float sx[S][W][64], sw[2][W][64];  // scales: each wave's tokens', and the weight's of two runs of blocks
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int KB = (a.K + kBlock - 1) / kBlock;
    const Place at = place<BM, BN>(a, splits);
    const int m0 = at.m0, n0 = at.n0;
    const int b0 = (int)((int64_t)KB * at.split / splits), b1 = (int)((int64_t)KB * (at.split + 1) / splits);
    const int wm0 = wave % WM * (BM / WM), wn0 = wave / WM * (BN / WN);
    const int rows_x = min(BM, a.M - m0), rows_w = min(BN, a.N - n0);
    Rsrc rx = rsrc(a.x + (int64_t)m0 * a.K, rows_x * a.K), rw = rsrc(a.w + (int64_t)n0 * a.K, rows_w * a.K);
    // lane i of a DMA fills position i % 8 of its row i / 8; rows past the last repeat it
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    int vx[DX], vw[DW];
#pragma unroll
    for (int j = 0; j < DX; ++j) vx[j] = min((wave * DX + j) * 8 + (lane >> 3), rows_x - 1) * a.K + chunk;
#pragma unroll
    for (int j = 0; j < DW; ++j) vw[j] = min((wave * DW + j) * 8 + (lane >> 3), rows_w - 1) * a.K + chunk;
    const unsigned part_x = lds_at(lds + wave * DX * 1024), part_w = lds_at(lds + BM * kBlock + wave * DW * 1024);
    unsigned lds_x = part_x, lds_w = part_w;  // the wave's part of stage 0
    auto dma = [&](int s, int b, int j) {
        const bool in = b * kBlock + chunk < a.K;  // (K ends inside the last block: zeros)
        if (j < DW)
            lds16(rw, lds_w + s * STAGE + j * 1024, in ? vw[j] : kOutside, b * kBlock);
        else
            lds16(rx, lds_x + s * STAGE + (j - DW) * 1024, in ? vx[j - DW] : kOutside, b * kBlock);
    };
    auto load = [&](int s, int b) {
#pragma unroll
        for (int j = 0; j < ND; ++j) dma(s, b, j);
    };
    // A block's scales of the tokens come with it (loads end in order: those asked
    // for later would hold up the DMAs before them: 77 x 5120 x 13824 in tiles of
    // 128 x 64 19.6 -> 16.9 us), the weight's of a run of blocks
    // (and of the one after it) during the run before.
    const int rows_s = max(min(a.M - m0 - wm0, 64), 1), nb = min((n0 + wn0) / kBlock, (a.N - 1) / kBlock);
    const float *const sx0 = a.sx + min(m0 + wm0, a.M - 1);
    auto load_scales = [&](int s, int b) { lds4(rsrc(sx0 + b * a.sx_stride, rows_s * 4), lds_at(sx[s][wave]), lane * 4); };
    auto load_run = [&](int run, int half) { lds4(rsrc(a.sw + (int64_t)nb * KB + run, min(KB - run, 64) * 4), lds_at(sw[half][wave]), lane * 4); };
    float f[MT], fn[MT], gn;
    auto read_scales = [&](int s, int half, int at) {
        gn = sw[half][wave][at];
#pragma unroll
        for (int t = 0; t < MT; ++t) fn[t] = sx[s][wave][16 * t + r];
    };
    auto take_scales = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t) f[t] = fn[t] * gn;
    };
    const int pos = r * kBlock + (c ^ (r & 7)) * 16;
    auto frag = [&](int from, int row) {
        const uint8_t *const s = lds + from;
        Frag<EXACT> v;
        v.set(*reinterpret_cast<const i32x4 *>(s + row * kBlock + pos), *reinterpret_cast<const i32x4 *>(s + row * kBlock + (pos ^ 64)));
        return v;
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0, 0, 0, 0};
    Frag<EXACT> xf[MT], wf[2];
    // Block b from stage s, whose first fragments are read, then those of b + 1
    // from `next`; block b + S - 1 to `to`, which held b - 1.
    auto block = [&](int s, int next, int to, int b, int run, int half) {
        f32x4 p[D + 1];
        const int bn = min(b + S - 1, b1 - 1);  // (past the end: the last again, unused)
        lds_x = part_x, lds_w = part_w;
        asm volatile("" : "+s"(lds_x), "+s"(lds_w));  // (added to where they are used)
#pragma unroll
        for (int i = 0; i < STEPS + D; ++i) {
            const int u = i / MT, t = i % MT;
            if (i < STEPS) {
                if (t == 0) {
                    if (u < NT - 1) {
                        wf[(u + 1) & 1] = frag(s * STAGE + BM * kBlock, wn0 + 16 * (u + 1));
                    } else {
                        // this wave's last fragments of b are read and its part of b + 1 has
                        // come; after the barrier everyone's
                        wait_loads<(S - 2) * (ND + 1), true>();
                        __builtin_amdgcn_s_barrier();
                        read_scales(next, half, b + 1 - run);
                        wf[(u + 1) & 1] = frag(next * STAGE + BM * kBlock, wn0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                p[i % (D + 1)] = mfma(wf[u & 1], xf[t]);
                if (i == 0) load_scales(to, bn);
#pragma unroll
                for (int j = 0; j < ND; ++j)
                    if (i == j * (STEPS - MT) / ND) dma(to, bn, j);
                if (u == NT - 1) xf[t] = frag(next * STAGE, wm0 + 16 * t);
            }
            if (i >= D) {
                const int j = i - D;
                acc[j % MT][j / MT] += p[j % (D + 1)] * f[j % MT];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        take_scales();
        __builtin_amdgcn_sched_barrier(0);
    };
    settle(rx, rw);
    load_run(b0, 0);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        load_scales(s, min(b0 + s, b1 - 1));
        load(s, min(b0 + s, b1 - 1));
    }
    wait_loads<(S - 2) * (ND + 1), true>();
    __builtin_amdgcn_s_barrier();
    read_scales(0, 0, 0);
    take_scales();
    wf[0] = frag(BM * kBlock, wn0);
#pragma unroll
    for (int t = 0; t < MT; ++t) xf[t] = frag(0, wm0 + 16 * t);
    constexpr int RUN = 48;
    static_assert(RUN % S == 0 && RUN < 64, "whole turns of the ring; the next run's first is among the lanes");
    for (int run = b0, half = 0; run < b1; run += RUN, half ^= 1) {
        if (run + RUN < b1) load_run(run + RUN, half ^ 1);
        for (int b = run; b < min(run + RUN, b1); b += S)
#pragma unroll
            for (int s = 0; s < S; ++s)
                if (b + s < b1) block(s, (s + 1) % S, (s + S - 1) % S, b + s, run, half);
    }
    wait_loads<0, true>();  // (no DMA after the wave's end)
    void *const out = splits > 1 ? part + (int64_t)at.split * a.M * a.N : a.y;
    const bool f32 = splits > 1 || a.f32;
    __builtin_amdgcn_s_barrier();  // (the stages are read: each wave turns its sums there)
    static_assert(S * STAGE >= W * 16 * NT * 64, "a place for each wave");
    i32x4 *const turn = reinterpret_cast<i32x4 *>(lds) + wave * (NT * 64);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = m0 + wm0 + 16 * t, n = n0 + wn0, rows = a.M - m;
        if (f32 && a.N % 4 == 0)
            turned<float, 16>(turn, acc[t], static_cast<float *>(out), m, rows, n, a.N);
        else if (!f32 && a.N % 8 == 0)
            turned<_Float16, 16>(turn, acc[t], static_cast<_Float16 *>(out), m, rows, n, a.N);
        else if (r < rows)
#pragma unroll
            for (int u = 0; u < NT; ++u) store_n4(out, f32, m + r, n + 16 * u + 4 * c, a.N, acc[t][u]);
    }
}

// y of the slices' partial sums, four neighbours a thread, in slice order.
__global__ __launch_bounds__(256) void reduce_kernel(const float *part, void *y, int64_t n, int splits, int f32) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if ((n & 3) == 0) {
        if (i >= n) return;
        f32x4 v = *reinterpret_cast<const f32x4 *>(part + i);
        for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4 *>(part + s * n + i);
        if (f32)
            *reinterpret_cast<f32x4 *>(static_cast<float *>(y) + i) = v;
        else
            *reinterpret_cast<half4 *>(static_cast<_Float16 *>(y) + i) = half4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
        return;
    }
    for (int64_t j = i; j < i + 4 && j < n; ++j) {
        float v = part[j];
        for (int s = 1; s < splits; ++s) v += part[s * n + j];
        if (f32)
            static_cast<float *>(y)[j] = v;
        else
            static_cast<_Float16 *>(y)[j] = (_Float16)v;
    }
}

// ------------------------------------------------------------ 256 x 256, f16 y
// Eight waves of 64 x 128, two stages, the 8-bit instruction. x and each half of
// w lie apart: once every wave has read x and the first half of block b (the
// middle of the block), their places take block b + 2, the second half's at the
// end, so that a DMA has 1 to 1.4 blocks' time (all of it after the end: 0.6 to
// 0.9; 4096 x 4096 x 22016 373 -> 354 us).
//
// A workgroup for each CU takes tiles until none is left, and their blocks of k
// are one stream: the next tile's first blocks come during the last ones of
// this, and its products run while y is on its way. The tiles that are left for
// the last round are halved along the tokens where that gives every CU one.
// Against a workgroup a tile: 4096 x 4096 x 22016 (5.4 tiles a CU) 353 -> 333 us,
// 512 x 11008 x 4096 108 -> 98, 4096 x 11008 x 4096 (exactly one) 158 -> 161,
// 8192^3 (four) 445 -> 455: the stream costs some 2 % where the tiles come out even.
constexpr int WIDE = 256;

struct Item {
    int m0, n0, rows;  // rows 0: none
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }  // (a quotient comes from the vector unit)

__global__ __launch_bounds__(512, 2) void wide_kernel(MmArgs a) {
    constexpr int WM = 4, WN = 2, W = WM * WN, MT = WIDE / WM / 16, NT = WIDE / WN / 16, HN = WIDE / WN / 2;
    constexpr int DX = WIDE / 8 / W, DW = WIDE / 16 / W;  // DMAs (8 rows) of a wave: of x, of each half of w
    constexpr int STEPS = MT * NT, MID = STEPS / 2, LAST = MT * (NT - 1);
    static_assert(MID + DX + DW < LAST && DW < MT, "a block's DMAs fit between its barriers");
    // two places each for x and the halves of w
    constexpr int XP = WIDE * kBlock, WP = WIDE / 2 * kBlock, X0 = 0, X1 = XP, A0 = 2 * XP, A1 = A0 + WP, B0 = A1 + WP, B1 = B0 + WP;
    __shared__ __align__(1024) uint8_t lds[B1 + WP];
    __shared__ __align__(16) float sx[2][W][64], sw[2][W][64];  // scales: of two blocks each wave's tokens', of two runs of 64 blocks w's
    __shared__ __align__(1024) i32x4 turn_of[W][8 * 16];  // eight tokens of a wave's 128 columns, on their way to y
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int KB = (a.K + kBlock - 1) / kBlock;  // (at least 2)
    // (waves w and w + 4 share a SIMD: of half a tile each SIMD has one)
    const int wn = wave % WN, wm0 = wave / WN * (WIDE / WM), wn0 = wn * (WIDE / WN);

    // This workgroup's tiles: an XCD takes a run of them, its CUs one after the other.
    const int tm = (a.M + WIDE - 1) / WIDE, tn = (a.N + WIDE - 1) / WIDE, tiles = tm * tn;
    const int xcd = blockIdx.x % 8, slot = blockIdx.x / 8, slots = gridDim.x / 8;
    const int mine = tiles / 8 + (xcd < tiles % 8 ? 1 : 0), base = xcd * (tiles / 8) + min(xcd, tiles % 8);
    const int full = uniform(mine / slots), left = mine - full * slots;
    const bool halves = 2 * left <= slots;
    const int items = full + (slot < (halves ? 2 * left : left) ? 1 : 0);
    auto item = [&](int i) {
        if (i >= items) return Item{0, 0, 0};
        const bool half = i == full && halves;
        const int tile = base + i * slots + (half ? slot / 2 : slot);
        const int panel = uniform(tile / (kPanel * tn)), at = tile - panel * kPanel * tn, wide = min(kPanel, tm - panel * kPanel);
        const int column = uniform(at / wide), m0 = (panel * kPanel + at - column * wide) * WIDE + (half ? slot % 2 * (WIDE / 2) : 0);
        return Item{m0, column * WIDE, max(min(half ? WIDE / 2 : WIDE, a.M - m0), 0)};
    };

    // What the DMAs read: a lane's first row of x, and of w (each wave column's
    // first 64 rows are the first half); rows past the tile's last lie outside the resources.
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    unsigned vx, vw;
    Rsrc rx, rw;
    const unsigned part_x = lds_at(lds + wave * DX * 1024), part_w = lds_at(lds + wave * DW * 1024);  // the wave's part of a place
    unsigned lds_x = part_x, lds_w = part_w;
    auto point = [&](Item t) {
        vx = vw = kOutside;
        if (t.rows == 0) return;  // (the resources stay: an offset is outside only while they hold the uniform offset)
        rx = rsrc(a.x + (int64_t)t.m0 * a.K, t.rows * a.K), rw = rsrc(a.w + (int64_t)t.n0 * a.K, min(WIDE, a.N - t.n0) * a.K);
        const int l = wave * DW * 8;
        vx = (wave * DX * 8 + (lane >> 3)) * a.K + chunk;
        vw = (l / HN * (2 * HN) + l % HN + (lane >> 3)) * a.K + chunk;
        settle(rx, rw);
    };
    static_assert(HN % (DW * 8) == 0, "a wave's rows of w are neighbours");
    auto dma = [&](Rsrc rs, unsigned to, unsigned v, int b) { lds16(rs, to, b * kBlock + chunk < a.K ? v : (unsigned)kOutside, b * kBlock); };
    auto dma_x = [&](int to, int b, int j) { dma(rx, lds_x + to + j * 1024, vx + j * 8 * a.K, b); };
    auto dma_a = [&](int to, int b, int j) { dma(rw, lds_w + to + j * 1024, vw + j * 8 * a.K, b); };
    auto dma_b = [&](int to, int b, int j) { dma(rw, lds_w + to + j * 1024, vw + (HN + j * 8) * a.K, b); };
    // The scales of block b of a tile: its wave's 64 tokens' to sx[q]; at the first
    // of 64 blocks w's of all of them to the other half of sw.
    int half = 1;
    auto load_scales = [&](Item t, int b, int q) {
        const int rows = max(min(a.M - t.m0, WIDE), 1), nb = min((t.n0 + wn0) / kBlock, (a.N - 1) / kBlock);
        lds4(rsrc(a.sx + b * a.sx_stride + t.m0, rows * 4), lds_at(sx[q][wave]), (wm0 + lane) * 4);
        if (b % 64 == 0) {
            half ^= 1;
            lds4(rsrc(a.sw + (int64_t)nb * KB + b, min(KB - b, 64) * 4), lds_at(sw[half][wave]), lane * 4);
        }
    };
    float f[MT], fn[MT], gn;
    auto read_scales = [&](int b, int q) {
        gn = sw[half][wave][b % 64];
#pragma unroll
        for (int t = 0; t < MT; ++t) fn[t] = sx[q][wave][16 * t + r];
    };
    auto take_scales = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t) f[t] = fn[t] * gn;
    };
    const int pos = r * kBlock + (c ^ (r & 7)) * 16;
    auto frag = [&](int from, int row) {
        const uint8_t *const s = lds + from + row * kBlock;
        Frag<false> v;
        v.set(*reinterpret_cast<const i32x4 *>(s + pos), *reinterpret_cast<const i32x4 *>(s + (pos ^ 64)));
        return v;
    };
    f32x4 acc[MT][NT];
    Frag<false> xf[MT], wf[2];
    Item now = item(0);
    if (now.rows == 0) return;  // (the whole workgroup)
    int i_item = 0, b = 0;
    bool active = wm0 < now.rows;
    auto clear = [&] {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0, 0, 0, 0};
    };

    // Block b from xs, was, wbs, whose first fragments are read, then the next
    // block's from xn and wan; the one after that to b's places.
    auto block = [&](int q, int xs, int was, int wbs, int xn, int wan) {
        int b2 = b + 2;
        if (b2 >= KB) {
            b2 -= KB;
            if (b2 == 0) point(item(i_item + 1));
        }
        lds_x = part_x, lds_w = part_w;
        asm volatile("" : "+s"(lds_x), "+s"(lds_w));  // (added to where they are used: 24 places are too many to keep)
        const bool last = b + 1 == KB;
        auto next_scales = [&] { load_scales(last ? item(i_item + 1) : now, last ? 0 : b + 1, q ^ 1); };
        if (active) {
            f32x4 p[D + 1];
#pragma unroll
            for (int i = 0; i < STEPS + D; ++i) {
                const int u = i / MT, t = i % MT;
                if (i < STEPS) {
                    if (t == 0) {
                        if (i == MID) {  // everyone has read x and the first half of w
                            wait_lds();
                            __builtin_amdgcn_s_barrier();
                        }
                        if (u == NT - 1) {  // everyone has read the rest, and the next block has come
                            wait_loads<DX + DW, true>();
                            __builtin_amdgcn_s_barrier();
                            read_scales(last ? 0 : b + 1, q ^ 1);
                            wf[(u + 1) & 1] = frag(wan, wn * HN);
                        } else {
                            wf[(u + 1) & 1] = u + 1 < NT / 2 ? frag(was, wn * HN + 16 * (u + 1)) : frag(wbs, wn * HN + 16 * (u + 1 - NT / 2));
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    p[i % (D + 1)] = mfma(wf[u & 1], xf[t]);
                    if (i == 1) next_scales();
                    if (i > MID && i - MID - 1 < DX) dma_x(xs, b2, i - MID - 1);
                    if (i > MID + DX && i - MID - DX - 1 < DW) dma_a(was, b2, i - MID - DX - 1);
                    if (i > LAST && i - LAST - 1 < DW) dma_b(wbs, b2, i - LAST - 1);
                    if (u == NT - 1) xf[t] = frag(xn, wm0 + 16 * t);
                }
                if (i >= D) {
                    const int j = i - D;
                    acc[j % MT][j / MT] += p[j % (D + 1)] * f[j % MT];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {  // (none of the wave's rows are in the tile)
            next_scales();
            wait_lds();
            __builtin_amdgcn_s_barrier();
            settle(rx, rw);
#pragma unroll
            for (int j = 0; j < DX; ++j) dma_x(xs, b2, j);
#pragma unroll
            for (int j = 0; j < DW; ++j) dma_a(was, b2, j);
            wait_loads<DX + DW, true>();
            __builtin_amdgcn_s_barrier();
            settle(rx, rw);
#pragma unroll
            for (int j = 0; j < DW; ++j) dma_b(wbs, b2, j);
            read_scales(last ? 0 : b + 1, q ^ 1);
            wf[0] = frag(wan, wn * HN);
#pragma unroll
            for (int t = 0; t < MT; ++t) xf[t] = frag(xn, wm0 + 16 * t);
        }
        take_scales();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto write = [&] {
        const int n = now.n0 + wn0;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int m = now.m0 + wm0 + 16 * t, rows = now.rows - wm0 - 16 * t;
            if (a.N % 8 == 0)
                turned<_Float16, 8>(turn_of[wave], acc[t], static_cast<_Float16 *>(a.y), m, rows, n, a.N);
            else if (r < rows)
#pragma unroll
                for (int u = 0; u < NT; ++u) store_n4(a.y, false, m + r, n + 16 * u + 4 * c, a.N, acc[t][u]);
        }
    };
    // After a block: whether it was the last of all.
    auto done = [&] {
        if (++b < KB) return false;
        if (active) write();
        if (++i_item == items) return true;
        now = item(i_item);
        if (now.rows == 0) return true;  // (half a tile past the last token)
        active = wm0 < now.rows;
        b = 0;
        clear();
        return false;
    };

    point(now);
    auto load = [&](int xs, int was, int wbs, int b) {
#pragma unroll
        for (int j = 0; j < DX; ++j) dma_x(xs, b, j);
#pragma unroll
        for (int j = 0; j < DW; ++j) dma_a(was, b, j);
#pragma unroll
        for (int j = 0; j < DW; ++j) dma_b(wbs, b, j);
    };
    load_scales(now, 0, 0);
    settle(rx, rw);
    load(X0, A0, B0, 0);
    load(X1, A1, B1, 1);
    clear();
    wait_loads<DX + 2 * DW, true>();
    __builtin_amdgcn_s_barrier();
    read_scales(0, 0);
    take_scales();
    wf[0] = frag(A0, wn * HN);
#pragma unroll
    for (int t = 0; t < MT; ++t) xf[t] = frag(X0, wm0 + 16 * t);
    while (true) {
        block(0, X0, A0, B0, X1, A1);
        if (done()) break;
        block(1, X1, A1, B1, X0, A0);
        if (done()) break;
    }
    wait_loads<0, true>();  // (no DMA after the wave's end)
}

// ------------------------------------------------------------------ the choice
// Estimated times (us), fitted to calls of 65 to 4096 tokens, K 1024 to 14336, N
// 1024 to 22016, weights cold or in the last cache: a launch, then for each round
// of workgroups a start and end and K's blocks, which take longer where all CUs
// load at once; slices add their sums' way through memory. Over 171 such shapes
// the chosen tile and slices take 0.2 to 0.5 % longer at the mean than the best
// ones (three cards, cold and not), 17 % at the most.
enum Kind { MV, R64x64, R64x128, R128x64, R128x128, R128x256, R256x128, R256x256 };
struct Rate {
    double few, all;  // a block on few of the CUs, on all (0: not built)
};
struct Tile {
    Kind kind;
    int bm, bn;
    double ends;  // a round's start and end
    Rate by8, by16;
};
constexpr Tile kTiles[] = {
    {R64x64, 64, 64, 1.7, {0.28, 0.29}, {0.44, 0.44}},     {R64x128, 64, 128, 2.9, {0.30, 0.38}, {0.59, 0.63}},
    {R128x64, 128, 64, 3.1, {0.33, 0.37}, {0.64, 0.63}},   {R128x128, 128, 128, 3.8, {0.44, 0.61}, {0.97, 1.02}},
    {R128x256, 128, 256, 4.2, {0.81, 0.90}, {0, 0}},       {R256x128, 256, 128, 3.6, {0, 0}, {1.63, 1.76}},
    {R256x256, 256, 256, 3.1, {1.06, 1.06}, {0, 0}},
};

struct Plan {
    Kind kind;
    int splits;
};

// Whether the f16 instruction sums, whose products are exact.
bool exact_sums(const st_context *ctx, const MmArgs &a) { return a.f32 || a.M <= 64 || st::tune(ctx, ST_TUNE_FP8_EXACT, 0) > 0; }

Plan plan(const st_context *ctx, const MmArgs &a) {
    const int forced = st::tune(ctx, ST_TUNE_FP8_TILE, -1), slices = st::tune(ctx, ST_TUNE_FP8_SPLITS, -1);
    Plan best{MV, 1};
    const bool can_mv = a.M <= 64, exact = exact_sums(ctx, a);
    if (can_mv && (forced == MV || (forced < 0 && a.M <= 48))) return best;
    double least = can_mv ? mv_us(ctx, a) : 1e30;
    const int KB = blocks(a.K);
    auto tiles_of = [&](const Tile &t) { return (int64_t)((a.M + t.bm - 1) / t.bm) * ((a.N + t.bn - 1) / t.bn); };
    // (a launch is of fewer than 2^32 threads: of the sizes that the call permits, exact sums in tiles of 64 x 64 can be more)
    auto fits = [&](const Tile &t, int s) {
        return tiles_of(t) * s * (t.kind == R64x64 && !exact ? 256 : 512) <= 0xFFFFFFFF && (s == 1 || (int64_t)a.M * a.N < (int64_t)1 << 33);
    };
    // (the 256 x 256 kernel brings two blocks of K at once)
    auto built = [&](const Tile &t) { return (exact ? t.by16 : t.by8).all != 0 && (t.kind != R256x256 || KB > 1) && fits(t, 1); };
    bool force = false;
    for (const Tile &t : kTiles) force |= t.kind == forced && built(t);
    if (force) least = 1e30;
    for (const Tile &t : kTiles) {
        if (!built(t) || (force ? t.kind != forced : a.M <= 64 && t.bm != 64)) continue;
        const Rate rate = exact ? t.by16 : t.by8;
        const int64_t tiles = tiles_of(t);
        for (int s = 1; s <= 8 && s <= KB; s *= 2) {
            const double sums = 4.0 * s * a.M * a.N;
            if (s > 1 && (t.kind == R256x256 || sums > (double)ctx->ws_bytes || !fits(t, s))) break;
            const int64_t rounds = tiles * s / ctx->num_cus;
            const double rest = (double)(tiles * s % ctx->num_cus) / ctx->num_cus;
            const auto round = [&](double on) { return t.ends + (KB + s - 1) / s * std::max(rate.few, rate.all * on); };
            const double us = 2.5 + rounds * round(1.0) + (rest > 0 ? round(rest) : 0.0) + (s > 1 ? 2.7 + sums / 4.1e6 : 0.0);
            if (force && slices > 0 ? s <= slices : us < least) least = us, best = {t.kind, s};
        }
    }
    return best;
}

template <int BM, int BN, int WM, int WN, int S, bool EXACT>
void run_ring(st_context *ctx, const MmArgs &a, int splits) {
    const dim3 grid((unsigned)((a.M + BM - 1) / BM * ((a.N + BN - 1) / BN) * splits));
    st::launch(ctx, ring_kernel<BM, BN, WM, WN, S, EXACT>, grid, dim3(64 * WM * WN), 0, a, ctx->ws, splits);
}

int run(st_context *ctx, const MmArgs &a, Plan p) {
    const bool exact = exact_sums(ctx, a);
    const char *name = "fp8_ring_kernel";
    switch (p.kind) {
        case MV: return mv(ctx, a);
        case R64x64:  // (f16 instruction: two waves a SIMD, so that one converts while the other multiplies: 256 x 2560 x 2560 15.2 -> 13.9 us)
            exact ? run_ring<64, 64, 4, 2, 4, true>(ctx, a, p.splits) : run_ring<64, 64, 2, 2, 4, false>(ctx, a, p.splits);
            break;
        case R64x128:
            exact ? run_ring<64, 128, 2, 4, 4, true>(ctx, a, p.splits) : run_ring<64, 128, 2, 4, 4, false>(ctx, a, p.splits);
            break;
        case R128x64:
            exact ? run_ring<128, 64, 4, 2, 4, true>(ctx, a, p.splits) : run_ring<128, 64, 4, 2, 4, false>(ctx, a, p.splits);
            break;
        case R128x128:
            exact ? run_ring<128, 128, 4, 2, 4, true>(ctx, a, p.splits) : run_ring<128, 128, 4, 2, 4, false>(ctx, a, p.splits);
            break;
        case R128x256: run_ring<128, 256, 2, 4, 3, false>(ctx, a, p.splits); break;
        case R256x128: run_ring<256, 128, 4, 2, 3, true>(ctx, a, p.splits); break;
        case R256x256: {
            st::launch(ctx, wide_kernel, dim3((unsigned)(std::max(ctx->num_cus, 8) / 8 * 8)), dim3(512), 0, a);
            name = "fp8_wide_kernel";
        }
    }
    if (int rc = st::launch_check(name)) return rc;
    if (p.splits == 1) return ST_OK;
    const int64_t n = (int64_t)a.M * a.N;
    st::launch(ctx, reduce_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, (const float *)ctx->ws, a.y, n, p.splits, a.f32);
    return st::launch_check("fp8_reduce_kernel");
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
    // (a launch is of fewer than 2^32 threads: of at most 64 tokens 256 for 32 columns, or 512 for 64; of more plan() takes
    // tiles that fit, and 128 x 128 for 512 always does)
    if (M > kMostRows || N > kMostRows || (int64_t)blocks(M) * blocks(N) >= (1 << 22))
        return st::fail(ST_ERR_SHAPE, "%s: M=%d, N=%d (each at most 2^28, fewer than 2^22 blocks of 128 x 128)", fn, M, N);
    if (!st::aligned16(x) || !st::aligned16(w) || !st::aligned16(y) || !aligned4(x_scale) || !aligned4(w_scale))
        return st::fail(ST_ERR_ALIGN, "%s: pointers must be 16-byte aligned (scales: 4)", fn);
    if (one_of(y, {x, x_scale, w, w_scale})) return st::fail(ST_ERR_INVALID, "%s: y in an input's buffer", fn);
    const MmArgs a{x, w, x_scale, w_scale, y, scale_stride, M, K, N, y_dtype == ST_F32};
    const st::OnDevice on(ctx);
    if (on.error != hipSuccess) return st::hip_fail(on.error, fn);
    return run(ctx, a, plan(ctx, a));
}
