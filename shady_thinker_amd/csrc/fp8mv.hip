// e4m3 rows times an e4m3 weight (st_fp8_gemm), up to 64 tokens: bound by the
// weight's bytes.
//
// A workgroup takes 16 NT columns, its W waves every W-th block of 128 k. A
// wave brings its blocks of both operands and their scales to LDS by DMA, S of
// them ahead, in slots of its own: it waits for its own loads only (and not for
// the other slots', whose number the waits count), and the waves meet once, when
// their sums are added in order. A row's 128 bytes are eight 16-byte chunks,
// chunk j of row r at j ^ (r % 8), so that fragment reads hit every bank once.
// e4m3 goes to f16 exactly and f16 products are exact in the matrix instruction's
// f32 sums (the 8-bit instruction's are not, see fp8mm.hip).
//
// Workgroups begin at different blocks of k: side by side at the same one, their
// rows' 128 bytes lie K apart, where K is a multiple of a few KiB in few channels
// of memory and caches (one token 8192 x 8192: 17.2 -> 13.5 us, 4096 x 22016 18.9
// -> 17.2). One token now takes (cold weights, in a captured graph) 2048 x 2048
// 3.4 us, 4096 x 4096 5.7, 11008 x 4096 10.5 (4.3 TB/s), 8192 x 8192 13.6 (4.9),
// 4096 x 22016 17.1 (5.3).
//
// Sizes of columns and waves (MI355X, cold weights; us of (NT, W), measured with
// two slots each and the same first block):
//   16 columns, 8 waves: up to a tile a CU (one token 4096 x 4096: (1, 8) 7.1, (2, 8) 6.9, (2, 4) 8.3); a workgroup a
//   CU, so three slots and more where they fit (11008 x 4096: 13.4 -> 10.8; 16 waves of three: 11.7)
//   16 columns, 4 or 8 waves, several workgroups a CU: up to 1.2
//   32 columns, 8 waves: up to 2 (4096 x 8192: (2, 8) 9.6, (1, 8) 10.9, (2, 4) 10.1), three slots (8192 x 8192: 18.2 -> 17.2)
//   then four waves and 32, 48 or 64 columns, whichever leaves the fullest CU
//   the fewest (4096 x 22016: 48 20.2, 32 20.7, 64 21.1; 28672: 64 24.4, 32 26.3, 48 28.2);
//   several workgroups a CU, so two slots (three, 48 columns: 15.8 -> 18.2, the weights in the last cache)
#include "fp8mm.hpp"

#include <algorithm>

namespace {

using namespace st::f8;

// X8: at most eight tokens, one DMA of x for a block. S: slots of a wave.
template <int MT, bool X8, int NT, int W, int S>
__global__ __launch_bounds__(64 * W) void mv_kernel(MmArgs a) {
    constexpr int XD = X8 ? 1 : 2 * MT, ND = 2 * NT + XD;  // DMAs of a slot, eight rows each
    constexpr int SLOT = ND * 1024, PART = W * SLOT;
    constexpr bool CROSS = NT == 3;  // columns on both sides of a border between the weight's blocks
    static_assert(!X8 || MT == 1, "eight tokens are one fragment");
    static_assert(SLOT >= MT * NT * 1024, "the waves' sums fit the first slots");
    __shared__ __align__(1024) uint8_t lds[S * PART];
    __shared__ __align__(16) float sx[S][W][64], sw[CROSS ? 2 : 1][W][64];  // scales: the slots' tokens', the weight's of each wave's next 64 blocks
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, c = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT);
    const int KB = (a.K + kBlock - 1) / kBlock;
    const int rows_w = min(16 * NT, a.N - n0);
    Rsrc rw = rsrc(a.w + (int64_t)n0 * a.K, rows_w * a.K), rx = rsrc(a.x, a.M * a.K);
    const int nb = n0 / kBlock, nb_last = (a.N - 1) / kBlock, cross = (nb + 1) * kBlock - n0;  // columns before the border
    // lane i of a DMA fills position i % 8 of its row i / 8; rows past the last repeat it
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    int vw[2 * NT], vx[XD];
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) vw[j] = min(8 * j + (lane >> 3), rows_w - 1) * a.K + chunk;
#pragma unroll
    for (int j = 0; j < XD; ++j) vx[j] = min(8 * j + (lane >> 3), a.M - 1) * a.K + chunk;
    const unsigned part = lds_at(lds + wave * SLOT);
    const int mine = (KB - wave + W - 1) / W;
    // (the block it begins with: another one for the XCDs' workgroups, and within an XCD)
    const int first = mine > 1 && mine <= 64 ? (int)((blockIdx.x / 8 + blockIdx.x) % mine) : 0;
    auto turn = [&](int i) { return i + first < mine ? i + first : i + first - mine; };
    auto load = [&](int s, int i) {  // the wave's block i to slot s
        if (i >= mine) return;
        const int b = wave + turn(i) * W;
        const bool in = b * kBlock + chunk < a.K;  // (K ends inside the last block)
        lds4(rsrc(a.sx + b * a.sx_stride, a.M * 4), lds_at(sx[s][wave]), lane * 4);
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) lds16(rw, part + s * PART + j * 1024, in ? vw[j] : kOutside, b * kBlock);
#pragma unroll
        for (int j = 0; j < XD; ++j) lds16(rx, part + s * PART + (2 * NT + j) * 1024, in ? vx[j] : kOutside, b * kBlock);
    };
    auto load_sw = [&](int i) {  // the weight's scales of the wave's blocks i to i + 63
        const int v = (wave + (i + lane) * W) * 4;
        lds4(rsrc(a.sw + (int64_t)nb * KB, KB * 4), lds_at(sw[0][wave]), v);
        if constexpr (CROSS) lds4(rsrc(a.sw + (int64_t)min(nb + 1, nb_last) * KB, KB * 4), lds_at(sw[1][wave]), v);
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
    auto step = [&](int s, int i) {
        const uint8_t *const at = lds + s * PART + wave * SLOT;
        if (i % 64 == 0 && i) {
            load_sw(i);
            wait_loads<0, false>();
        }
        // (the other slots' may be in flight)
        static_assert(S <= 4, "a wait for each number of them");
        const int others = min(S - 1, mine - 1 - i);
        if (others == 0) wait_loads<0, false>();
        if (others == 1) wait_loads<ND + 1, false>();
        if (others == 2) wait_loads<2 * (ND + 1), false>();
        if (others == 3) wait_loads<3 * (ND + 1), false>();
        const int is = turn(i) % 64;
        const float w0 = sw[0][wave][is], w1 = CROSS ? sw[CROSS][wave][is] : 0.0f;
        Frag<true> w[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) w[u] = frag(at + u * 2048, pos);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const Frag<true> x = frag(at + (2 * NT + 2 * t) * 1024, xpos);
            const float f = sx[s][wave][16 * t + r];
#pragma unroll
            for (int u = 0; u < NT; ++u) acc[t][u] += mfma(w[u], x) * (f * (CROSS && 16 * u >= cross ? w1 : w0));
        }
        wait_lds();  // (the fragments are read: the slot may be filled)
        load(s, i + S);
    };
    settle(rw, rx);
    load_sw(0);
#pragma unroll
    for (int s = 0; s < S; ++s) load(s, s);
    for (int i = 0; i < mine; i += S)
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (i + s < mine) step(s, i + s);
    wait_loads<0, true>();
    __syncthreads();
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) sums[(wave * MT * NT + t * NT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * NT * 64; i += 64 * W) {
        const int q = i >> 6, l = i & 63;
        f32x4 v = sums[i];
#pragma unroll
        for (int w = 1; w < W; ++w) v += sums[w * MT * NT * 64 + i];
        const int m = 16 * (q / NT) + (l & 15);
        if (m < a.M) store_n4(a.y, a.f32, m, n0 + 16 * (q % NT) + 4 * (l >> 4), a.N, v);
    }
}

struct Shape {
    int nt, w;
    bool deep;  // a workgroup a CU: its slots may fill LDS
};

Shape shape(const st_context *ctx, const MmArgs &a) {
    const int tiles = (a.N + 15) / 16, cus = ctx->num_cus;
    if (tiles <= cus) return {1, 8, true};
    if (a.M > 32) return {2, 4, false};
    if (5 * tiles <= 6 * cus) return {1, a.M <= 16 ? 8 : 4, false};  // (several workgroups a CU: no second round for a few)
    if (tiles <= 2 * cus) return {2, 8, false};
    Shape best{2, 4, false};
    int least = 1 << 30;
    for (int nt = 2; nt <= (a.M <= 16 ? 4 : 3); ++nt) {
        const int cost = ((tiles + nt - 1) / nt + cus - 1) / cus * nt;  // tiles of the fullest CU
        if (cost <= least) least = cost, best.nt = nt;
    }
    return best;
}

template <int MT, bool X8, int NT, int W, int S = 2>
void run(st_context *ctx, const MmArgs &a) {
    st::launch(ctx, mv_kernel<MT, X8, NT, W, S>, dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT))), dim3(64 * W), 0, a);
}

template <int MT, bool X8>
void by_shape(st_context *ctx, const MmArgs &a, Shape s) {
    if constexpr (MT == 4) {
        s.nt == 1 ? run<MT, X8, 1, 7, 2>(ctx, a) : run<MT, X8, 2, 4, 2>(ctx, a);
    } else if constexpr (MT == 3) {
        s.nt == 1 ? run<MT, X8, 1, 8>(ctx, a) : run<MT, X8, 2, 4>(ctx, a);
    } else {
        if constexpr (MT == 1) {
            if (s.deep) return run<MT, X8, 1, 8, 4>(ctx, a);
            if (s.nt == 1) return run<MT, X8, 1, 8>(ctx, a);
            if (s.nt == 4) return run<MT, X8, 4, 4>(ctx, a);
        } else {
            if (s.nt == 1) return s.deep ? run<MT, X8, 1, 8, 3>(ctx, a) : run<MT, X8, 1, 4>(ctx, a);
        }
        if constexpr (MT == 1) if (s.nt == 2 && s.w == 8) return run<MT, X8, 2, 8, 3>(ctx, a);
        if (s.nt == 2) return s.w == 8 ? run<MT, X8, 2, 8>(ctx, a) : run<MT, X8, 2, 4>(ctx, a);
        run<MT, X8, 3, 4>(ctx, a);
    }
}

}  // namespace

namespace st {
namespace f8 {

// Of 49 to 64 tokens (fewer always come here): a start, and the fullest CUs'
// blocks, which come faster where CUs are idle (fitted at K 1024 to 14336, N 1024
// to 22016).
double mv_us(const st_context *ctx, const MmArgs &a) {
    const Shape s = shape(ctx, a);
    const double rounds = (double)((a.N + 15) / 16) / s.nt / ctx->num_cus;
    return 2.3 + std::max(0.6, rounds) * blocks(a.K) * (s.nt == 1 ? 0.205 : rounds <= 1.0 ? 0.28 : 0.345);
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
