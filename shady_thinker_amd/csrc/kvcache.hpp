// The paged key-value cache's layout (st_kv_cache) on the device, and the
// argument checks its entry points share.
#pragma once

#include "common.hpp"

namespace st {
namespace kv {

constexpr int kTile = 16;  // tokens of a tile

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Kernel arguments: the cache, page sizes as shifts.
struct Cache {
    void *k, *v;
    float *k_scale, *v_scale;
    int num_pages, page_shift, heads;

    __host__ __device__ int tiles_shift() const { return page_shift - 4; }
    // (page, head)'s first tile and first scale; 64 bits: a cache has more
    // than 2^32 elements
    __host__ __device__ int64_t tile(int page, int head, int tile_of_page) const {
        return (((int64_t)page * heads + head) << tiles_shift()) + tile_of_page;
    }
    __host__ __device__ int64_t scale(int page, int head, int place) const {
        return (((int64_t)page * heads + head) << page_shift) + place;
    }
};

// Where place t of a tile lies in the value pieces: its half, its place in it.
__host__ __device__ constexpr int v_half(int t) { return (t >> 2) & 1; }
__host__ __device__ constexpr int v_place(int t) { return (t & 3) | ((t >> 3) << 2); }
__host__ __device__ constexpr int v_token(int half, int place) { return (place >> 2) * 8 + half * 4 + (place & 3); }

// Eight int8 (two dwords) as exact f16: v + 128 under the exponent of 1024,
// less 1152.
__device__ __forceinline__ half8 i8_to_half8(u32x2 w) {
    const unsigned a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;  // v + 128
    const unsigned bias = 0x64646464u;
    const u32x4 r = {__builtin_amdgcn_perm(bias, a, 0x04010400u), __builtin_amdgcn_perm(bias, a, 0x04030402u),
                     __builtin_amdgcn_perm(bias, b, 0x04010400u), __builtin_amdgcn_perm(bias, b, 0x04030402u)};
    const _Float16 c = (_Float16)1152.0f;
    const half8 c8 = {c, c, c, c, c, c, c, c};
    return __builtin_bit_cast(half8, r) - c8;
}

// ST_OK and the device form, or an error.
inline int check_cache(const char *fn, const st_kv_cache *c, Cache *out) {
    if (!c || !c->k || !c->v) return fail(ST_ERR_INVALID, "%s: no cache", fn);
    if (c->dtype != ST_F16 && c->dtype != ST_I8) return fail(ST_ERR_INVALID, "%s: cache dtype %d (f16 or int8)", fn, c->dtype);
    if (c->dtype == ST_I8 && (!c->k_scale || !c->v_scale)) return fail(ST_ERR_INVALID, "%s: an int8 cache needs its scales", fn);
    int shift = 4;
    while (shift < 8 && (1 << shift) != c->page_size) ++shift;
    if ((1 << shift) != c->page_size)
        return fail(ST_ERR_SHAPE, "%s: page size %d (16, 32, 64, 128 or 256)", fn, c->page_size);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(ST_ERR_SHAPE, "%s: head dim %d (64, 128 or 256)", fn, c->head_dim);
    if (c->num_pages < 1 || c->num_pages > (0x7FFFFFFF >> shift) || c->n_kv_heads < 1 || c->n_kv_heads > 1024)
        return fail(ST_ERR_SHAPE, "%s: %d pages of %d heads (slots are 32-bit, at most 1024 heads)", fn, c->num_pages, c->n_kv_heads);
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
        return fail(ST_ERR_ALIGN, "%s: cache pointers must be 16-byte aligned", fn);
    *out = Cache{c->k, c->v, c->k_scale, c->v_scale, c->num_pages, shift, c->n_kv_heads};
    return ST_OK;
}

}  // namespace kv
}  // namespace st
