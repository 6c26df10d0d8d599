/*
 * shady_hip.h: C ABI of the MI355X (gfx950) quantized-linear backend.
 *
 * Drop-in for the GPTQ linear path of tmzt/shady-thinker: the Rust host keeps
 * `Model::gptq_matvec` / `Model::fused_silu_gptq_down` and its call sites
 * (src/model.rs:357-408, called from Model::forward src/model.rs:669-969 and
 * InferenceSession::generate_tokens src/inference.rs:72-131); inside, those
 * helpers call these functions instead of GpuContext::dispatch
 * (src/gpu.rs:188-234) with a WGSL shader.
 *
 * Conventions
 *  - Plain pointers and sizes only. Every tensor argument is a device pointer
 *    (from st_alloc or any hipMalloc allocation) unless the name says `host`.
 *  - Layouts are the reference's, unmodified (src/weights.rs:398 uploads the
 *    GPTQ safetensors bytes verbatim):
 *      qweight u32[K/8, N]  eight 4-bit values per word along K, low nibble =
 *                           lowest k (src/shaders/gptq_matvec.wgsl:51-59)
 *      scales  f16[K/gs, N] (read as u32 pairs by the WGSL, :41-45)
 *      qzeros  u32[K/gs, N/8] eight zero points per word along N (AutoGPTQ;
 *                           dropped by the reference, src/weights.rs:372-374)
 *      x       [M, K] row-major, y [M, N] row-major (M = 1 for decode)
 *    INT8 weights (no reference counterpart) are int8[N, K] row-major with
 *    f32 per-output-channel scales[N].
 *  - Every call is asynchronous and ordered on the context's stream, like the
 *    reference's single queue (src/gpu.rs:176-242). st_flush() waits.
 *  - Return value: ST_OK (0) or an st_status code; st_last_error() gives the
 *    message for the calling thread. The Rust side `expect`s on non-zero to
 *    keep the reference's panic semantics.
 *  - A context is not thread-safe (the reference serialises through
 *    `&mut GpuContext`).
 *  - No call allocates. The context's workspace (st_context_reserve_workspace)
 *    holds the prefill GEMM's pre-processed A and split-K partials, the
 *    split-K partials of multi-token (M > 1) decode calls on linears with few
 *    16-column tiles, and the split f32 x of multi-token GPTQ calls with
 *    act-order; one-token decode calls of linears use none. Attention and
 *    log probabilities keep the partial results of their chunks there (and
 *    cut less where it is small). Calls on one context
 *    are ordered by its stream, so they never overlap on it.
 */
#ifndef SHADY_HIP_H
#define SHADY_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct st_context st_context;

typedef enum {
    ST_OK = 0,
    ST_ERR_INVALID = 1,     /* null pointer / bad enum */
    ST_ERR_SHAPE = 2,       /* K, N, M or group size not supported */
    ST_ERR_ALIGN = 3,       /* pointer not 16-byte aligned */
    ST_ERR_UNSUPPORTED = 4, /* valid request this build does not implement */
    ST_ERR_HIP = 5,         /* HIP runtime error */
    ST_ERR_WORKSPACE = 6,   /* context workspace too small */
    ST_ERR_OOM = 7
} st_status;

typedef enum { ST_F32 = 0, ST_F16 = 1, ST_BF16 = 2, ST_I8 = 3 } st_dtype;

/* flags */
#define ST_FLAG_ZEROS_PLUS_ONE 0x1u /* qzeros hold z - 1 (AutoGPTQ v1 files) */
#define ST_FLAG_TILED 0x2u          /* weights in the tiled layout of st_gptq_i4_repack / st_int8_repack */
#define ST_FLAG_NORM_PLUS_ONE 0x4u  /* st_qk_norm_rope_store, st_add_rmsnorm: norm weights hold w - 1 (the reference's rmsnorm multiplies by 1 + w) */
#define ST_FLAG_ROPE_PAIRS 0x8u     /* st_qk_norm_rope_store: rotates dims (2j, 2j + 1), not (j, j + rot / 2) */

/* ------------------------------------------------------------ runtime */

/* Message of the last failed call on this thread ("" if none). */
const char *st_last_error(void);

/* The kernels that this thread's calls have launched since its last call of
 * st_launches (the newest 64 at most), oldest first: writes up to `max` names
 * (static strings) and returns how many. Several kernels stand behind one
 * entry point; this says which a call took. */
int st_launches(const char **names, int max);

/* Version string of the built library (kernels + ABI revision). */
const char *st_version(void);

/* Replaces GpuContext::new (src/gpu.rs:17-78): binds `device`, creates one
 * stream and the split-K workspace (default 64 MiB). */
int st_context_create(int device, st_context **out);

/* Replaces GpuContext::from_device_queue (src/gpu.rs:24-33): run on a caller
 * stream (hipStream_t passed as void*; NULL = the device's null stream)
 * instead of the context's own. Does not synchronise (ordering between the
 * old and the new stream is the caller's); legal during stream capture. */
int st_context_set_stream(st_context *ctx, void *hip_stream);
void *st_context_stream(st_context *ctx);

/* Grow the split-K workspace to at least `bytes` (call at init, never on the
 * hot path; kernels never allocate). */
int st_context_reserve_workspace(st_context *ctx, size_t bytes);

int st_context_destroy(st_context *ctx);

/* Kernel-path overrides of one context. No counterpart in the reference (its
 * WGSL path has one shader per op); for tests that force each path and for
 * tuning. Every setting starts at -1 (automatic: the library's shape rules
 * choose); a call made after a change uses the new value. Nothing is read
 * from the environment. */
typedef enum {
    ST_TUNE_DECODE_KERNEL = 0, /* 1-4 tokens on tiled weights: 0 register-ring, 1 streaming */
    ST_TUNE_STAGE_MODE,        /* register-ring, one token block: 1 staging waves, 2 per-wave staging */
    ST_TUNE_STAGE_ROUNDS,      /* register-ring staging waves: 64-item rounds each (1..4) */
    ST_TUNE_WAVES,             /* register-ring, one tile per workgroup: waves (4..16) */
    ST_TUNE_NO_COOP,           /* 1: register-ring per-wave fallback only */
    ST_TUNE_ONE_TILE,          /* 1: one 16-column tile per workgroup */
    ST_TUNE_NO_CHUNK,          /* 1: no K-chunked cooperative staging (several tokens) */
    ST_TUNE_NO_KSPLIT,         /* 1: no split-K of several-token decode on few tiles */
    ST_TUNE_SPLIT_TILES_CU,    /* several-token decode: split K up to this many tiles per CU */
    ST_TUNE_TOKEN_BLOCK,       /* decode: tokens per launch (1..16) */
    ST_TUNE_I4MM_MIN_M,        /* GPTQ decode: fewest tokens for the f16-MFMA kernels (default 5; on at most one tile per CU 9 with K below 2048, 3 under act-order with M K of 12288 or silu(a) b) */
    ST_TUNE_I4MM_MIN_TILES,    /* GPTQ decode: fewest 16-column tiles for the f16-MFMA kernels */
    ST_TUNE_I8MM_MIN_M,        /* INT8 decode: fewest tokens for the f16-MFMA kernel */
    ST_TUNE_GEMM_CB,           /* prefill GEMM: workgroup tile of 128 (1), 256 (2) or 512 (3) columns; set, the skinny kernel takes no GEMM call */
    ST_TUNE_GEMM_NO_SPLIT,     /* 1: prefill GEMM without split-K; set (0 or 1), the skinny kernel takes no GEMM call */
    ST_TUNE_STREAM_WAVES,      /* streaming decode kernel: waves per workgroup (8 or 16) */
    ST_TUNE_STREAM_TILES_WG,   /* streaming decode kernel: 16-column tiles per workgroup (0: a workgroup per CU) */
    ST_TUNE_STREAM_SYNC,       /* streaming decode kernel: ring blocks between workgroup barriers (0: none) */
    ST_TUNE_SPLIT_REDUCE_KERNEL, /* several-token split-K decode: 1 reduce kernel, 0 fused (default: fused up to 8 tokens) */
    ST_TUNE_I4MM_WAVES,        /* f16-MFMA GPTQ decode: 16 forces 16-wave workgroups (default: 12 when the tiles use at most 12) */
    ST_TUNE_I4MM_PAIR,         /* f16-MFMA gate/up: 0 gives each wave one source (default 1: both sources of a tile per wave) */
    ST_TUNE_I4MM_PREPASS,      /* f16-MFMA GPTQ decode, f32 x: 1 splits x in a pre-pass launch (default: in the kernel, unless act-order) */
    ST_TUNE_I4MM_SPLIT_TILES,  /* f16-MFMA GPTQ decode on at most one 16-column tile per CU: 0 keeps the limb kernels */
    ST_TUNE_FP8_TILE,          /* st_fp8_gemm: tokens x columns of a workgroup: 0 the few tokens' kernel (up to 64), 1 64 x 64, 2 64 x 128, 3 128 x 64, 4 128 x 128, 5 128 x 256, 6 256 x 128, 7 256 x 256 (6: not for f16 y of more than 64 tokens unless FP8_EXACT; 5, 7: only for it; 7: K of more than 128; one that is not built for the call, or too small for a launch, gives way to the automatic choice) */
    ST_TUNE_FP8_SPLITS,        /* st_fp8_gemm with a tile set: slices of K (1, 2, 4 or 8) */
    ST_TUNE_FP8_EXACT,         /* st_fp8_gemm, f16 y of more than 64 tokens: 1 keeps products exact there too (default 0: see st_fp8_gemm) */
    ST_TUNE_COUNT
} st_tune;
int st_context_set_tune(st_context *ctx, int knob, int value);
int st_context_get_tune(st_context *ctx, int knob, int *value);

/* Kernel timing, in place of the reference's wgpu timestamp-less submits
 * (src/gpu.rs:188-242 has no timing): arms two hipEvent_t (created by the
 * caller, passed as void*) on the context. The next kernel launch records
 * `start` at its kernel's start; every launch records `stop` at its kernel's
 * end (hipExtLaunchKernel's dispatch timestamps, the duration a profiler
 * reports, without the gap between launches), so over one entry-point call
 * the pair spans its kernels. Stays armed until called again; NULL, NULL
 * disarms. Not for stream capture. */
int st_context_set_timing_events(st_context *ctx, void *start, void *stop);

/* Pins the context's workspace (delta +1) or releases a pin (-1): a captured
 * HIP graph holds kernels that point into the workspace, so while any pin is
 * held st_context_reserve_workspace refuses to reallocate it. DecoderStack's
 * capture (the host mirror of src/model.rs:669-969) takes one for the life
 * of its graph; no reference counterpart (wgpu has no graphs). */
int st_context_pin_workspace(st_context *ctx, int delta);

/* Replaces GpuContext::create_buffer / create_storage_buffer (src/gpu.rs:80-103): device
 * allocation, size rounded up to 4 bytes, 256-byte aligned. */
int st_alloc(st_context *ctx, size_t bytes, void **out);
int st_free(st_context *ctx, void *ptr);

/* Replaces GpuContext::upload_buffer (src/gpu.rs:105-117): host -> device,
 * returns when the data is on the device. */
int st_upload(st_context *ctx, void *dst, const void *host_src, size_t bytes);

/* Replaces GpuContext::write_buffer (src/gpu.rs:278-282): stream-ordered
 * host -> device write at a byte offset. */
int st_write(st_context *ctx, void *dst, size_t offset, const void *host_src, size_t bytes);

/* Replaces GpuContext::read_buffer (src/gpu.rs:252-276): waits for all queued
 * work, then copies device -> host. */
int st_read(st_context *ctx, const void *src, void *host_dst, size_t bytes);

/* Replaces GpuContext::copy_buffer (src/gpu.rs:245-250), stream-ordered. */
int st_copy(st_context *ctx, void *dst, const void *src, size_t bytes);

/* Replaces GpuContext::flush (src/gpu.rs:237-242): wait for the stream. */
int st_flush(st_context *ctx);

/* -------------------------------------------------------- GPTQ int4 */

/* y = x . dequant(W), W[k, n] = (q[k, n] - z[g(k), n]) * scales[g(k), n].
 * Replaces Model::gptq_matvec (src/model.rs:357-381) dispatching
 * gptq_matvec(_4t).wgsl (src/shaders/gptq_matvec_4t.wgsl:20-86).
 *   x        [M, K] in x_dtype (ST_F32 or ST_F16)
 *   qzeros   NULL = symmetric z = 8, the reference's only mode
 *   perm     NULL, or int32[K] from st_gptq_i4_act_order (then qweight is the
 *            act-order-sorted copy): x is read as x[:, perm[k]]
 *   y        f32 [M, N]
 *   flags    ST_FLAG_ZEROS_PLUS_ONE, ST_FLAG_TILED (qweight from st_gptq_i4_repack)
 * Requires K % group_size == 0, group_size in {64, 128, 256}, N % 8 == 0,
 * 1 <= M <= 32, 16-byte aligned qweight and x. Accumulation: exact integer
 * products of the nibbles with a 3 x 8-bit split of x scaled by a power of
 * two per group, f32 across groups (rel-L2 vs f64 ~3e-7). From 5 tokens on
 * tiled weights (with at most one 16-column tile per CU from 9 with K below
 * 2048, and from 3 under perm with M K of 12288 at least): f16 MFMA on exact
 * (q - z) and x (f16 x as is; f32 x scaled by a power of two per token and at
 * most 512 k and split into two f16 parts, together 22 bits, whose products are
 * summed apart within a group), f32 sums; rel-L2 vs f64 of f32 x 0.8e-7 to
 * 1.7e-7, the weights read once for up to 32 tokens. K may be split across
 * workgroups, with partial sums in the context workspace, where x gathered under
 * perm comes first. The same rule applies to st_gptq_i4_gate_up_silu, and but for
 * the last condition to st_gptq_i4_silu_matvec (from 3 tokens under perm). */
int st_gptq_i4_matvec(st_context *ctx, const void *x, int x_dtype,
                      const uint32_t *qweight, const uint16_t *scales,
                      const uint32_t *qzeros, const int32_t *perm, float *y,
                      int M, int K, int N, int group_size, uint32_t flags);

/* No counterpart in the reference: for callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc). st_gptq_i4_matvec with everything its kernels keep
 * beyond the inputs and outputs (x gathered under act-order, as it is or split
 * into f16 rows, and split-K partial sums) in a fixed array of
 * ST_NOALLOC_SCRATCH_BYTES that the library holds on every GPU it runs on,
 * from the context's creation until the process ends, instead of the
 * context workspace. Allocates nothing. A call whose scratch would exceed
 * the array fails with ST_ERR_WORKSPACE and launches nothing. The check is
 * conservative: for f32 x (and for f16 x under act-order) it counts two f16
 * rows per token and a factor per 128 k, 4 M K + M K / 32 bytes (f16 x with
 * perm: 2 M K), with M capped at 32, whichever kernel the call then takes (f32 x
 * without perm needs none of it); split-K partials are not counted (they shrink or go unsplit
 * to fit the array). Every call on
 * one GPU shares that GPU's array (nothing in it needs to start at zero;
 * each call overwrites what it reads): calls that overlap on one GPU (other
 * streams or contexts) race. */
#define ST_NOALLOC_SCRATCH_BYTES (8u << 20)
int st_gptq_i4_matvec_noalloc(st_context *ctx, const void *x, int x_dtype, const uint32_t *qweight,
                              const uint16_t *scales, const uint32_t *qzeros, const int32_t *perm, float *y, int M,
                              int K, int N, int group_size, uint32_t flags);

/* y = (silu(a) * b) . dequant(W), silu(v) = v / (1 + exp(-v)).
 * Replaces Model::fused_silu_gptq_down (src/model.rs:383-408) dispatching
 * fused_silu_gptq(_4t).wgsl (src/shaders/fused_silu_gptq_4t.wgsl:26-81).
 * a, b: f32 [M, K]. Other arguments as st_gptq_i4_matvec. */
int st_gptq_i4_silu_matvec(st_context *ctx, const float *a, const float *b,
                           const uint32_t *qweight, const uint16_t *scales,
                           const uint32_t *qzeros, const int32_t *perm, float *y,
                           int M, int K, int N, int group_size, uint32_t flags);

/* y = silu(x . dequant(Wg)) * (x . dequant(Wu)), both [K, N].
 * Replaces fused_gate_up_silu(_4t).wgsl (src/shaders/fused_gate_up_silu_4t.wgsl:28-91,
 * declared at src/model.rs:8; the reference's forward runs gate and up as two
 * gptq_matvec calls at src/model.rs:803-808). Both weights share perm.
 * 1 <= M <= 32; other arguments as st_gptq_i4_matvec. */
int st_gptq_i4_gate_up_silu(st_context *ctx, const void *x, int x_dtype,
                            const uint32_t *qweight_gate, const uint16_t *scales_gate,
                            const uint32_t *qzeros_gate, const uint32_t *qweight_up,
                            const uint16_t *scales_up, const uint32_t *qzeros_up,
                            const int32_t *perm, float *y, int M, int K, int N,
                            int group_size, uint32_t flags);

/* Materialise dequant(W) as out[K, N] in out_dtype (ST_F32 exact; ST_BF16
 * round-to-nearest-even, which is src/weights.rs:257-313
 * dequant_gptq_to_bf16). g_idx NULL = k / group_size (no act-order);
 * otherwise the original int32 g_idx[K] of the checkpoint. */
int st_gptq_i4_dequant(st_context *ctx, const uint32_t *qweight, const uint16_t *scales,
                       const uint32_t *qzeros, const int32_t *g_idx, void *out, int out_dtype,
                       int K, int N, int group_size, uint32_t flags);

/* Upload-time repack into the decode kernels' tiled layout (no reference
 * counterpart; an optional step of the weight upload, src/weights.rs:398):
 * per 16-column tile and group, the 64 lanes' words are contiguous, so the
 * kernel reads 1 KiB contiguous per group with 128-bit loads. Dequantized
 * values are unchanged (a permutation of whole words). qweight_tiled must hold
 * st_gptq_i4_tiled_words(K, N, group_size) words; pass ST_FLAG_TILED to the
 * matvec entry points with it. */
size_t st_gptq_i4_tiled_words(int K, int N, int group_size);
int st_gptq_i4_repack(st_context *ctx, const uint32_t *qweight, uint32_t *qweight_tiled, int K, int N,
                      int group_size);

/* Upload-time act-order preparation (the reference drops .g_idx,
 * src/weights.rs:372-374). Sorts K by group: perm_out[j] = the original row
 * placed at position j (stable, ascending g_idx), and qweight_out = qweight
 * with its rows permuted the same way (re-packed nibbles; dequantized values
 * unchanged). Each group must hold exactly group_size rows. Scales and
 * qzeros are unchanged. g_idx is a device pointer; blocks until done. */
int st_gptq_i4_act_order(st_context *ctx, const uint32_t *qweight, const int32_t *g_idx,
                         uint32_t *qweight_out, int32_t *perm_out, int K, int N,
                         int group_size);

/* bf16 matvec: y[M, N] = x[M, K] . W^T, W bf16 row-major [N, K] (two bf16 per
 * u32, low half first), x f32 or f16 (x_dtype), y f32, 1 <= M <= 8,
 * K % 8 == 0, K <= 10240 (M <= 4) or 5120 (M <= 8). Replaces src/shaders/bf16_matvec.wgsl:21-72 (the
 * lm_head / tied-embedding projection, dispatched at src/model.rs:455-468
 * and :824-831); f32 accumulation, results within 1e-4 rel-L2 of f64. */
int st_bf16_matvec(st_context *ctx, const void *x, int x_dtype, const uint16_t *w, float *y, int M, int K,
                   int N);

/* Prefill GEMM: C[M, N] = A[M, K] . dequant(W), A f16, C in c_dtype (ST_F32
 * or ST_F16). No reference counterpart (the reference prefills token by
 * token, src/inference.rs:93-95). MFMA f16 on weights (q - z) s rounded once to
 * f16, f32 accumulation (rel-L2 vs f64 ~2e-4). perm as st_gptq_i4_matvec. */
int st_gptq_i4_gemm(st_context *ctx, const uint16_t *a, const uint32_t *qweight,
                    const uint16_t *scales, const uint32_t *qzeros, const int32_t *perm,
                    void *c, int c_dtype, int M, int K, int N, int group_size,
                    uint32_t flags);

/* Gate and up projections of one MLP for M tokens in one call:
 * c_gate = a . dequant(W_gate) and c_up = a . dequant(W_up), both [M, N],
 * from one pre-processed A and one launch whose grid holds the tiles of both
 * weights (short prompts may take a launch for each). The M-token form of the gate/up
 * half of the reference's MLP (src/model.rs:803-811, the separate gate and
 * up matvecs it runs one token at a time); st_gptq_i4_silu_gemm then takes
 * c_gate and c_up for the down projection. Both weights share K, N,
 * group_size, flags and perm; either may have qzeros or not. Each output is
 * bit for bit what st_gptq_i4_gemm gives for that weight. */
int st_gptq_i4_gate_up_gemm(st_context *ctx, const uint16_t *a, const uint32_t *gate_qweight,
                            const uint16_t *gate_scales, const uint32_t *gate_qzeros,
                            const uint32_t *up_qweight, const uint16_t *up_scales,
                            const uint32_t *up_qzeros, const int32_t *perm, void *c_gate, void *c_up,
                            int c_dtype, int M, int K, int N, int group_size, uint32_t flags);

/* Prefill GEMM on silu(gate) * up: C[M, N] = (silu(gate) * up)[M, K] .
 * dequant(W), gate and up f16 [M, K], silu(v) = v / (1 + exp(-v)) in f32,
 * the product rounded once to f16. The M-token form of
 * Model::fused_silu_gptq_down (src/model.rs:383-408, fused_silu_gptq(_4t).wgsl),
 * which the reference runs one token at a time (src/model.rs:803-811). Other
 * arguments as st_gptq_i4_gemm. */
int st_gptq_i4_silu_gemm(st_context *ctx, const uint16_t *gate, const uint16_t *up,
                         const uint32_t *qweight, const uint16_t *scales, const uint32_t *qzeros,
                         const int32_t *perm, void *c, int c_dtype, int M, int K, int N,
                         int group_size, uint32_t flags);

/* ------------------------------------------------------------- INT8 */

/* y[M, N] = x[M, K] . (w[N, K]^T * scale[N]), int8 symmetric per output
 * channel. No reference counterpart. x in x_dtype (ST_F16 or ST_F32),
 * 1 <= M <= 32, K % 128 == 0, N % 4 == 0. flags: ST_FLAG_TILED when w is in
 * the layout of st_int8_repack (else row-major int8[N, K]). Two or more
 * tokens with f16 x on tiled weights run on f16 MFMA (every product exact,
 * f32 sums; the weights are read once for all tokens); otherwise exact
 * integer products with a split of x as for st_gptq_i4_matvec. */
int st_int8_matvec(st_context *ctx, const void *x, int x_dtype, const int8_t *w,
                   const float *scale, float *y, int M, int K, int N, uint32_t flags);

/* INT8 prefill GEMM (W8A16): C[M, N] = A[M, K] . (w[N, K]^T * scale[N]),
 * A f16 row-major, C f32 or f16 (c_dtype). No reference counterpart: the
 * north star's INT8 GEMM for prefill, the M-token form of st_int8_matvec
 * for M above its 32 (the reference prefills token by token through the
 * matvec, src/inference.rs:93-95). Every product is exact in f32 (int8 and
 * f16 are exact in f16), the sums are f32, the channel scale is applied once
 * per output. K % 128 == 0, N % 4 == 0; a and w 16-byte aligned; flags:
 * ST_FLAG_TILED for st_int8_repack's layout. Small grids split K across
 * workgroups (f32 partials in the context workspace, added in a fixed order). */
int st_int8_gemm(st_context *ctx, const uint16_t *a, const int8_t *w, const float *scale, void *c,
                 int c_dtype, int M, int K, int N, uint32_t flags);

/* Upload-time INT8 repack (no reference counterpart): row-major w[N, K] ->
 * tiles of 16 rows in which, per 128-k group, each of a wave's 64 lanes
 * holds 32 contiguous bytes, so the kernel reads 2 KiB contiguous per group.
 * Values are unchanged (a permutation of 16-byte pieces). w_tiled must hold
 * st_int8_tiled_bytes(K, N) bytes; pass ST_FLAG_TILED to st_int8_matvec. */
size_t st_int8_tiled_bytes(int K, int N);
int st_int8_repack(st_context *ctx, const int8_t *w, int8_t *w_tiled, int K, int N);

/* ------------------------------------------ 8-bit floating point */

/* e4m3 (OCP: finite, at most 448, NaN 0x7F) in blocks with float32 scales, the
 * format of block-scaled checkpoints; no reference counterpart, as INT8.
 *   rows    x8 [M][K] with x_scale [ceil(K / 128)][scale_stride]: token m's dims
 *           of block b are x8 times x_scale[b][m] (a block's scales side by side
 *           by token, scale_stride >= M of them)
 *   weight  w [N][K] row-major with w_scale [ceil(N / 128)][ceil(K / 128)]: one
 *           for each 128 x 128
 * K is a multiple of 16; it and N may end inside a block. Quantising makes a
 * block's scale max|x| times the f32 nearest to 1 / 448, at least 2^-126, and
 * rounds the f32 quotient x / scale to nearest, even. A block with a NaN has a
 * NaN scale; one with an infinity an infinite scale, its infinities 448 of their
 * sign and the rest 0. */

/* r = residual + x and its RMS norm y = r / sqrt(mean(r^2) + eps) * weight
 * (1 + weight: ST_FLAG_NORM_PLUS_ONE), to e4m3 rows (y8, y_scale), to y, or to
 * both: replaces rmsnorm.wgsl and add_rmsnorm.wgsl (src/model.rs:685-691,
 * 799-802, 820-823).
 *   residual, residual_out  M rows of D of res_dtype (ST_F32 or ST_F16); the norm
 *             is of the sum before it is rounded to it. They may be one buffer.
 *   x         x_dtype (ST_F32 or ST_F16), or NULL, with residual_out NULL: the
 *             norm of the residual alone
 *   weight    f32 [D]
 *   y         y_dtype (ST_F32 or ST_F16) or NULL; it may be x's buffer, or the
 *             residual's where the sum does not go there
 *   *_stride  elements from one row to the next
 * residual_out may also be x's buffer. Buffers that are one have one type and
 * stride; otherwise outputs share no element with another argument. f32
 * arithmetic. M less than 2^22; D a multiple of 16, at most 32768. Pointers and
 * strides in whole 16 bytes (y_scale: 4). */
int st_add_rmsnorm(st_context *ctx, const void *residual, int res_dtype, int64_t res_stride, const void *x,
                   int x_dtype, int64_t x_stride, void *residual_out, int64_t out_stride, const float *weight,
                   float eps, void *y, int y_dtype, int64_t y_stride, uint8_t *y8, float *y_scale,
                   int64_t scale_stride, int M, int D, uint32_t flags);

/* Rows of e4m3 of M rows a [K], or of silu(a) * b where b is given (the input
 * of a down projection), silu(v) = v / (1 + exp(-v)); dtype ST_F32 or ST_F16,
 * *_stride elements from one row to the next. Less than 2^24 units of a row's
 * 2048 dims. Pointers and strides in whole 16 bytes (y_scale: 4). Outputs share
 * no element with inputs. */
int st_fp8_quant(st_context *ctx, const void *a, const void *b, int dtype, int64_t a_stride, int64_t b_stride,
                 uint8_t *y8, float *y_scale, int64_t scale_stride, int M, int K);

/* y[m][n] = sum_b x_scale[b][m] w_scale[n / 128][b] sum_{k in b} x8[m][k] w[n][k],
 * y [M][N] of y_dtype (ST_F32 or ST_F16), any M and N (at most 2^28, and fewer
 * than 2^22 blocks of 128 x 128 of y), in memory of its own. x8, w and y 16-byte
 * aligned (scales: 4).
 * Sums are f32, in a fixed order for each size. With f32 y, and f16 y of at most
 * 64 tokens, products are exact. f16 y of more tokens comes from the 8-bit matrix
 * instruction, which keeps a product to 2^-13 of the power of two of the largest
 * of its eight neighbouring k, so that sums which cancel lose what lies below,
 * and a token's row is not quite the same in a batch of 64 and of 65. By rel-L2
 * that is 1.4e-5 on normal activations, 2.8e-5 with some channels at 16 times the
 * rest, 6.8e-5 with one at 1000 times (measured, weights normal), beside f16's own
 * 2.1e-4. ST_TUNE_FP8_EXACT 1 keeps products exact there too, at up to twice the
 * time. */
int st_fp8_gemm(st_context *ctx, const uint8_t *x8, const float *x_scale, int64_t scale_stride, const uint8_t *w,
                const float *w_scale, void *y, int y_dtype, int M, int K, int N);

/* ----------------------------------------- key-value cache and attention */

/* A paged key-value cache of one layer (device pointers, owned by the caller).
 * Slot s is place s % page_size of page s / page_size; tokens lie in tiles of
 * 16 places, so that the attention's matrix instructions take 16-byte (f16)
 * or 8-byte (int8) pieces as they are, and whole tiles are contiguous:
 *   k  [num_pages][n_kv_heads][page_size / 16][head_dim / 8][16][8]
 *      eight dims of a token side by side
 *   v  [num_pages][n_kv_heads][page_size / 16][2][head_dim][8]
 *      eight places of a dim side by side: half h holds places 4 h .. 4 h + 3
 *      and 8 + 4 h .. 8 + 4 h + 3 of the tile, in this order
 *   k_scale, v_scale  f32 [num_pages][n_kv_heads][page_size], ST_I8 only: a
 *      token's head is its int8 values times its scale
 * dtype ST_F16 or ST_I8; page_size 16, 32, 64, 128 or 256; head_dim 64, 128
 * or 256; every pointer 16-byte aligned. The reference keeps one contiguous
 * f32 cache per sequence (fused_split_qknorm_kvstore.wgsl, src/model.rs:971-1029). */
typedef struct {
    void *k, *v;
    float *k_scale, *v_scale;
    int dtype;
    int num_pages, page_size, n_kv_heads, head_dim;
} st_kv_cache;

/* RMS norms of the queries and keys of each head, their rotation, and the
 * write of keys and values into the cache, in one launch: replaces
 * fused_split_qknorm_kvstore.wgsl:1-230 (dispatched between q|k|v and the
 * attention, src/model.rs:715-726).
 *   q, k, v   T tokens of x_dtype (ST_F32 or ST_F16); *_stride elements from
 *             one token to the next (the three may be parts of one q|k|v
 *             row); heads of k and v side by side, those of q q_head_stride
 *             elements apart (2 head_dim where each head's query is followed
 *             by its gate, as the reference's gated q). q and q_out NULL:
 *             keys and values only.
 *   q_weight, k_weight  f32 [head_dim] or NULL (no norm):
 *             y = x / sqrt(mean(x^2) + eps) * w (1 + w: ST_FLAG_NORM_PLUS_ONE)
 *   cos, sin  f32 [n_pos][rot / 2] or both NULL (no rotation): the first rot
 *             dims (a multiple of 16) of q and k at the token's position,
 *             dims (j, j + rot / 2), or (2j, 2j + 1) with ST_FLAG_ROPE_PAIRS:
 *             (a, b) -> (a c - b s, b c + a s). Positions of several axes:
 *             tables of one row per token.
 *   positions int32 [T] (NULL without rotation); a token whose position is
 *             not in [0, n_pos) gets NaN queries and is not stored
 *   slots     int32 [T]; a slot outside the cache (a negative one: padding)
 *             is not written
 *   q_out     [T][n_heads][head_dim] of q_dtype (ST_F32 or ST_F16)
 * f32 arithmetic, one rounding to what is stored. An int8 cache gets, for
 * each token and head, scale = max|y| / 127 and round(y / scale). Two tokens
 * of one call with one slot: which of them stays is undefined. Pointers and
 * strides in whole 16 bytes. */
int st_qk_norm_rope_store(st_context *ctx, const st_kv_cache *cache, const void *q, const void *k, const void *v,
                          int x_dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride, int q_head_stride,
                          const float *q_weight, const float *k_weight, float eps, const float *cos,
                          const float *sin, int rot, int n_pos, const int32_t *positions, const int32_t *slots,
                          void *q_out, int q_dtype, int T, int n_heads, uint32_t flags);

/* Cached tokens read back, dequantised: k_out and v_out [T][n_kv_heads]
 * [head_dim] of out_dtype (ST_F32 or ST_F16, int8 values times their scale
 * rounded once). A slot outside the cache reads as zeros. For a prefix taken
 * out of a cache or moved to another (the reference copies whole cache
 * buffers, src/model.rs:1021-1029). */
int st_kv_read(st_context *ctx, const st_kv_cache *cache, const int32_t *slots, void *k_out, void *v_out,
               int out_dtype, int T);

/* Attention of new rows over the cache: rows of sequence b are q_start[b] ..
 * q_start[b + 1] (NULL: one row for each sequence, T == B), the newest of its
 * kv_len[b] tokens, all of them in the cache already (so row i of n has
 * position kv_len - n + i). Replaces gqa_attention_head.wgsl:1-124,
 * gqa_reduce.wgsl:1-65 and sigmoid_mul.wgsl (src/model.rs:540-592).
 *   s_j = scale q . k_j, capped cap tanh(s_j / cap) where cap > 0 (of any
 *   size; past 2^100 it is none), plus
 *   slopes[head] (j - position) where slopes (f32 [n_heads]) is given;
 *   key j is visible if j <= position and, where window > 0, j > position -
 *   window; out = sum_j softmax(s)_j v_j over the visible keys (a row that
 *   sees none: zeros), times sigmoid(gate) where gate is given
 *   q, out    [T][n_heads][head_dim] of q_dtype, out_dtype (ST_F32 or ST_F16);
 *             n_heads a multiple of the cache's heads, head h reads key head
 *             h / (n_heads / n_kv_heads)
 *   table     int32 [B][table_stride]: page of tokens page_size i ..; entries
 *             past a sequence's last token are not read; tokens of a page
 *             outside the cache are never read and count as not visible
 *   kv_len    int32 [B], q_start int32 [B + 1]: device arrays; a captured
 *             graph may be replayed after they, table and the cache changed
 *             (out-of-range values are clamped to the table and to T; if
 *             q_start decreases anywhere, out may be left as it is)
 *   gate      gate_dtype, gate_stride elements between tokens,
 *             gate_head_stride between heads (the gates of the reference's
 *             gated q lie beside its queries)
 * Rows of q and out outside every sequence are left alone. What a row does
 * not see may be anything; a NaN query, or a NaN key or scale that a row sees,
 * makes the row and head NaN, a value that is not finite its dim infinite or
 * NaN. f32 scores,
 * softmax and sums. With f32 q or out the products keep 22 bits of q and of
 * the softmax weights; with f16 both, the weights are rounded to f16. Chunks
 * of a long cache meet in the context workspace, in a fixed order. */
int st_paged_attention(st_context *ctx, const st_kv_cache *cache, const void *q, int q_dtype, const int32_t *table,
                       int table_stride, const int32_t *kv_len, const int32_t *q_start, float scale, float cap,
                       int window, const float *slopes, const void *gate, int gate_dtype, int64_t gate_stride,
                       int gate_head_stride, void *out, int out_dtype, int T, int B, int n_heads);

/* ------------------------------------------------------------ logits */

/* Log probabilities of given tokens, their rank, the entropy and the top
 * alternatives of M rows of logits, in one pass. The reference reads its
 * logits back and samples on the CPU (src/model.rs:836-968).
 *   logits    [M] rows of V, `stride` elements apart, dtype ST_F32 or ST_F16
 *   tokens    int32 [M] or NULL (then neither logprob nor rank)
 *   logprob   f32 [M] or NULL: log softmax(logits)[token], natural logarithm;
 *             NaN for a token outside the vocabulary
 *   entropy   f32 [M] or NULL: -sum p log p
 *   rank      int32 [M] or NULL: how many tokens come before the given one by
 *             (value, lower index first); -1 for one outside the vocabulary
 *   top_ids   int32 [M][top], top_logprobs f32 [M][top] or NULL: the `top`
 *             first tokens in that order; top 0..32, at most V
 * -inf logits are tokens of probability 0. A row with a NaN, a +inf or
 * nothing but -inf has no distribution: its log probabilities and entropy
 * are NaN (a NaN orders as +inf). V <= 2^20. f32 arithmetic; a likely
 * token's log probability keeps f32's relative precision down to 0. */
int st_token_logprobs(st_context *ctx, const void *logits, int dtype, int64_t stride, const int32_t *tokens,
                      float *logprob, float *entropy, int32_t *rank, int32_t *top_ids, float *top_logprobs,
                      int M, int V, int top);

#ifdef __cplusplus
}
#endif

#endif /* SHADY_HIP_H */
