/*
 * wush_int4.h -- C ABI of the MI355X (gfx950) WUSH INT4 W4A4 library
 * (libwush_int4.so).
 *
 * Every entry point takes plain device pointers, element counts and a HIP
 * stream; it validates its arguments, enqueues its kernels on `stream` and
 * returns a hipError_t value (hipSuccess == 0).  Nothing here allocates:
 * outputs and the optional split-K workspace come from the caller, so every
 * call is safe under HIP graph capture.  Launches are asynchronous.
 *
 * Data formats (identical to the reference's my_int4._C tensors):
 *   codes  uint8, two signed INT4 codes per byte, element 2k in the low
 *          nibble, element 2k+1 in the high nibble (docs/SPEC.md:10-11;
 *          my_int4/rtn_int4.py:53-55); codes are in [-7, 7].
 *   scales bf16 bit patterns (uint16), one per 32-element group along K.
 *   T      bf16 (K/32, 32, 32): T[c][j][i], x'_j = sum_i x_i * T[c][j][i].
 *   y      fp16 bit patterns (uint16), row-major (M, N).
 * Bad arguments return hipErrorInvalidValue and launch nothing.
 *
 * Citations are to files of the reference repository (rib12316/WUSH_int4_kernel).
 */
#ifndef WUSH_INT4_H
#define WUSH_INT4_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WUSH_INT4_ABI_VERSION 1

/* Element type of the activations handed to wush_quant_int4. */
enum wush_dtype {
    WUSH_DTYPE_BF16 = 0,
    WUSH_DTYPE_F16 = 1,
    WUSH_DTYPE_F32 = 2
};

/* ABI version of the loaded library (WUSH_INT4_ABI_VERSION). */
int wush_abi_version(void);

/* One-time set-up of every visible device: the prefill kernel's dynamic LDS
 * limit (a function attribute) and the decode GEMV's occupancy table.  Call
 * it once before capturing any entry point in a HIP graph (the torch module
 * calls it at import).  An entry point called on a device that was not set up
 * runs the set-up there first, which sets a function attribute and so must not
 * happen during a capture.  Thread-safe; returns the first error, or
 * hipSuccess.  Replaces the reference's lazy static-flag attribute set-up
 * (csrc/gemm_cutlass_int4.cu:62-67, :111-119). */
int wush_init(void);

/* Text for a status returned by any entry point. */
const char *wush_error_string(int status);

/* Group-wise sigma-clip INT4 quantization, bit-exact with the reference.
 * x: n_groups*32 contiguous values of type `dtype`; q: n_groups*16 bytes;
 * s: n_groups bf16 scales.
 * Replaces quant_int4() in csrc/quant_int4.cu:109-134 (bf16 input, bound at
 * csrc/bindings.cpp:38) and, for fp16/fp32 input, the torch reference
 * my_int4/rtn_int4.py:33-55. */
int wush_quant_int4(const void *x, int dtype, uint8_t *q, uint16_t *s,
                    int64_t n_groups, hipStream_t stream);

/* WUSH block-diagonal transform fused with the quantization, bit-exact with
 * the reference's sequential form: x'_j = sum_i x_i*T[c][j][i] (fp32, i
 * ascending, every product and sum rounded), then wush_quant_int4's math on
 * x'.  x: rows*K bf16; t: (K/32)*1024 bf16; q: rows*K/2; s: rows*K/32.
 * Replaces fused_transform_quant_int4 (csrc/fused_tq_int4.cu:87-118) and the
 * _smallm / _v3 / _wmma variants (csrc/fused_tq_smallm.cu:89-121,
 * csrc/fused_tq_v3.cu:109-140, csrc/fused_tq_wmma.cu:131-162), which share
 * its contract (csrc/bindings.cpp:60-68). */
int wush_fused_tq(const uint16_t *x, const uint16_t *t, uint8_t *q, uint16_t *s,
                  int64_t rows, int64_t K, hipStream_t stream);

/* The transform stage of wush_fused_tq's rows kernel alone, for one block:
 * x'[r][j] = sum_i x[r][i] * t[j][i] (fp32, i ascending, every sum rounded),
 * x rows*32 bf16, t 32*32 bf16, xp rows*32 fp32.  Runs the same code path as
 * wush_fused_tq for the same values (fp32 MFMA steps, fma loop or mul-then-add
 * loop, chosen per 64 rows).  No counterpart in the reference, whose transform
 * is internal to fused_transform_quant_int4 (csrc/fused_tq_int4.cu:38-84): it
 * lets tests compare x' itself, which the codes and scales see only near a
 * rounding boundary. */
int wush_fused_tq_transform32(const uint16_t *x, const uint16_t *t, float *xp, int64_t rows,
                              hipStream_t stream);

/* Decode GEMV for 1 <= M <= 8: y[m][n] = sum_g sx[m][g]*sw[n][g]*D[m][n][g]
 * with D the exact int32 dot of group g.  xq: M*K/2; xs: M*K/32; wq: N*K/2;
 * ws: N*K/32; y: M*N fp16.  Shapes that wush_gemv_int4_supported rejects
 * return hipErrorInvalidValue (wush_gemm_s4 takes any shape).
 * Replaces w4a4_gemv (csrc/gemv_int4.cu:191-223, M == 1) and w4a4_gemv_multi
 * (csrc/gemv_int4.cu:145-189, M <= 8). */
int wush_gemv_int4(const uint8_t *xq, const uint16_t *xs, const uint8_t *wq, const uint16_t *ws,
                   uint16_t *y, int64_t M, int64_t N, int64_t K, hipStream_t stream);

/* 1 if wush_gemv_int4 runs (M, N, K), else 0.  The rule depends on the
 * library's build (its tuning macros): 1 <= M <= 8, K % 32 == 0, and either
 * the activations fit the staged kernel's 64 KiB of LDS (M*K/2 + M*K/4
 * bytes) or the shape is one of the K-split kernel's (by default M = 7, 8,
 * K a multiple of 2048 in [8192, 32768], N > 32768), which keeps them in
 * registers.  A host that routes products between wush_gemv_int4 and
 * wush_gemm_s4 asks this instead of restating the rule.  The reference has
 * no counterpart: its w4a4_gemv_multi checks M <= 8 and fails at launch when
 * its shared memory does not fit (csrc/gemv_int4.cu:160-169). */
int wush_gemv_int4_supported(int64_t M, int64_t N, int64_t K);

/* Bytes of workspace wush_gemm_s4 uses for (M, N, K); 0 when it needs none:
 * fp32 split-K partials, and for prefill shapes with N >= 8192 the
 * activations converted once to fp16 operands (M*K*2 bytes, padded to 256
 * rows and 256 of K).  A caller may pass a larger buffer; a smaller one makes
 * wush_gemm_s4 choose a plan that needs no more than it is given: another K
 * split or another kernel, whose results agree within the tolerance below, not
 * bit for bit. */
size_t wush_gemm_s4_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* Bytes of workspace with which wush_gemm_s4 runs its fastest plan; at least
 * wush_gemm_s4_workspace_bytes, and more where that plan also converts the
 * activations to fp16 operands on weights of fewer than 8192 rows (M > 64,
 * K % 64 == 0, 16-byte aligned scales, from about 2^32 multiply-adds): with
 * fewer bytes than this, wush_gemm_s4 runs the plan of
 * wush_gemm_s4_workspace_bytes there.  The reference has no counterpart. */
size_t wush_gemm_s4_best_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* Group-scaled W4A4 GEMM, any M >= 1, K % 32 == 0: the product of
 * wush_gemv_int4, y (M, N) fp16.  On int8 MFMA with exact int32 group dots,
 * except for three ranges that run fp16 MFMA on code*scale operands (exact
 * after a power-of-two shift per row and column, for scales down to 2^-29 of
 * the row's or column's largest; with converted activations the outputs of
 * rows and columns beyond that are computed apart, in fp64, otherwise such
 * scales lose low bits) accumulated in fp32 over all of K: M > 64 with
 * K % 64 == 0, from about 2^32 multiply-adds (3e9, 4.8e9 for N < 2048; twice
 * that for K % 256 != 0; or 192 tiles of 128 x 256 outputs at N >= 8192 and
 * K % 256 == 0), when the workspace holds the converted activations (see the
 * two functions above); without that room M > 128 with K % 256 == 0, at least 64 tiles of 256x256 or N >= 2048, and
 * at least 128 workgroups counting the K slices of at least 32 groups each
 * that the workspace holds from M = 512; and 32 < M <= 64 with 49953 <= N <=
 * 57344 and K % 1024 == 0 (16-byte aligned codes and scales).
 * Both agree with the fp64 product to 2e-3 relative Frobenius (tested); a row
 * or column with a non-finite scale gives NaN there.
 * Replaces w4a4_gemm_s4 (csrc/gemm_s4.cu:320-379) and the superseded
 * w4a4_gemm / _v1 / _v2 (csrc/gemm_int4.cu:89-130, csrc/gemm_wmma.cu:128-172,
 * csrc/gemm_wmma2.cu:141-181) that compute the same product. */
int wush_gemm_s4(const uint8_t *xq, const uint16_t *xs, const uint8_t *wq, const uint16_t *ws,
                 uint16_t *y, int64_t M, int64_t N, int64_t K,
                 void *workspace, size_t workspace_bytes, hipStream_t stream);

/* wush_gemm_s4's plan for a workspace of wush_gemm_s4_best_workspace_bytes,
 * run over `rows` activation rows at a time (a multiple of 64, or at least M)
 * on a 16-byte aligned workspace of wush_gemm_s4_rows_workspace_bytes for the
 * same operands and rows.  Every value of `rows` gives the same bits, those of
 * that wush_gemm_s4 call: for callers short of memory that must not get other
 * results for it.  Slower, the shorter the runs.  The reference has no
 * counterpart. */
size_t wush_gemm_s4_rows_workspace_bytes(const uint8_t *xq, const uint16_t *xs, const uint8_t *wq,
                                         const uint16_t *ws, int64_t M, int64_t N, int64_t K, int64_t rows);
int wush_gemm_s4_rows(const uint8_t *xq, const uint16_t *xs, const uint8_t *wq, const uint16_t *ws,
                      uint16_t *y, int64_t M, int64_t N, int64_t K, int64_t rows,
                      void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Kernels of the GEMM entry points, as the two plan queries name them. */
enum wush_gemm_kernel {
    WUSH_GEMM_INT8_TILES = 0,       /* int8 MFMA tiles through LDS */
    WUSH_GEMM_INT8_STREAM = 1,      /* int8 MFMA, weights streamed (M <= 64) */
    WUSH_GEMM_FP16_TILES = 2,       /* fp16 MFMA tiles, operands converted per tile */
    WUSH_GEMM_FP16_CONVERTED = 3,   /* fp16 MFMA tiles on activations converted into the workspace */
    WUSH_GEMM_FP16_STREAM = 4,      /* fp16 MFMA, weights streamed (32 < M <= 64) */
    WUSH_GEMM_TENSOR_TILES = 5      /* per-tensor int8 MFMA tiles */
};

/* The plan wush_gemm_s4 runs for (M, N, K) with 16-byte aligned operands and
 * `workspace_bytes` of 16-byte aligned workspace: plan = {kernel, output rows
 * of a workgroup, columns, K slices}.  Host only, no device is touched; for
 * tests and tuning.  The reference has no counterpart. */
int wush_gemm_s4_plan(int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int32_t plan[4]);

/* The same for wush_gemm_s4_tensor_scale. */
int wush_gemm_s4_tensor_scale_plan(int64_t M, int64_t N, int64_t K, int32_t plan[4]);

/* Bytes of the static split-K scratch that wush_gemm_s4_noalloc uses: one
 * array per device, held from the library's load until the process ends. */
#define WUSH_GEMM_SCRATCH_BYTES (64u << 20)

/* Status of wush_gemm_s4_noalloc if no plan of the shape fits
 * WUSH_GEMM_SCRATCH_BYTES (wush_error_string explains it).  The planner
 * always has one (a single K slice needs no scratch), so this is a guard. */
#define WUSH_ERROR_SCRATCH_TOO_SMALL 0x57550001

/* wush_gemm_s4 that allocates nothing and takes no workspace: its split-K
 * partials (if the plan splits K) go to the library's static scratch of
 * WUSH_GEMM_SCRATCH_BYTES on the current device.  The plan is the one
 * wush_gemm_s4 chooses for a workspace of WUSH_GEMM_SCRATCH_BYTES that holds
 * split-K partials only, and the results are those of such a call, bit for
 * bit: a shape whose full split of K would need more partials than the
 * scratch holds is split into fewer slices.  The scratch never holds
 * converted activations, so where wush_gemm_s4 with a workspace converts them
 * once (M > 64, from about 2^32 multiply-adds) this entry point runs the
 * per-tile fp16 tiles or the int8 tiles: equal to the parity tolerance, not
 * bit for bit.  Nothing needs clearing
 * between calls: every partial is written before it is summed.  All calls on
 * one device share its scratch, so calls that overlap on one device (on
 * different streams, or from different host threads without ordering) race.
 * No counterpart in the reference: for callers that cannot allocate device
 * memory (code under HIP graph capture that must not call hipMalloc, tight
 * serving loops, harnesses that forbid allocation). */
int wush_gemm_s4_noalloc(const uint8_t *xq, const uint16_t *xs, const uint8_t *wq, const uint16_t *ws,
                         uint16_t *y, int64_t M, int64_t N, int64_t K, hipStream_t stream);

/* Self-test of the int8 MFMA operand layout the GEMM relies on:
 * c (8x8 int32) = a (8x32 int8, row-major) @ b (32x8 int8, row-major).
 * Replaces s4_atom_selftest (csrc/gemm_s4.cu:74-82). */
int wush_mfma_selftest(const int8_t *a, const int8_t *b, int32_t *c, hipStream_t stream);

/* Per-tensor INT4 quantization: code = clamp(rint(x * inv_scale), -7, 7),
 * packed like the group codes, n bf16 values (n % 32 == 0) -> n/2 bytes.
 * inv_scale_dev, when not NULL, is a device pointer to the fp32 inverse
 * scale and overrides inv_scale.
 * Replaces quant_int4_tensor_scale / _dev (csrc/fast_path.cu:42-59, :92-109). */
int wush_quant_int4_tensor_scale(const uint16_t *x, uint8_t *q, int64_t n, float inv_scale,
                                 const float *inv_scale_dev, hipStream_t stream);

/* Largest K of wush_gemm_s4_tensor_scale: the int8 MFMA multiplies 16*code
 * operands, so the int32 accumulator holds 256 * sum(qx*qw), up to
 * 256 * 64 * K with codes of -8; 256 * 64 * 131040 < 2^31. */
#define WUSH_TENSOR_SCALE_MAX_K 131040

/* Per-tensor W4A4 GEMM: y = alpha * (xq @ wq^T) with an exact int32 dot over
 * all of K, y (M, N) fp16, K % 32 == 0, K <= WUSH_TENSOR_SCALE_MAX_K (larger K
 * is rejected with hipErrorInvalidValue).  alpha_dev, when not NULL, is a
 * device pointer to the fp32 alpha and overrides alpha.
 * Replaces w4a4_gemm_cutlass / _dev (csrc/gemm_cutlass_int4.cu:132-188). */
int wush_gemm_s4_tensor_scale(const uint8_t *xq, const uint8_t *wq, uint16_t *y,
                              int64_t M, int64_t N, int64_t K, float alpha,
                              const float *alpha_dev, hipStream_t stream);

/* ------------------------------------------------------------------------
 * 8-bit operators around the W4A4 layers.  The reference has no counterpart of
 * anything below.
 * ------------------------------------------------------------------------ */

/* Largest K of the W8A8 entry points: 128 * 128 * 131056 < 2^31. */
#define WUSH_W8A8_MAX_K 131056

/* Per-token INT8 quantization of x (rows, K), bf16 or fp16, rows `row_stride`
 * elements apart:
 *   s[m] = max(amax_k |x[m][k]| / 127, 2^-126)
 *   q[m][k] = clamp(rint(x[m][k] * (1 / s[m])), -127, 127)
 * every step one fp32 operation.  A row with a non-finite value gets s = NaN and
 * zero codes.  q: rows*K, s: rows fp32.  K % 16 == 0, K <= WUSH_W8A8_MAX_K, x
 * and q 16-byte aligned, row_stride a multiple of 8. */
int wush_quant_int8_token(const void *x, int dtype, int8_t *q, float *s, int64_t rows, int64_t K,
                          int64_t row_stride, hipStream_t stream);

/* W8A8 product: y[m][n] = (sum_k xq[m][k] wq[n][k]) * xs[m] * ws[n], the sum
 * exact in int32, then two fp32 products and one rounding to `dtype` (bf16 or
 * fp16).  xq (M, K), wq (N, K) int8; xs M, ws N fp32; y (M, N).  Any M, N up to 2^26;
 * K % 16 == 0, K <= WUSH_W8A8_MAX_K; xq and wq 16-byte aligned.  The result's
 * bits depend on neither the workspace nor the plan.  Bytes of workspace with which
 * it runs its fastest plan (int32 partial sums of a split K) are asked of
 * wush_gemm_w8a8_workspace_bytes; with fewer, K is not split. */
size_t wush_gemm_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K);
int wush_gemm_w8a8(const int8_t *xq, const float *xs, const int8_t *wq, const float *ws, void *y, int dtype,
                   int64_t M, int64_t N, int64_t K, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Kernels of wush_gemm_w8a8, as its plan query names them. */
enum wush_w8a8_kernel {
    WUSH_W8A8_DOT = 0,              /* dot products of whole weight rows (M <= 4) */
    WUSH_W8A8_TILES = 1,            /* int8 MFMA tiles through LDS (K % 64 == 0) */
    WUSH_W8A8_STREAM = 2            /* int8 MFMA on weights straight from memory */
};

/* The plan wush_gemm_w8a8 runs with `workspace_bytes` of 16-byte aligned workspace:
 * plan = {kernel, output rows of a workgroup, columns, K slices}.  Host only, no device is
 * touched; for tests and tuning. */
int wush_gemm_w8a8_plan(int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int32_t plan[4]);

/* Both in one call: y = W8A8 product of x (M, K), bf16 or fp16 as y, rows
 * row_stride elements apart, with the same bits as wush_quant_int8_token followed by
 * wush_gemm_w8a8.  The workspace (16-byte aligned, of at least
 * wush_linear_w8a8_workspace_bytes) holds the codes. */
size_t wush_linear_w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K);
int wush_linear_w8a8(const void *x, int64_t row_stride, const int8_t *wq, const float *ws, void *y, int dtype,
                     int64_t M, int64_t N, int64_t K, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* A paged key/value cache in 8 bits: `pages` pages of page_size tokens (16,
 * 32, 64 or 128) for `heads` key/value heads of head_dim channels (64 or 128).
 *   k        int8 (pages, heads, page_size, head_dim)
 *   v        int8 (pages, heads, head_dim, page_size): channel by channel, the
 *            order in which the attention's second product reads it
 *   k_scale, v_scale  fp32 (pages, heads), not negative: a code stands for code * scale
 *            (in attention a value scale below 2^-40, the least that append writes, counts as 2^-40)
 * k and v 16-byte aligned. */
typedef struct wush_kv8_cache {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int64_t pages;
    int32_t heads, page_size, head_dim;
} wush_kv8_cache;

/* Longest sequence that a cache holds: a length beyond it (or below 0) counts as 0. */
#define WUSH_KV8_MAX_LENGTH (1 << 30)

/* The batch that the next two take, all on the device: block_table (seqs,
 * table_stride) int32, a sequence's pages in order; seq_lens (seqs) int32, each
 * sequence's length INCLUDING the call's new tokens, which are its last ones; cu_q
 * (seqs + 1) int32, where each sequence's new tokens begin among the `tokens` rows, from 0
 * up to tokens, or NULL for one new token each (tokens == seqs).  A page number out
 * of [0, pages) stands for no page: nothing is written there, and no query sees
 * its tokens; so do tokens behind the table's end.  Rows that cu_q gives to no sequence (before its
 * first entry, from its last one on) put nothing into the cache and come out as zeros. */

/* Rotates q and k by position, and puts k and v into the cache, of which the
 * new tokens' pages change.  q (tokens, q_heads, head_dim), k, v (tokens, heads,
 * head_dim), bf16 or fp16, each with a token and a head stride: strides = {q token, q head, k token,
 * k head, v token, v head} in elements, multiples of 8, all pointers 16-byte
 * aligned.  Row p of cos_sin (positions, rot) fp32 holds rot / 2 cosines, then rot / 2 sines;
 * positions behind its end take its last row.  The first rot channels (a
 * multiple of 16, at most head_dim; 0: none, and cos_sin may be NULL) turn in pairs (i, i + rot / 2), or (2 i,
 * 2 i + 1) if `interleaved`: (a, b) -> (a c - b s, b c + a s), each product and sum
 * rounded to fp32.  q_out (tokens, q_heads, head_dim), contiguous, rounded once;
 * q_heads = 0: none.
 *   A (page, head)'s scale is s' = max(s, amax of its new tokens / 127, 2^-40),
 * s counting only where it holds older tokens; new codes are
 * clamp(rint(x * (1 / s')), -127, 127), older ones become rint(code * (s / s')).  A non-finite
 * value makes its (page, head)'s scale NaN until the page is begun anew, and what attends to it NaN.
 * Running the same call again changes nothing.  No two sequences of a call may
 * write to one page. */
int wush_kv8_append(const void *q, const void *k, const void *v, int dtype, const int64_t strides[6],
                    const float *cos_sin, int64_t positions, int64_t rot, int interleaved,
                    const wush_kv8_cache *cache, const int32_t *block_table, int64_t table_stride,
                    const int32_t *seq_lens, const int32_t *cu_q, int64_t seqs, int64_t tokens, int64_t q_heads,
                    void *q_out, hipStream_t stream);

/* Attention of the new tokens' queries over the cache (their own keys and
 * values already in it): for the query at position p of its sequence and query head hq, key/value
 * head hq / (q_heads / heads),
 *   out = sum_t softmax_t(cap(scale * q . k_t)) v_t over t in [max(0, p - window + 1), p]
 * with window 0 for all t <= p, and cap(x) = softcap * tanh(x / softcap), softcap 0 for
 * none; scale finite, of either sign.  A query that sees no token gets zeros; one with a non-finite value
 * NaN if it sees any.  q (tokens, q_heads, head_dim)
 * bf16 or fp16 with a token and a head stride (multiples of 8, 16-byte aligned);
 * out (tokens, q_heads, head_dim) contiguous, of the same type.
 *   Scores, sums and outputs are held in fp32.  Fewer bits than that: of q, 2^-23 of its row's
 * largest value; of a score with softcap, 2^-22 of a softcap up to 256, above it 2^-20 of the score; and the
 * weights p_t * v_scale of the sum over v, rounded to 11 bits (fp16), to fewer below 2^-26 of the row's
 * largest and to none from 2^-37 on.  How the work is split, and with it the order of sums, depends on the
 * sizes, window and max_len, not on the values.
 *   max_len: a bound of seq_lens that the host knows (0: the table's room). It only
 * decides how the work is split (a captured call keeps the split that it was captured with).  The workspace, of at least
 * wush_kv8_attention_workspace_bytes for the same arguments (ragged: whether
 * cu_q is given), 16-byte aligned, holds partial results. */
size_t wush_kv8_attention_workspace_bytes(const wush_kv8_cache *cache, int64_t seqs, int64_t tokens, int ragged,
                                          int64_t q_heads, int64_t table_stride, int64_t window, int64_t max_len);
int wush_kv8_attention(const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride,
                       const wush_kv8_cache *cache, const int32_t *block_table, int64_t table_stride,
                       const int32_t *seq_lens, const int32_t *cu_q, int64_t seqs, int64_t tokens, int64_t q_heads,
                       float scale, int64_t window, float softcap, int64_t max_len, void *out, void *workspace,
                       size_t workspace_bytes, hipStream_t stream);

/* The plan wush_kv8_attention runs for the same arguments: plan = {query rows of a
 * workgroup (16, 128 or 256), stretches of the cache, tokens of a stretch, sequences of a
 * round if single tokens' sequences are taken by length, else 0}.  Host only, no device is touched;
 * for tests and tuning. */
int wush_kv8_attention_plan(const wush_kv8_cache *cache, int64_t seqs, int64_t tokens, int ragged, int64_t q_heads,
                            int64_t table_stride, int64_t window, int64_t max_len, int32_t plan[4]);

/* Pages as values: k, v (n, heads, page_size, head_dim) bf16 or fp16, code *
 * scale rounded once, of the n pages listed (device int32).  A page number out
 * of range gives NaN. */
int wush_kv8_read(const wush_kv8_cache *cache, const int32_t *pages, int64_t n, int dtype, void *k, void *v,
                  hipStream_t stream);

/* ------------------------------------------------------------------------
 * Products in 8-bit floating point, and layers of experts on them.  Codes are e4m3 bytes (four
 * exponent bits, three fraction bits, no infinities, largest 448).
 * ------------------------------------------------------------------------ */

/* Largest K of the e4m3 entry points. */
#define WUSH_FP8_MAX_K 131056

/* Quantization of x (rows, K), bf16 or fp16, rows `row_stride` elements apart, with a scale for each
 * row and block b of 128 channels (the last one may be shorter):
 *   A = max(amax |x[m][k in b]|, 448 * 2^-126),  s[b][m] = A / 448,  q[m][k] = e4m3(448 x[m][k] / A)
 * A / 448 rounded to fp32, the code the one nearest to the quotient itself, halves to even.  A block with a
 * non-finite value gets s = NaN and zero codes.  q: rows*K bytes; s: (K / 128, rows) fp32, block by block.
 * K % 16 == 0, K <= WUSH_FP8_MAX_K, at most 2^26 rows, x and q 16-byte aligned, row_stride a multiple of 8. */
int wush_quant_fp8_block(const void *x, int dtype, uint8_t *q, float *s, int64_t rows, int64_t K,
                         int64_t row_stride, hipStream_t stream);

/* Product with a scale for each row of x and block of 128 channels, and each block of 128 x 128 weights:
 *   y[m][n] = sum_b (sum_{k in b} xq[m][k] wq[n][k]) * xs[b][m] * ws[n / 128][b]
 * sums in fp32, the two scales multiplied first, rounded once to `dtype` (bf16 or fp16).  xq (M, K), wq (N, K) codes; xs (K / 128, M), ws
 * (N / 128, K / 128) fp32, sizes rounded up; y (M, N).  M, N up to 2^26, K % 16 == 0, K <= WUSH_FP8_MAX_K;
 * xq and wq 16-byte aligned, and y too where N % 8 == 0.  The order of the sums depends on M, N, K and the workspace: of the size asked of
 * wush_gemm_fp8_workspace_bytes it holds partial sums of a split K; with less, K is not split. */
size_t wush_gemm_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K);
int wush_gemm_fp8(const uint8_t *xq, const float *xs, const uint8_t *wq, const float *ws, void *y, int dtype,
                  int64_t M, int64_t N, int64_t K, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Kernels of wush_gemm_fp8, as its plan query names them. */
enum wush_fp8_kernel {
    WUSH_FP8_DOT = 0,               /* fp32 dot products of whole weight rows: M = 1 with K <= 32768, M = 2 with K <= 16384, M = 3
                                       and 4 with K <= 8192 */
    WUSH_FP8_TILES = 1              /* MFMA tiles through LDS, whose products are cut at 2^-13 of the largest of 8 */
};

/* The plan wush_gemm_fp8 runs with `workspace_bytes` of 16-byte aligned workspace:
 * plan = {kernel, output rows of a workgroup, columns, K slices}.  Host only, no device is
 * touched; for tests and tuning. */
int wush_gemm_fp8_plan(int64_t M, int64_t N, int64_t K, size_t workspace_bytes, int32_t plan[4]);

/* Both in one call: y = product of x (M, K), bf16 or fp16 as y, rows row_stride elements apart, quantized
 * as above.  The workspace (16-byte aligned, of at least wush_linear_fp8_workspace_bytes) holds the codes. */
size_t wush_linear_fp8_workspace_bytes(int64_t M, int64_t N, int64_t K);
int wush_linear_fp8(const void *x, int64_t row_stride, const uint8_t *wq, const float *ws, void *y, int dtype,
                    int64_t M, int64_t N, int64_t K, void *workspace, size_t workspace_bytes, hipStream_t stream);

#define WUSH_MOE_MAX_EXPERTS 1024
#define WUSH_MOE_MAX_CHOICES 64

/* How a router chooses: k experts of those of the best keep_groups of `groups` groups of equal size
 * (experts one after another), a group's score being the sum of its group_best (1 or 2) largest. */
typedef struct wush_moe_choice {
    int32_t k, groups, keep_groups, group_best;
    int32_t sigmoid;                /* scores sigmoid(x), else softmax(x) over all experts */
    int32_t renorm;                 /* weights divided by their sum */
    float scale;                    /* factor of the weights */
} wush_moe_choice;

/* The router's choice for each row of logits (rows, experts), bf16, fp16 or fp32, rows `row_stride`
 * elements apart: scores s, choices by c = s + bias (experts fp32, all in 64 bits).  Where bias is NULL x itself
 * orders the experts, and the groups too with a group_best of 1, as exact scores would: logits whose scores are equal in
 * 64 bits (sigmoids above some 37) still differ.  Sums of two scores are in 64 bits, with a bias or without.
 * ids (rows, k) the k experts of the largest c in the groups that stay, in falling order, equal ones by rising
 * index; weights (rows, k) = s[ids], with renorm divided by their sum (a sum of 0 gives zeros), times scale, in
 * 64 bits and rounded once.  A NaN counts below every number.  A row of nothing but -inf has scores of 0; with softmax
 * a NaN or +inf makes all of the row's scores NaN.  experts <= 1024, groups <= 64, k <= 64. */
int wush_moe_route(const void *logits, int dtype, int64_t row_stride, const float *bias, int64_t rows, int64_t experts,
                   const wush_moe_choice *choice, float *weights, int32_t *ids, hipStream_t stream);

/* A layer of E gated experts: y[t] = sum_j weights[t][j] * down_e(silu(gate_e(x[t])) * up_e(x[t])), e = ids[t][j]
 * (an id out of [0, E) adds nothing).  x (T, H), rows row_stride elements apart, and y (T, H) bf16 or fp16; weights fp32
 * and ids int32 (T, k).  w_up codes (E, 2 I, H), the gate's I rows before the up projection's, s_up
 * (E, 2 I / 128, H / 128); w_down (E, H, I), s_down (E, H / 128, I / 128).  Both inner inputs are quantized as by
 * wush_quant_fp8_block, all else in fp32, but for an expert's rows of a bf16 y, which may be held in
 * fp16 with a power of two for each 64 columns; y rounded once.  H % 16 == 0, I % 128 == 0, E <= 1024, k <= 64.  The workspace is 16-byte
 * aligned, of at least wush_moe_experts_fp8_workspace_bytes. */
size_t wush_moe_experts_fp8_workspace_bytes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int dtype);
int wush_moe_experts_fp8(const void *x, int dtype, int64_t row_stride, const float *weights, const int32_t *ids,
                         const uint8_t *w_up, const float *s_up, const uint8_t *w_down, const float *s_down, void *y,
                         int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, void *workspace,
                         size_t workspace_bytes, hipStream_t stream);

/* Ways of wush_moe_experts_fp8, as its plan query names them, and which of their products the e4m3 matrix instruction
 * makes, which cuts a product at 2^-13 of the largest of the 8 that it adds at once. */
enum wush_moe_experts_way {
    WUSH_MOE_DOT = 0,               /* dot products, an expert's weights read for each choice; none */
    WUSH_MOE_ROWS = 1,              /* rows sorted by expert, tiles of 32 x 64; the down projection's */
    WUSH_MOE_FUSED = 2              /* tiles of 64 or 128 x 256; the down projection's, and a bf16 y's experts' rows are fp16 */
};

/* The plan wush_moe_experts_fp8 runs: plan = {way, rows of a tile (0: no tiles), whether most experts have one
 * tile, whose weights bypass the caches, tokens taken at once}.  Host only, no device is touched; for tests and tuning. */
int wush_moe_experts_fp8_plan(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I, int dtype, int32_t plan[4]);

#ifdef __cplusplus
}
#endif

#endif /* WUSH_INT4_H */
