/*
 * sbq.h - C ABI of the MI355X (gfx950) quantized-linear library (libsbq.so).
 *
 * This is the drop-in boundary for the quantized-linear hot path of
 * spikingbrain-cpu: the `int8` (weight-only, symmetric per-output-channel
 * int8, fp32 scales) and `int8-dyn` (W8A8 with dynamic per-tensor asymmetric
 * uint8 activations, fbgemm semantics) formats of spikingbrain_cpu/quant.py.
 *
 * Conventions (all entry points):
 *   - plain pointers and sizes only; every pointer named `d_*` or documented as
 *     "device" is HIP device memory owned by the caller.  The library never
 *     allocates device memory: scratch space is passed in as `workspace`.
 *   - `stream` is a hipStream_t passed as void* (NULL = the null stream).
 *     Every call is asynchronous on that stream and reentrant: the library
 *     keeps no mutable state between calls.
 *   - matrices are row-major; `ld*` is the row stride in elements.  Row and
 *     column counts (M, N, K) above 2^31 - 1 are rejected with SBQ_ERR_ARG.
 *   - return value: SBQ_OK (0) or a negative SBQ_ERR_* code; nothing throws.
 *     sbq_status_string() names a code.
 *
 * Reference interfaces replaced (paths relative to the reference repository):
 *   sbq_quantize_per_channel  <- spikingbrain_cpu/quant.py:25-29 quantize_per_channel
 *   sbq_repack_w8             <- spikingbrain_cpu/quant.py:33-39 Int8Linear.__init__ buffers
 *                                and quant.py:57-61 DynamicInt8Linear.__init__ (linear_prepack)
 *   sbq_linear_w8             <- spikingbrain_cpu/quant.py:41-53 Int8Linear.forward
 *   sbq_act_qparams           <- spikingbrain_cpu/quant.py:65 (the per-tensor activation
 *                                quantization parameters chosen inside
 *                                torch.ops.quantized.linear_dynamic)
 *   sbq_act_quant_per_tensor  <- spikingbrain_cpu/quant.py:65 (those parameters and the
 *                                uint8 activations linear_dynamic multiplies)
 *   sbq_linear_w8a8           <- spikingbrain_cpu/quant.py:63-66 DynamicInt8Linear.forward
 *   sbq_argmax_rows           <- spikingbrain_cpu/engine.py:30-31 (greedy sampling,
 *                                int(logits.argmax()) over the lm_head output of
 *                                model.py:447), so the logits need not leave the GPU
 *   sbq_linear_w8_argmax,     <- spikingbrain_cpu/model.py:445-447 (lm_head) and
 *   sbq_linear_w8a8_argmax       engine.py:30-31 (its greedy token) in one launch
 *   sbq_sample_rows           <- spikingbrain_cpu/engine.py:29-42 sample (temperature,
 *                                top-k, top-p and the draw) over the lm_head logits
 *   sbq_tree_attention        <- spikingbrain_cpu/model.py:208-229 attention over the cached
 *                                keys (and over a tree of drafted tokens)
 *   sbq_qk_norm_rope          <- spikingbrain_cpu/model.py:260-270 (the head norms) and
 *                                model.py:46-51 (the rotation), before the attention
 * Additions without a counterpart: the 4-bit linears (sbq_linear_w4), the bounded
 * cache (sbq_kv_append, sbq_kv_take), the paged cache of several sequences
 * (sbq_paged_append, sbq_paged_read, sbq_paged_attention), the choice among
 * drafted tokens (sbq_verify_drafts).
 */
#ifndef SBQ_H_
#define SBQ_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define SBQ_OK 0
#define SBQ_ERR_ARG (-1)        /* bad size / stride / null pointer           */
#define SBQ_ERR_DTYPE (-2)      /* unsupported dtype code                      */
#define SBQ_ERR_ALIGN (-3)      /* pointer not aligned as the entry requires   */
#define SBQ_ERR_WORKSPACE (-4)  /* workspace missing or too small              */
#define SBQ_ERR_LAUNCH (-5)     /* hipLaunchKernel / HIP runtime error         */
#define SBQ_ERR_DEVICE (-6)     /* current device is not a gfx950 GPU          */

/* ---- dtype codes -------------------------------------------------------- */
#define SBQ_F32 0
#define SBQ_F16 1
#define SBQ_BF16 2

/* Library version string, e.g. "sbq 0.1.0 gfx950". */
const char* sbq_version(void);

/* Human-readable name of a status code. */
const char* sbq_status_string(int status);

/* Checks that the current HIP device is a gfx950 part the kernels were built
 * for.  Returns SBQ_OK or SBQ_ERR_DEVICE.  Optional: every compute entry point
 * reports a launch failure on its own. */
int sbq_check_device(void);

/* ---- weight quantization and packing ------------------------------------ */

/* quantize_per_channel (spikingbrain_cpu/quant.py:25-29):
 *   scale[n] = max(max_k |w[n,k]|, 1e-8f) / 127.0f      (IEEE fp32 division)
 *   q[n,k]   = clamp(rint(w[n,k] / scale[n]), -127, 127) (IEEE fp32 division,
 *                                                         round-half-even)
 * w: device [N, K] (row stride ldw) of dtype w_dtype (F32, F16 or BF16; the
 * value is widened to fp32 exactly, as weight.float() does).
 * q: device int8 [N, K] (row stride ldq).  scale: device fp32 [N]. */
int sbq_quantize_per_channel(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ldw,
                             int8_t* q, int64_t ldq, float* scale, void* stream);

/* Bytes of the packed weight layout for an [N, K] int8 matrix:
 * round_up(N,16) * round_up(K,64).  The layout is a grid of 1 KiB tiles
 * [N/16][K/64]; tile (nt,kc) holds rows nt*16..+15, columns kc*64..+63, with
 * byte  lane*16 + j,  lane = g*16 + r,  equal to  q[nt*16+r][kc*64+g*16+j] ^ 0x80
 * (offset binary, padding = 0x80 i.e. q = 0).  One tile is exactly one
 * 64-lane x 16-byte wavefront load and one MFMA 16x16 operand fragment pair. */
int64_t sbq_packed_bytes(int64_t N, int64_t K);

/* Repack (the loader hook of spikingbrain_cpu/loader.py:46-51,94; the buffers of
 * quant.py:33-39 and the prepack of quant.py:57-61):
 *   q: device int8 [N, K] (row stride ldq)  ->  packed: device, sbq_packed_bytes(N,K)
 *   colsum: device int32 [N] or NULL; colsum[n] = sum_k q[n,k]  (needed by
 *   sbq_linear_w8a8 for the activation zero-point correction). */
int sbq_repack_w8(const int8_t* q, int64_t N, int64_t K, int64_t ldq,
                  uint8_t* packed, int32_t* colsum, void* stream);

/* sbq_quantize_per_channel and sbq_repack_w8 in one pass over the weight:
 * scale, packed, and where asked for the int8 rows q (NULL: not written) and
 * colsum (NULL: not written), the same values as those two calls. */
int sbq_quantize_pack_w8(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ldw,
                         int8_t* q, int64_t ldq, float* scale, uint8_t* packed,
                         int32_t* colsum, void* stream);

/* Inverse of sbq_repack_w8: packed -> q [N, K] (row stride ldq). */
int sbq_unpack_w8(const uint8_t* packed, int64_t N, int64_t K, int8_t* q, int64_t ldq,
                  void* stream);

/* ---- int8 weight-only linear (Int8Linear.forward, quant.py:41-53) -------- */

/* y[m,n] = (sum_k x[m,k] * q[n,k]) * scale[n] (+ bias[n])
 * x: device [M, K] (row stride ldx), dtype F32, F16 or BF16.
 *    F16/BF16 inputs are used exactly (BF16 staged for the prefill GEMM: exact
 *    down to 2^28 below each row's maximum).  F32 inputs: on the decode paths
 *    (M <= 16, and the general GEMV up to 32 tokens) and on every path of a
 *    ragged K split into bf16 hi + remainder (relative representation error
 *    <= 2^-16); on the staged prefill path of 64 | K one fp16 plane of the row
 *    scaled by a power of two (11 significant bits: about 3e-4 relative L2 on
 *    the outputs).
 * packed: from sbq_repack_w8.  scale: device fp32 [N].  bias: device fp32 [N]
 * or NULL.  y: device [M, N] (row stride ldy), dtype F32, F16 or BF16.
 * Accumulation is fp32.  Routes (16-byte aligned rows, 64 | K): M <= 16 the
 * HBM-streaming MFMA GEMV; 16 < M <= 64 the row-tile GEMV on narrow layers
 * (N <= 4096 with little x to read, or wherever the workspace below is
 * missing), else the LDS-tiled MFMA GEMM.  Ragged K (K % 64 != 0), with the
 * workspace below: x copied to rows of whole tiles, then the GEMV (M <= 16) or
 * the tiled GEMM on those, up to 32 tokens only where that pays (longer K and
 * wider layers); what is left up to 32 tokens, and misaligned rows of whole
 * tiles, the general GEMV.
 * workspace: optional (NULL, 0 is valid).  With >= sbq_w8_workspace_bytes(M,
 * K, x_dtype) bytes the prefill GEMM runs its fastest path: F16 x with per-row
 * sums from a pre-pass; BF16 / F32 x staged as a power-of-two scaled fp16 plane
 * for the same fp16 MFMA kernel (aligned rows, 64 | K); ragged K as above, in
 * x's own dtype or (F32) bf16 high and remainder planes.  With
 * sbq_linear_workspace_bytes it also splits K over workgroups on small grids.
 * Without it, F16 / BF16 run a slower tiled GEMM and F32 and ragged K a
 * register-staged one. */
int sbq_linear_w8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                  const uint8_t* packed, const float* scale, const float* bias, int64_t N,
                  void* y, int y_dtype, int64_t ldy,
                  void* workspace, size_t workspace_bytes, void* stream);

/* sbq_linear_w8 with its N columns stored as parts: the columns belong to
 * consecutive parts whose widths are multiples of 4, and part p is a dense
 * [M, width] matrix of y_dtype starting at element M * pstart(p) of y, where
 * start(p) is the part's first column and pstart(p) the sum of the earlier
 * widths, each rounded up to a multiple of 64.  For projections fused into
 * one layer whose outputs go separate ways (model.py:262-264, 363-365): the
 * parts leave the launch contiguous, with no copies after it.
 * y: device, 16-byte aligned, M * (sum of the widths, each rounded up to 64)
 * elements.  parts: device int32 [N/4][2], per 4 columns the width of their
 * part and start/4 | ((pstart - start)/4) << 20 (so N < 2^22, and padding
 * below 2^14 columns before any part), written by sbq_parts_table from the
 * widths (a host array; SBQ_ERR_ARG when they do not fit the table).
 * Everything else as sbq_linear_w8. */
int sbq_parts_table(const int64_t* widths, int count, int32_t* parts, void* stream);
int sbq_linear_w8_parts(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                        const uint8_t* packed, const float* scale, const float* bias, int64_t N,
                        void* y, int y_dtype, const int32_t* parts,
                        void* workspace, size_t workspace_bytes, void* stream);

/* `count` (1..SBQ_MAX_GROUP) independent weight-only linears that share M, K,
 * x_dtype and y_dtype, in one launch where the decode path applies: linear i
 * is y_i = linear(x_i, packed_i, scale_i, bias_i) exactly as sbq_linear_w8
 * defines it (x_i rows of stride ldx[i], y_i [M, N[i]] of stride ldy[i]).
 * The arguments are host arrays of `count` device pointers / sizes; `bias`
 * may be NULL (no biases) or hold NULL entries.  For decode shapes (M <= 16,
 * K % 64 == 0, 16-byte aligned x rows) the linears run as one GEMV launch:
 * the launch ramp and tail of a small projection are paid once per group
 * (two 4096 x 4096 projections of different inputs: 2 x 5.1 us -> 7.5 us).
 * Otherwise each runs as sbq_linear_w8 without a workspace (a caller that has
 * one is faster with separate calls for ragged K and M > 16).  Results may differ
 * from separate sbq_linear_w8 calls in the fp32 summation order (the group is
 * tiled as one layer of its summed rows).  No counterpart in the reference:
 * it is for callers holding several independent projections of one step
 * (model.py: the two lora up-projections, the SSE and SWA output projections
 * of a hybrid layer). */
#define SBQ_MAX_GROUP 4
int sbq_linear_w8_grouped(int count, const void* const* x, const int64_t* ldx, int x_dtype,
                          int64_t M, int64_t K, const uint8_t* const* packed,
                          const float* const* scale, const float* const* bias, const int64_t* N,
                          void* const* y, const int64_t* ldy, int y_dtype, void* stream);

/* Workspace bytes that let sbq_linear_w8 run its fastest prefill path for an
 * [M, K] input of x_dtype, and ragged K (K % 64 != 0) as rows of whole tiles:
 * 2 * M floats, plus the staged activations, plus alignment slack.  Staged are
 * BF16 and F32 x of 64 | K, M * K * 2 bytes, and every ragged x, M *
 * ceil(K/64)*64 elements of 2 bytes (F16, BF16) or 4 (F32).  0 for a bad
 * argument.  No counterpart in the reference (its CPU matmul needs no
 * scratch). */
int64_t sbq_w8_workspace_bytes(int64_t M, int64_t K, int x_dtype);

/* Workspace bytes that let sbq_linear_w8 (w8a8 = 0) or sbq_linear_w8a8
 * (w8a8 = 1) run their fastest path for y [M, N] = x [M, K] * W^T with x of
 * x_dtype: the sizes of sbq_w8_workspace_bytes / sbq_w8a8_workspace_bytes
 * plus, for shapes that reach the tiled GEMM with a grid that would leave CUs
 * idle, the tile counters and fp32 / int32 partial tiles of a GEMM that
 * splits K over workgroups (its
 * last split per tile adds the partials in a fixed order, so results do not
 * depend on timing).  Those entry points split K only when given this much;
 * with the smaller sizes they run the same shapes unsplit.  0 for a bad
 * argument.  No counterpart in the reference (its CPU matmul needs no
 * scratch). */
int64_t sbq_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_dtype, int w8a8);

/* Plan of the tiled prefill GEMM for y [M, N] = x [M, K] * W^T with x of
 * x_dtype, as sbq_linear_w8 (w8a8 = 0) and sbq_linear_w8a8 (w8a8 = 1) run it
 * when given sbq_linear_workspace_bytes of workspace: returns the block
 * configuration id (>= 0) and stores in *splits (if not NULL) the number of
 * workgroups K is split over, or 0 when calls of this shape (16-byte aligned
 * rows, that workspace) never reach the GEMM: the decode GEMVs and the
 * row-tile GEMV run them.  Host-only: needs no GPU.
 * SBQ_ERR_ARG / SBQ_ERR_DTYPE for a bad argument.  No counterpart in the
 * reference (diagnostics and tests of the configuration choice). */
int sbq_gemm_config(int64_t M, int64_t N, int64_t K, int x_dtype, int w8a8, int* splits);

/* The general decode GEMV's configuration for an [M, K] input of x_dtype
 * (weight-only: the kernel that runs misaligned rows and ragged K where
 * padding the rows does not pay, and 17..32 tokens on the layers the
 * row-tile GEMV leaves; int8-dyn: 17..32 tokens alone, since up to 16 never
 * reach it and report unsupported): info[0..8] = supported (0 / 1), row
 * tiles of x, weight tiles per group, K tiles per wave, waves per
 * workgroup, activation mode (0 registers, 1 LDS, 2 chunks), staging
 * chunks per thread, LDS bytes, and whether a kernel instance exists for
 * it.  Host-only: needs no GPU.  SBQ_ERR_ARG / SBQ_ERR_DTYPE for a bad
 * argument.  No counterpart in the reference (diagnostics and tests of the
 * configuration choice). */
int sbq_gemv_config(int64_t M, int64_t K, int x_dtype, int w8a8, int32_t* info);

/* ---- int8-dyn W8A8 linear (DynamicInt8Linear.forward, quant.py:63-66) ---- */

/* Workspace bytes sbq_linear_w8a8 / sbq_act_qparams need for an [M, K] input:
 * 2.5 KiB of activation statistics plus M * ceil(K/64)*64 bytes for the
 * quantized activations of the paths with a quantize pre-pass (M > 16, ragged
 * or misaligned x, and decode inputs beyond what the GEMV quantizes itself), M
 * floats of per-token scales (sbq_linear_w8a8_token), plus alignment slack. */
int64_t sbq_w8a8_workspace_bytes(int64_t M, int64_t K);

/* The activation quantization parameters that fbgemm's dynamic linear chooses
 * for the whole tensor x [M, K] (uint8, qmin 0, qmax 255, no range reduction):
 *   lo = min(min x, 0), hi = max(max x, 0)
 *   scale = (double)(hi - lo) / 255, replaced by 0.1 when fp32(scale) == 0 or
 *   1/fp32(scale) overflows; scales below 6.1e-5 are raised to 6.1e-5 with
 *   lo/hi rescaled; zero_point chosen from lo or hi by the smaller error term
 *   and rounded half-even (all in double), clamped to [0, 255].
 * Results: *scale_out (device fp32[1]) and *zp_out (device int32[1]). */
int sbq_act_qparams(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                    float* scale_out, int32_t* zp_out,
                    void* workspace, size_t workspace_bytes, void* stream);

/* The activation quantization itself, the step inside
 * quantized::linear_dynamic (spikingbrain_cpu/quant.py:65) that the int8-dyn
 * entry points below fuse into their kernels: the (scale, zero_point) of
 * sbq_act_qparams, then
 *   xq[m,k] = clamp(rint(fma(x[m,k], 1/scale, zero_point)), 0, 255)
 * (one rounding, half to even) into device uint8 xq [M, K] with row stride
 * ldq >= K; sbq_linear_w8a8's acc equals sum_k (xq[m,k] - zp) * q[n,k].
 * Results: *scale_out (device fp32[1]), *zp_out (device int32[1]).
 * workspace: >= sbq_w8a8_workspace_bytes(M, K) bytes. */
int sbq_act_quant_per_tensor(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                             uint8_t* xq, int64_t ldq, float* scale_out, int32_t* zp_out,
                             void* workspace, size_t workspace_bytes, void* stream);

/* y[m,n] = fp32(acc[m,n]) * fp32(s_x * scale[n]) (+ bias[n]) where
 *   xq[m,k]  = clamp(rint(fma(x[m,k], 1/s_x, zp)), 0, 255)   (one rounding)
 *   acc[m,n] = sum_k (xq[m,k] - zp) * q[n,k]                  (exact int32)
 * which is bit-exact with torch.ops.quantized.linear_dynamic (fbgemm) on the
 * same fp32 inputs.  colsum: from sbq_repack_w8 (required).
 * acc_out: device int32 [M, N] (row stride N) or NULL; when given, the raw
 * int32 accumulators are written too (the bit-exactness check).
 * workspace: >= sbq_w8a8_workspace_bytes(M, K) bytes of device memory. */
int sbq_linear_w8a8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                    const uint8_t* packed, const float* scale, const int32_t* colsum,
                    const float* bias, int64_t N,
                    void* y, int y_dtype, int64_t ldy, int32_t* acc_out,
                    void* workspace, size_t workspace_bytes, void* stream);

/* sbq_linear_w8a8 with its columns stored as parts (see
 * sbq_linear_w8_parts for y and parts). */
int sbq_linear_w8a8_parts(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                          const uint8_t* packed, const float* scale, const int32_t* colsum,
                          const float* bias, int64_t N, void* y, int y_dtype,
                          const int32_t* parts, void* workspace, size_t workspace_bytes,
                          void* stream);

/* `count` (1..SBQ_MAX_GROUP) independent int8-dyn linears of one M, K and
 * dtypes: y_i = sbq_linear_w8a8(x_i, packed_i, scale_i, colsum_i, bias_i,
 * N_i) for each i, every x_i quantized with its own (s_x, zp).  Arguments as
 * in sbq_linear_w8_grouped, plus host arrays of the column sums (required)
 * and one workspace of >= sbq_w8a8_workspace_bytes(M, K) bytes.  For decode
 * shapes whose x fits the fused GEMV (each workgroup reduces its linear's
 * min/max itself) the linears run as one launch; larger decode inputs, given
 * `count` times those bytes, as two: every input quantized into its own share,
 * then one GEMV; otherwise one by one as sbq_linear_w8a8, sharing the
 * workspace in stream order.  Bit-exact with
 * separate calls (integer accumulation).  No counterpart in the reference:
 * it is for callers holding several independent int8-dyn projections of one
 * step (model.py: the two lora up-projections, the SSE and SWA output
 * projections of a hybrid layer). */
int sbq_linear_w8a8_grouped(int count, const void* const* x, const int64_t* ldx, int x_dtype,
                            int64_t M, int64_t K, const uint8_t* const* packed,
                            const float* const* scale, const int32_t* const* colsum,
                            const float* const* bias, const int64_t* N, void* const* y,
                            const int64_t* ldy, int y_dtype, void* workspace,
                            size_t workspace_bytes, void* stream);

/* Largest quantized-activation scratch of sbq_linear_w8a8_noalloc:
 * M * ceil(K/64)*64 bytes must not exceed it (e.g. M = 2048 at K = 4096,
 * M = 512 at K = 12288). */
#define SBQ_NOALLOC_XQ_BYTES (8 << 20)

/* sbq_linear_w8a8 without a workspace: no counterpart in the reference.  It is
 * for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc); it calls no
 * allocating routine.  Same arguments, results and bit-exactness as
 * sbq_linear_w8a8.  Its scratch (activation min/max partials, (s_x, zp), the
 * quantized activations) is a static device array of 2304 bytes +
 * SBQ_NOALLOC_XQ_BYTES that each GPU the library runs on holds until the
 * process ends; the first call on a device looks up that device's copy (make
 * it outside graph capture).  Inputs with M * ceil(K/64)*64 >
 * SBQ_NOALLOC_XQ_BYTES return SBQ_ERR_WORKSPACE before any launch.  Every call
 * on one GPU shares that GPU's array: calls that overlap on one GPU (other
 * streams, other threads) race on it.  Nothing in it needs clearing between
 * calls (each call writes every byte it reads). */
int sbq_linear_w8a8_noalloc(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                            const uint8_t* packed, const float* scale, const int32_t* colsum,
                            const float* bias, int64_t N,
                            void* y, int y_dtype, int64_t ldy, int32_t* acc_out, void* stream);

/* Per-token symmetric W8A8: an opt-in granularity with no counterpart in the
 * reference, whose int8-dyn (quant.py:63-66, sbq_linear_w8a8 above) is
 * per-tensor asymmetric; it does not reproduce the reference's outputs.  Each
 * activation row is quantized exactly as quantize_per_channel (quant.py:25-29)
 * quantizes a weight row:
 *   s_t[m] = max(max_k |x[m,k]|, 1e-8) / 127      (IEEE fp32 division)
 *   xq[m,k] = clamp(rne(x[m,k] / s_t[m]), -127, 127)
 *   acc[m,n] = sum_k xq[m,k] * q[n,k]            (int32, exact; acc_out nullable)
 *   y[m,n] = fp32(acc) * fp32(s_t[m] * scale[n]) (with a bias: one fma)
 * workspace: >= sbq_w8a8_workspace_bytes(M, K) bytes; with
 * sbq_linear_workspace_bytes the GEMM splits K over workgroups on small grids.
 * Small decode inputs are quantized in the HBM-streaming int8 MFMA GEMV itself;
 * otherwise the row quantizer runs first, then that GEMV on the s8 rows (M <=
 * 16), the row-tile GEMV on narrow layers (M <= 64) or the tiled int8 MFMA
 * GEMM. */
int sbq_linear_w8a8_token(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                          const uint8_t* packed, const float* scale, const float* bias, int64_t N,
                          void* y, int y_dtype, int64_t ldy, int32_t* acc_out,
                          void* workspace, size_t workspace_bytes, void* stream);

/* ---- lm_head and the greedy token in one pass ---------------------------- */

/* Bytes of the argmax state of the two entry points below. */
#define SBQ_ARGMAX_WS_BYTES 16640

/* Int8Linear.forward over the lm_head weights (model.py:445-447 ->
 * quant.py:41-53) followed by greedy token selection (engine.py:30-31,
 * int(logits.argmax())):
 *   y      = the fp32 logits [M, N] (row stride ldy), as sbq_linear_w8
 *            computes them;
 *   idx[m] = the first n with y[m, n] maximal over row m, NaN above every
 *            number (torch.argmax; the same token sbq_argmax_rows picks on y).
 * At decode sizes (M <= 16, K % 64 == 0, 16-byte aligned x rows) the token is
 * picked inside the GEMV launch (its last workgroup decodes it); other shapes
 * run sbq_linear_w8 (with the optional workspace, as there) and then
 * sbq_argmax_rows.  argmax_ws: SBQ_ARGMAX_WS_BYTES of device memory, 8-byte
 * aligned, all zero before the first call; every call leaves it zero again.
 * Calls that can overlap (other streams) need their own argmax_ws.  idx:
 * device int64 [M]. */
int sbq_linear_w8_argmax(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                         const uint8_t* packed, const float* scale, const float* bias, int64_t N,
                         float* y, int64_t ldy, int64_t* idx,
                         void* workspace, size_t workspace_bytes, void* argmax_ws, void* stream);

/* The same for DynamicInt8Linear.forward (quant.py:63-66): y as
 * sbq_linear_w8a8 computes it (bit-exact with fbgemm), then the greedy token.
 * workspace: as for sbq_linear_w8a8.  argmax_ws: as above. */
int sbq_linear_w8a8_argmax(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                           const uint8_t* packed, const float* scale, const int32_t* colsum,
                           const float* bias, int64_t N, float* y, int64_t ldy, int64_t* idx,
                           void* workspace, size_t workspace_bytes, void* argmax_ws, void* stream);

/* ---- greedy token selection (engine.py:30-31) ---- */

/* idx[m] = the first n with y[m, n] maximal over row m of fp32 y [M, N] (row
 * stride ldy); NaN ranks above every number (torch.argmax semantics).
 * idx: device int64 [M]. */
int sbq_argmax_rows(const float* y, int64_t M, int64_t N, int64_t ldy, int64_t* idx, void* stream);

/* ---- non-greedy sampling (engine.py:29-42, sample) ---- */

/* Workspace bytes of sbq_sample_rows for M rows (about 270 KB per row, for
 * any vocabulary size up to 2^23).  0 for a bad argument. */
int64_t sbq_sample_workspace_bytes(int64_t M, int64_t V);

/* tokens[m] = the engine's sample() of row m of fp32 logits [M, V] (row
 * stride ld), as spikingbrain_cpu/engine.py:29-42 computes it:
 *   temperature <= 0: the greedy token (sbq_argmax_rows; u and the workspace
 *     may be NULL);
 *   z = logits / temperature (fp32 division); top_k > 0: tokens below the
 *     min(top_k, V)-th largest z are masked; p = softmax(z);
 *   0 < top_p < 1: a token is kept while the probability mass of the tokens
 *     above it stays below top_p, the tokens taken in the order of z (of
 *     two tokens of equal fp32 probability the larger z first; the
 *     reference's sort leaves their order open); of tokens of equal z at
 *     that boundary, as many as the rule admits, first in vocabulary order
 *     (a stable sort's order);
 *   the draw: the first index (vocabulary order) whose prefix of kept mass
 *     exceeds u[m] * (kept mass), u: device fp32 [M] uniforms in [0, 1), one
 *     per row, drawn by the caller (torch.multinomial's distribution; the
 *     caller's generator supplies the randomness).
 * Masses are exact sums of the fp32 probabilities truncated to 2^-40, so the
 * result does not depend on timing.  A row with a NaN, or an infinite
 * maximum after the division (where the reference raises), gets token -1.
 * tokens: device int64 [M].  M <= 65535, V <= 2^23 (a row's mass, at most
 * V * 2^40, fits 64 bits).  Rows are independent. */
int sbq_sample_rows(const float* logits, int64_t M, int64_t V, int64_t ld, float temperature, int64_t top_k,
                    float top_p, const float* u, int64_t* tokens, void* workspace, size_t workspace_bytes,
                    void* stream);

/* ---- linears with 4-bit weights and group scales ------------------------ */

/* The int8 weight-only linear's counterpart at half the weight bytes; no
 * counterpart in the reference.  A row of the weight has one scale per group
 * of 32, 64 or 128 consecutive columns (the last group of a ragged K is
 * shorter), held in bf16:
 *   scale[n,G] = bf16(max(max_{k in G} |w[n,k]|, 1e-8f) / 7.0f)
 *   q[n,k]     = clamp(rint(w[n,k] / fp32(scale[n,G])), -7, 7)
 * (IEEE fp32 divisions, half to even; the weights must be finite).
 * w: device [N, K] (row stride ldw), F32, F16 or BF16.  q: device int8 [N, K]
 * (row stride ldq).  scale: device bf16 [N, ceil(K/group)]. */
int sbq_quantize_groups(const void* w, int w_dtype, int64_t N, int64_t K, int64_t ldw, int group,
                        int8_t* q, int64_t ldq, void* scale, void* stream);

/* The layout that sbq_linear_w4 streams.  packed: ceil(N/16) x ceil(K/128)
 * tiles of 1 KiB; tile (nt,kt) holds rows nt*16..+15 and columns
 * kt*128..+127, its 32-bit word lane*4 + s, lane = g*16 + r, the 8 columns
 * kt*128 + 32s + 8g + j of row nt*16 + r: column j = 2i in bits 4i..4i+3,
 * column 2i + 1 in bits 16+4i..19+4i, each as q + 8 (padding 8, that is 0).
 * gscale: bf16 [ceil(N/16)][ceil(K/128) * 128/group][16], the 16 rows of a
 * tile side by side (padding 0).  q: values outside -8..7 are clamped.
 * packed and gscale: device, 16-byte aligned. */
int64_t sbq_w4_packed_bytes(int64_t N, int64_t K);
int64_t sbq_w4_scale_count(int64_t N, int64_t K, int group);
int sbq_repack_w4(const int8_t* q, int64_t N, int64_t K, int64_t ldq, const void* scale, int group,
                  uint8_t* packed, void* gscale, void* stream);
/* The inverse. */
int sbq_unpack_w4(const uint8_t* packed, const void* gscale, int64_t N, int64_t K, int group,
                  int8_t* q, int64_t ldq, void* scale, void* stream);

/* y[m,n] = sum_G fp32(scale[n,G]) * (sum_{k in G} q[n,k] * x[m,k]) (+ bias[n])
 * x: device [M, K] (row stride ldx), F32, F16 or BF16, any alignment
 * (16-byte aligned rows are faster).  fp16 and bf16 are used exactly, fp32 to
 * 22 significant bits (of each value, or 2^-39 of the largest in its 128
 * columns).  Accumulation is fp32.  bias: device fp32 [N] or NULL.  y: device
 * [M, N] (row stride ldy), F32, F16 or BF16.  Meant for M up to 64; more rows
 * run in blocks of 64 that each read the weight again. */
int sbq_linear_w4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx,
                  const uint8_t* packed, const void* gscale, const float* bias, int64_t N, int group,
                  void* y, int y_dtype, int64_t ldy, void* stream);

/* ---- attention over a cache and a tree of drafted tokens ----------------- */

/* Most query tokens of one sbq_tree_attention call. */
#define SBQ_ATTN_MAX_T 1024

/* The attention of model.py:208-229 for T query tokens over a cache whose
 * slots carry their positions, and over the keys of the T tokens themselves
 * where they are given (drafts that are not in the cache: a tree of drafted
 * tokens, verified in one pass):
 *   out[t,h] = sum_s p[t,h,s] v[s, h / (heads / kv_heads)],
 *   p[t,h,:] = softmax of scale * q[t,h] . k[s, ...] over what t sees:
 *   cached slot s iff 0 <= slot_pos[s] <= q_pos[t], and with a window
 *     (window > 0) slot_pos[s] > q_pos[t] - window;
 *   draft j (k_new[j], v_new[j], at position q_pos[j]) iff tree[t * tree_ld +
 *     j] != 0 (tree NULL: iff j <= t), and with a window q_pos[j] > q_pos[t] -
 *     window.
 * A row that sees nothing (or only scores of -infinity) is 0.  What a row does
 * not see does not reach it, infinities and NaN included.
 * q: device [T, heads, D], strides q_st and q_sh in elements, unit stride in
 * D; F32, or the cache's type.  k, v: device [slots, kv_heads, D], both with
 * strides k_ss and k_sh; k_new, v_new (NULL: none): device [T, kv_heads, D]
 * of the cache's type, both with strides n_ss and n_sh.  slot_pos: device
 * int64 [slots].  q_pos: device int64 [T].  out: device [T, heads, D] of q's
 * type, no two elements in one place, apart from every input.  1 <= D <= 256, heads a multiple of kv_heads, T <= SBQ_ATTN_MAX_T,
 * slots <= 2^30.
 * Scores, maxima and sums are fp32; with 2-byte queries the weights p are
 * rounded to their type (half to even; in fp16 at half a step of each down to
 * 2^-28 of the largest) for the product with v, with F32 queries everything is
 * fp32.  scale * q . k is to stay below 2^27 in magnitude, or be infinite.  Unit strides and 16-byte aligned rows of a
 * D of 64, 128 or 256 are the fastest.
 * weight: NULL, or device fp32 [slots]: weight[s] += sum_{t,h} p[t,h,s], the
 * attention weight the cached slots received (for eviction by it); calls
 * that add to one array must not overlap in time.
 * workspace: >= sbq_attn_workspace_bytes bytes, any content; one call at a
 * time.  The result does not depend on timing. */
int64_t sbq_attn_workspace_bytes(int64_t T, int64_t heads, int64_t kv_heads, int64_t D, int64_t slots,
                                 int weight);
int sbq_tree_attention(const void* q, int q_dtype, int64_t T, int64_t heads, int64_t D, int64_t q_st,
                       int64_t q_sh, const void* k, const void* v, int kv_dtype, int64_t slots,
                       int64_t kv_heads, int64_t k_ss, int64_t k_sh, const int64_t* slot_pos,
                       const int64_t* q_pos, const void* k_new, const void* v_new, int64_t n_ss,
                       int64_t n_sh, const uint8_t* tree, int64_t tree_ld, int64_t window, float scale,
                       void* out, int64_t o_st, int64_t o_sh, float* weight, void* workspace,
                       size_t workspace_bytes, void* stream);

/* ---- a bounded cache, evicted by attention weight ------------------------ */

/* A cache of `slots` slots that holds more positions than it has room for: it
 * gives up the slots that received the least attention weight (weight [slots],
 * the running sums sbq_tree_attention adds to).  Slots are given up in this
 * order, equal ones by their index: free slots (slot_pos < 0); then by
 * weight, the least first (-0 equals 0, NaN last); last the slots of the `recent` newest
 * positions.  No counterpart in the reference.
 *
 * sbq_kv_append: T new tokens, at positions *start .. *start + T - 1, take the
 * first T slots of that order, in ascending slot order (the newest positions
 * are those >= *start + T - recent): their keys and values (k_new, v_new:
 * device [T, kv_heads, D], strides n_ss and n_sh, F32, F16 or BF16) are
 * rounded to the cache's type and written to k, v (device [slots, kv_heads,
 * D], strides k_ss and k_sh), slot_pos is set, weight is 0, and *end = *start
 * + T.  start, end: device int64[1], the same one or not.  0 <= recent <=
 * slots, T <= slots.  k_new and v_new must not overlap the cache.  Slots that
 * hold positions from *start on already are not replaced: where tokens are taken
 * back, free their slots (slot_pos -1) first.
 *
 * sbq_kv_take: the used slots among the last `capacity` of that order (newest:
 * >= *end - recent) of a cache of any size are copied, in slot order, to the
 * first slots of another (strides t_ss and t_sh) with their positions and
 * weights; its other slots become free (slot_pos -1, weight 0; k and v left
 * as they were), *to_end = *end.  The two must not overlap.
 *
 * workspace: >= sbq_kv_workspace_bytes(slots, T or capacity), any content; one
 * call at a time. */
int64_t sbq_kv_workspace_bytes(int64_t slots, int64_t count);
int sbq_kv_append(int64_t* slot_pos, float* weight, int64_t slots, int64_t* end, const int64_t* start,
                  int64_t recent, void* k, void* v, int kv_dtype, int64_t kv_heads, int64_t D,
                  int64_t k_ss, int64_t k_sh, const void* k_new, const void* v_new, int new_dtype,
                  int64_t T, int64_t n_ss, int64_t n_sh, void* workspace, size_t workspace_bytes,
                  void* stream);
int sbq_kv_take(const int64_t* slot_pos, const float* weight, int64_t slots, const int64_t* end,
                const void* k, const void* v, int kv_dtype, int64_t kv_heads, int64_t D, int64_t k_ss,
                int64_t k_sh, int64_t capacity, int64_t recent, int64_t* to_pos, float* to_weight,
                int64_t* to_end, void* to_k, void* to_v, int64_t t_ss, int64_t t_sh, void* workspace,
                size_t workspace_bytes, void* stream);

/* ---- head norms and rotation to the positions --------------------------- */

/* model.py:260-270: the RMS norm of each head's queries and keys and their
 * rotation, in one pass.  For every vector x of D columns:
 *   y = x / sqrt(mean(x^2) + eps) * w          (w NULL: y = x)
 *   (y[a], y[b]) <- (y[a] cos - y[b] sin, y[b] cos + y[a] sin) for each pair
 *     i < pairs, at the angle position * inv_freq[i]: a = i, b = i + pairs, or
 *     with `interleaved` a = 2i, b = 2i + 1; columns from 2 * pairs on stay.
 * The angle is exact (a 64-bit product, reduced in 64 bits), everything else
 * fp32, rounded once to the output's type.
 * q: device [tokens, heads, D], k: device [tokens, kv_heads, D] (kv_heads 0:
 * none) of one type, strides in elements, unit stride in D <= 256.
 * positions: device int64, below 2^53 (and so their angles); token t stands at
 * positions[t / per] + t % per.
 * inv_freq: device fp32 [pairs].  q_weight, k_weight: device [D] of
 * weight_dtype, or NULL.  q_out, k_out: device, of q's type, the input itself
 * (with its strides) or apart from both inputs. */
int sbq_qk_norm_rope(const void* q, const void* k, int dtype, int64_t tokens, int64_t heads,
                     int64_t kv_heads, int64_t D, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh,
                     const int64_t* positions, int64_t per, const float* inv_freq, int64_t pairs,
                     int interleaved, const void* q_weight, const void* k_weight, int weight_dtype,
                     float eps, void* q_out, void* k_out, int64_t qo_st, int64_t qo_sh, int64_t ko_st,
                     int64_t ko_sh, void* stream);

/* ---- a paged cache of several sequences ---------------------------------- */

/* Cache types beside SBQ_F32, SBQ_F16 and SBQ_BF16: 8-bit codes with a scale. */
#define SBQ_I8 3
#define SBQ_E4M3 4
/* Most query tokens of a sequence in one sbq_paged_attention call. */
#define SBQ_PAGED_MAX_T 1024

/* A pool of pages that the sequences' positions are spread over.  No
 * counterpart in the reference, whose engine holds one sequence.
 * k, v: device [pages][kv_heads][page][row], row = D rounded up to a multiple
 * of 16, columns from D on zero; page a power of two from 16 to 1024.
 * k_scale, v_scale: device fp32 [pages][kv_heads][page] for SBQ_I8 and
 * SBQ_E4M3 (else not looked at): a vector is its codes times its scale.
 * table: device int32 [sequences][max_pages]: position p of sequence b stands
 * in page table[b][p / page], row p % page; an entry outside 0 .. pages - 1
 * is no page: what stands there is neither written nor seen.  Pages that two
 * sequences write to must differ.  length: device int64 [sequences]: positions
 * held.  max_pages * page <= 2^30, sequences <= 65536, T (count) * kv_heads <=
 * 2^30.  k, v and the scales are 16-byte aligned, E4M3 codes finite.
 *
 * sbq_paged_append: T new tokens of each sequence (k_new, v_new: device
 * [sequences, T, kv_heads, D], both with strides n_sb, n_st, n_sh, F32, F16 or
 * BF16, apart from the pool), of which the first counts[b] (NULL: all; device int64, limited to 0 ..
 * T) are there, go to the positions start[b] on (device int64; may be `length`
 * itself, not a part of it elsewhere); length[b] = start[b] + counts[b], at
 * most max_pages * page (a token past that is dropped; a start below 0 stores
 * nothing and leaves length 0).  8-bit caches:
 *   scale = max |x| / 127 (I8) or / 448 (E4M3), code = the nearest to x / scale
 * (fp32 IEEE divisions, half to even; a scale of 0: codes 0).  A vector with
 * an infinity or NaN reads back as NaN (scale NaN, codes 0).
 *
 * sbq_paged_read: positions start[b] .. start[b] + count - 1 of each sequence,
 * to k_out, v_out (device [sequences, count, kv_heads, D], strides o_sb, o_st,
 * o_sh in any order of the axes, no two elements in one place, rounded to out_dtype);
 * positions that it does not hold are 0. */
int sbq_paged_append(void* k, void* v, float* k_scale, float* v_scale, int cache_dtype, int64_t pages,
                     int64_t page, int64_t kv_heads, int64_t D, const int32_t* table, int64_t sequences,
                     int64_t max_pages, int64_t* length, const int64_t* start, const int64_t* counts,
                     const void* k_new, const void* v_new, int new_dtype, int64_t T, int64_t n_sb,
                     int64_t n_st, int64_t n_sh, void* stream);
int sbq_paged_read(const void* k, const void* v, const float* k_scale, const float* v_scale,
                   int cache_dtype, int64_t pages, int64_t page, int64_t kv_heads, int64_t D,
                   const int32_t* table, int64_t sequences, int64_t max_pages, const int64_t* length,
                   const int64_t* start, int64_t count, void* k_out, void* v_out, int out_dtype,
                   int64_t o_sb, int64_t o_st, int64_t o_sh, void* stream);

/* The attention of T tokens of each sequence over its pages:
 *   out[b,t,h] = sum_p softmax_p(scale * q[b,t,h] . k[b,p]) v[b,p], key head
 *   h / (heads / kv_heads),
 * over the positions p < length[b] that token t sees: p <= start[b] + t, and
 * with a window (> 0) p > start[b] + t - window.  start NULL: length[b] -
 * counts[b], the tokens appended last.  Tokens from counts[b] (NULL: T) on
 * see nothing.  A row that sees nothing is 0.
 * What a row does not see does not reach it, infinities and NaN included.
 * q: device [sequences, T, heads, D], T <= SBQ_PAGED_MAX_T, F32, or the
 * cache's type (8-bit caches: any); out: the same shape and type, its axes in any
 * order, no two elements in one place, apart from every input.
 * Scores, maxima and sums are fp32.  The other factors are multiplied as they are,
 * or where the cache's type has fewer bits in pieces of it (8 bits: of fp16): BF16
 * caches 24 bits of fp32 queries and their weights, 16 of the weights of BF16
 * queries; F16 and 8-bit caches each element of an fp32 query, and each weight (8
 * bits: times its value's scale), to 2^-22 of itself or 2^-39 of the row's largest,
 * whichever is more (F16, scores from 2^23 on: weights 2^-25 of the largest).
 * scale * q . k is to be finite, below 2^27 in magnitude, |v| below 2^127; over F32
 * and BF16 caches results keep their bits down to 2^-126 times the positions that a
 * row sees.
 * workspace: >= sbq_paged_attn_workspace_bytes bytes (0: NULL will do), any
 * content; one call at a time.  The result does not depend on timing; how a
 * long sequence is split, and so its last bits, goes by all sequences' lengths. */
int64_t sbq_paged_attn_workspace_bytes(int64_t sequences, int64_t T, int64_t heads, int64_t kv_heads,
                                       int64_t D, int64_t page, int64_t max_pages, int64_t window,
                                       int cache_dtype);
int sbq_paged_attention(const void* q, int q_dtype, int64_t T, int64_t heads, int64_t q_sb, int64_t q_st,
                        int64_t q_sh, const void* k, const void* v, const float* k_scale,
                        const float* v_scale, int cache_dtype, int64_t pages, int64_t page,
                        int64_t kv_heads, int64_t D, const int32_t* table, int64_t sequences,
                        int64_t max_pages, const int64_t* length, const int64_t* start,
                        const int64_t* counts, int64_t window, float scale, void* out, int64_t o_sb,
                        int64_t o_st, int64_t o_sh, void* workspace, size_t workspace_bytes,
                        void* stream);

/* ---- drafted tokens against the target's probabilities ------------------- */

/* B sequences with T drafted tokens each (counts[b] of them where counts,
 * device int64 [B], is given; limited to 0 .. T).  p: the target's
 * probabilities, device [B, T + 1, V] (row t: after the drafts before t), q:
 * those that the drafts were drawn from, device [B, T, V], or NULL (each draft
 * was certain); strides p_sb, p_st, q_sb, q_st in elements, unit stride in V
 * <= 2^23, both F32, F16 or BF16, none negative; a row need not sum to 1.
 * tokens: device int64 [B, T].  u: device fp32 [B, T + 1] uniforms in [0, 1).
 *   kept[b]: the drafts before the first t with not u[b,t] q[x] < p[x];
 *   token[b]: the first index (vocabulary order) whose prefix of mass exceeds
 *     u[b,T] * (whole mass), the mass being max(p - q, 0) of the refused
 *     draft's rows (p's own where nothing is left), or p's row counts[b].
 * Products and sums are 64-bit.  A draft outside 0 .. V - 1 is refused.  token
 * is -1 where the whole mass is 0, infinite or NaN.  B, T <= 65535.
 * kept, token: device int64 [B].  workspace: >= sbq_verify_workspace_bytes bytes
 * (0: NULL will do), any content; one call at a time.  All three lie apart from
 * each other and from the inputs, first byte to last (SBQ_ERR_ARG). */
int64_t sbq_verify_workspace_bytes(int64_t B, int64_t V);
int sbq_verify_drafts(const void* p, int64_t p_sb, int64_t p_st, const void* q, int64_t q_sb, int64_t q_st,
                      int dtype, int64_t B, int64_t T, int64_t V, const int64_t* tokens, const float* u,
                      const int64_t* counts, int64_t* kept, int64_t* token, void* workspace,
                      size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SBQ_H_ */
