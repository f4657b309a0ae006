/*
 * b200_whisper.h - C ABI of the sm_100a kernels behind the ggml backend plugin (libggml-b200.so).
 *
 * Two libraries:
 *   libb200_kernels.so  exports every b200_* function below (plain pointers and sizes, no ggml types).
 *   libggml-b200.so     exports ggml_backend_init / ggml_backend_score, the entry points that ggml's
 *                       dynamic loader binds (ggml/src/ggml-backend-impl.h:215-218, looked up by
 *                       ggml/src/ggml-backend-reg.cpp:236-253).  Its graph_compute maps every node of a
 *                       whisper graph onto the functions declared here.
 *
 * Every function returns 0 on success or a cudaError_t value (B200_ERR_* for argument errors).  Device
 * pointers are plain CUDA device pointers on the current device.  `stream` is a cudaStream_t passed
 * as void* (NULL = legacy default stream).  Nothing here synchronises the stream.
 *
 * Arithmetic contract: each kernel reproduces the operation order of the AVX2/FMA/F16C build of the
 * reference CPU backend (lane-wise partial sums, FMA placement, F16 round trips), so results are
 * expected to be bit-identical to it, not merely close.
 */
#ifndef B200_WHISPER_H
#define B200_WHISPER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200_ERR_ARG      10001   /* unsupported shape / type / alignment */
#define B200_ERR_NO_DEVICE 10002  /* no CUDA device: the library never falls back to the CPU */

/* ggml type ids used at this boundary (ggml/include/ggml.h:354-387) */
#define B200_TYPE_F32  0
#define B200_TYPE_F16  1
#define B200_TYPE_Q5_0 6
#define B200_TYPE_Q8_0 8
#define B200_TYPE_I32  26
#define B200_TYPE_BF16 30

/* ---- block formats ---------------------------------------------------------------------------
 * ggml stores 32 weights per block: block_q5_0 = {f16 d; u8 qh[4]; u8 qs[16]} (22 B),
 * block_q8_0 = {f16 d; i8 qs[32]} (34 B)  (ggml/src/ggml-common.h:187-214).  Neither size allows
 * aligned vector loads, so device memory holds the same bytes as three (two) planes of one tensor:
 *   Q5_0: qs[nb][16] | qh[nb] (u32) | d[nb] (f16)         Q8_0: qs[nb][32] | d[nb] (f16)
 * Total size is unchanged (22*nb / 34*nb bytes).  These run on the host and allocate nothing. */
int b200_blocks_to_planes(int type, const void * blocks, void * planes, int64_t nb_total,
                          int64_t nb_first, int64_t nb_count);   /* replaces nothing: layout helper */
int b200_planes_to_blocks(int type, const void * planes, void * blocks, int64_t nb_total,
                          int64_t nb_first, int64_t nb_count);
/* The same conversions on the device: `blocks_dev` holds nb_count raw ggml blocks (as read from a model file,
 * src/whisper.cpp:1874-1960, or produced by the quantize tool), `planes_dev` is the whole tensor's plane storage.
 * The plugin's set_tensor / get_tensor use them: one upload of the file's bytes plus one launch per weight tensor. */
int b200_blocks_to_planes_device(int type, const void * blocks_dev, void * planes_dev, int64_t nb_total, int64_t nb_first,
                                 int64_t nb_count, void * stream);
int b200_planes_to_blocks_device(int type, const void * planes_dev, void * blocks_dev, int64_t nb_total, int64_t nb_first,
                                 int64_t nb_count, void * stream);

/* dequantize_row_q5_0 / dequantize_row_q8_0 (ggml/src/ggml-quants.c:296-320, 349-362) on planes. */
int b200_dequantize(int type, const void * planes, int64_t nb_total, int64_t nb_first, int64_t nb_count,
                    float * out, void * stream);

/* quantize_row_q8_0, AVX2 variant (ggml/src/ggml-cpu/ggml-cpu-quants.c:808-866): rows of f32 ->
 * int8 qs[n_rows][k] and the f16-rounded scale widened to f32, d[n_rows][k/32]. */
int b200_quantize_q8_0(const float * x, int64_t n_rows, int64_t k, int64_t row_stride_bytes,
                       int8_t * qs, float * d, void * stream);

/* ggml_compute_forward_mul_mat for Q5_0 / Q8_0 weights (ggml/src/ggml-cpu/ggml-cpu.c:1266-1458 with
 * ggml_vec_dot_q5_0_q8_0 / ggml_vec_dot_q8_0_q8_0, ggml-cpu-quants.c:3076-3100, 3869-3886):
 * dst[n*dst_stride + m] = sum_k W[m][k] * X[n][k], activations already quantised by
 * b200_quantize_q8_0.  w_planes covers the WHOLE weight tensor (nb_total blocks). */
int b200_mul_mat_q(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                   const int8_t * xq, const float * xd, int64_t N,
                   float * dst, int64_t dst_stride, void * stream);

/* Same contract for 1..8 activation columns given as f32 (row stride in bytes): quantisation of the
 * activations is fused, no scratch is needed.  The batch-1 / beam decode path. */
int b200_mul_mat_vec_q(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                       const float * x, int64_t x_stride_bytes, int64_t N,
                       float * dst, int64_t dst_stride, void * stream);

/* Fused form of the above for the decode step: the product value passes through up to four steps, in the
 * order given, before it is stored - the ADD / SCALE / UNARY(GELU) / CPY nodes that follow a MUL_MAT node in
 * the whisper decoder graph (src/whisper.cpp:2533-2830), evaluated with the same single-precision
 * operations, so the stored bits equal those of the unfused node sequence.
 *   B200_EP_ADD   v = v + ptr[m + n*stride_n]   (stride_n = 0: bias broadcast over columns)
 *   B200_EP_SCALE v = v * scalar
 *   B200_EP_GELU  v = gelu_table(v)
 * store_f16 != 0 stores round-to-nearest-even f16 (the F32->F16 CPY into the KV cache) instead of f32. */
#define B200_EP_ADD   1
#define B200_EP_SCALE 2
#define B200_EP_GELU  3
typedef struct { int kind; const float * ptr; int64_t stride_n; float scalar; } b200_ep_step;
typedef struct { int n_steps; b200_ep_step step[4]; int store_f16; } b200_epilogue;
int b200_mul_mat_vec_q_ep(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                          const float * x, int64_t x_stride_bytes, int64_t N,
                          void * dst, int64_t dst_stride, const b200_epilogue * ep, void * stream);

/* b200_mul_mat_q with the same epilogue steps applied to every product value (encoder and prompt path). */
int b200_mul_mat_q_ep(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                      const int8_t * xq, const float * xd, int64_t N,
                      void * dst, int64_t dst_stride, const b200_epilogue * ep, void * stream);

/* The same kernel with every column described on its own: column n reads x (K floats, 16-byte aligned), writes
 * dst (M f32, or M f16 when store_f16) and adds add[s] (M floats) at epilogue step s when kind[s] == B200_EP_ADD.
 * This is how single-token decode steps of several whisper_states that run in lock-step share one pass over
 * the weights (up to 8 columns per launch).  No counterpart in the reference, which decodes state by state. */
typedef struct { const float * x; void * dst; const float * add[4]; } b200_gemv_col;
typedef struct { int n_steps; int kind[4]; float scalar[4]; int store_f16; } b200_gemv_ep;
int b200_mul_mat_vec_q_cols(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                            const b200_gemv_col * cols, int n_cols, const b200_gemv_ep * ep, void * stream);

/* Up to 32 columns per launch, quantised beforehand: b200_quantize_cols gathers columns that live at unrelated
 * addresses (K floats each) into xq[n_cols][K] / xd[n_cols][K/32]; b200_mul_mat_cols_q multiplies them with the
 * weights (cols[n].x is ignored, dst/add as above).  A CTA keeps a few weight rows in shared memory for all
 * columns, so the weights are read once for the whole group.  No counterpart in the reference. */
int b200_quantize_cols(const float * const * x_cols, int n_cols, int64_t K, int8_t * xq, float * xd, void * stream);
int b200_mul_mat_cols_q(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                        const int8_t * xq, const float * xd, const b200_gemv_col * cols, int n_cols,
                        const b200_gemv_ep * ep, void * stream);

/* Up to three b200_mul_mat_cols_q products on the SAME quantised columns in one launch (the Q, K and V projections of
 * a decoder layer): job i has its own weights (w_planes[i], nb_total[i], M[i] rows; all jobs share K and the type), its own
 * outputs cols[i][0..n_cols) and its own epilogue ep[i] (ep or ep[i] may be NULL).  No counterpart in the reference. */
int b200_mul_mat_cols_q_multi(int wtype, int n_jobs, const void * const * w_planes, const int64_t * nb_total, const int64_t * M,
                              int64_t K, const int8_t * xq, const float * xd, const b200_gemv_col * const * cols, int n_cols,
                              const b200_gemv_ep * const * ep, void * stream);

/* The same product (ggml_compute_forward_mul_mat with ggml_vec_dot_q5_0_q8_0 / ggml_vec_dot_q8_0_q8_0, same bits)
 * for many columns on the tensor pipe.  The integer lane sums of the AVX2 dot product are exact in an f16 MMA with
 * f32 accumulation, the per-block float chain is replayed as in b200_mul_mat_q.  Operands are repacked once:
 *   b200_mma_pack_weights: planes -> h[nb_total][16] u32 (the block's 32 integers as f16 pairs, pair 4r+t stored at
 *                          position 4t+r) and d[nb_total] f32; 68 bytes per block, both 16-byte aligned.  No
 *                          counterpart in the reference (layout helper, done once per weight tensor).
 *   b200_mma_quantize:     quantize_row_q8_0 (ggml-cpu-quants.c:808-866) writing the same integers in that format.
 *   b200_mul_mat_mma_ep:   dst[n*dst_stride + m] with the epilogue steps of b200_mul_mat_q_ep; K % 128 == 0. */
int b200_mma_pack_weights(int wtype, const void * w_planes, int64_t nb_total, void * h, float * d, void * stream);
int b200_mma_quantize(const float * x, int64_t n_rows, int64_t k, int64_t row_stride_bytes, void * h, float * d, void * stream);
int b200_mul_mat_mma_ep(const void * wh, const float * wd, int64_t M, int64_t K,
                        const void * xh, const float * xd, int64_t N,
                        void * dst, int64_t dst_stride, const b200_epilogue * ep, void * stream);

/* The same product once more (ggml_compute_forward_mul_mat, ggml/src/ggml-cpu/ggml-cpu.c:1266-1458, with
 * ggml_vec_dot_q5_0_q8_0 / ggml_vec_dot_q8_0_q8_0, ggml-cpu-quants.c:3076-3100, 3869-3886; same bits) on the
 * fifth-generation tensor cores: tcgen05.mma with a fresh tensor-memory accumulator per 32-block gives the eight
 * exact integer lane sums of every (row, column, block), epilogue warps drain tensor memory into the reference's
 * float chain.  Arguments as b200_mul_mat_q_ep: weights as planes (no repacked copy is needed, Q5_0 is unpacked in
 * the shared-memory stage), activations quantised by b200_quantize_q8_0.  Any M, N >= 1, K % 32 == 0.
 * b200_mul_mat_tc_status: 0, or the code of a device-side wait that ran out in an earlier launch (the launch then
 * returned without finishing its tiles); synchronises with the device. */
int b200_mul_mat_tc_ep(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                       const int8_t * xq, const float * xd, int64_t N,
                       void * dst, int64_t dst_stride, const b200_epilogue * ep, void * stream);
int b200_mul_mat_tc_status(void);
/* The same with every column described on its own (cols[n].dst / cols[n].add as in b200_mul_mat_cols_q, cols[n].x is
 * ignored; at most 64 columns): single-token decode steps of many whisper_states in one pass over the weights.  No
 * counterpart in the reference, which decodes state by state. */
int b200_mul_mat_tc_cols(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                         const int8_t * xq, const float * xd, const b200_gemv_col * cols, int n_cols,
                         const b200_gemv_ep * ep, void * stream);

/* NORM -> MUL(gamma) -> ADD(beta) in one pass (ops.cpp:3109-3158 followed by binary-ops.cpp:50-137), each of the
 * three roundings kept: y = ((x - mean) * rstd) * gamma + beta. */
int b200_layer_norm(const float * x, const float * gamma, const float * beta, float * y, int64_t ne00, int64_t nrows,
                    int64_t x_row_stride_bytes, int64_t y_row_stride_bytes, float eps, void * stream);

/* No counterpart in the reference.  b200_mul_mat_q needs the activations quantised into scratch memory that
 * the caller allocates.  Some callers cannot allocate device memory at the point where they need a product:
 * code that runs inside another framework's memory plan (all device memory handed out up front), hosts that
 * forbid the implicit device-wide synchronisation of cudaMalloc/cudaFree on a latency-critical path, or a
 * plugin callback that is only given input and output pointers.  For them this entry point does the same
 * work - quantise N rows of f32 activations (row stride in bytes), then the Q5_0/Q8_0 product - with the
 * scratch held in a fixed device array that is part of this library's image (b200_static_scratch_bytes()
 * bytes, resident on every GPU that loads the library until the process exits).  It calls no allocator.
 *  - N*K + 4*N*K/32 bytes (plus padding to 256) must fit; otherwise B200_ERR_TOO_LARGE is returned.  All
 *    arguments (NULL pointers, alignment, strides, weight extent) are checked first: an error return means nothing
 *    was launched.
 *  - The first call on each device looks up the array's device address (with that device current); make that
 *    first call outside any stream capture.
 *  - All calls share the one array and it keeps the previous call's contents.  Every byte a call reads is
 *    written by that same call first, so nothing needs clearing, but two calls that may overlap on the GPU
 *    (different streams, no ordering between them) race on it. */
#define B200_ERR_TOO_LARGE 10003
int64_t b200_static_scratch_bytes(void);
int b200_mul_mat_q_static(int wtype, const void * w_planes, int64_t nb_total, int64_t M, int64_t K,
                          const float * x, int64_t x_stride_bytes, int64_t N,
                          float * dst, int64_t dst_stride, void * stream);

/* mul_mat with F16 src0 (ggml_vec_dot_f16, ggml/src/ggml-cpu/vec.cpp:128-167): src1 is f32 (rounded
 * to f16 first, ggml-cpu.c:1329-1362) or f16.  Strides in bytes; src0 [K, M, ne02, ne03],
 * src1 [K, N, ne12, ne13] with ne12 % ne02 == 0, dst f32 contiguous [M, N, ne12, ne13]. */
int b200_mul_mat_f16(const void * src0, const int64_t * ne0, const int64_t * nb0,
                     const void * src1, int src1_type, const int64_t * ne1, const int64_t * nb1,
                     float * dst, const int64_t * nbd, void * stream);

/* ggml_compute_forward_flash_attn_ext_f16 (ggml/src/ggml-cpu/ops.cpp:6638-6851) for head size 64,
 * F16 K/V, optional F16 mask; the running F16 accumulator and its rounding order are kept.
 * q f32 [64, n_q, n_head] (strides nbq1, nbq2 bytes), k/v f16 [64, n_kv, n_head], mask f16
 * [n_kv, >=n_q] or NULL, dst f32 [64, n_head, n_q] contiguous. */
int b200_flash_attn_ext(const float * q, int64_t nbq1, int64_t nbq2,
                        const void * k, int64_t nbk1, int64_t nbk2,
                        const void * v, int64_t nbv1, int64_t nbv2,
                        const void * mask, int64_t nbm1,
                        float * dst, int64_t n_q, int64_t n_kv, int64_t n_head, float scale, void * stream);

/* The decode-shaped form of the above, one entry per query row (at most 32): each row has its own query, K/V
 * views, mask row, output and key count, so rows of different whisper_states (different KV caches, different
 * lengths) go out in one launch.  dst receives [n_head][64] f32 per row.  No counterpart in the reference. */
typedef struct { const float * q; const void * k; const void * v; const void * mask; float * dst; int64_t n_kv; } b200_fa_row;
int b200_flash_attn_decode_rows(const b200_fa_row * rows, int n_rows, int64_t n_head, int64_t nbq2, int64_t nbk1, int64_t nbk2,
                                int64_t nbv1, int64_t nbv2, float scale, void * stream);
/* The same, and additionally every output row quantised as b200_quantize_cols would do it afterwards (row i ->
 * xq[i][n_head*64], xd[i][n_head*2]): saves the separate quantisation launch before the output projection. */
int b200_flash_attn_decode_rows_q(const b200_fa_row * rows, int n_rows, int64_t n_head, int64_t nbq2, int64_t nbk1, int64_t nbk2,
                                  int64_t nbv1, int64_t nbv2, float scale, int8_t * xq, float * xd, void * stream);

/* ggml_compute_forward_norm_f32 (ops.cpp:3109-3158): rows of ne00 f32, row strides in bytes. */
int b200_norm(const float * x, float * y, int64_t ne00, int64_t ne01, int64_t ne02, int64_t ne03,
              const int64_t * nbx, const int64_t * nby, float eps, void * stream);

/* b200_layer_norm for rows that live at unrelated addresses (at most 64; rows of several decoder states). */
typedef struct { const float * x; float * y; } b200_ln_row;
int b200_layer_norm_rows(const b200_ln_row * rows, int n_rows, const float * gamma, const float * beta, int64_t ne00, float eps, void * stream);
/* The same, and additionally every output row quantised as b200_quantize_cols would do it afterwards (row i ->
 * xq[i][ne00], xd[i][ne00/32]; ne00 a multiple of 32): saves the separate quantisation launch before the products that
 * consume the rows.  No counterpart in the reference beyond quantize_row_q8_0 itself. */
int b200_layer_norm_rows_q(const b200_ln_row * rows, int n_rows, const float * gamma, const float * beta, int64_t ne00, float eps,
                           int8_t * xq, float * xd, void * stream);

/* ADD (op 0) / MUL (op 1) with ggml broadcasting of src1 (ggml/src/ggml-cpu/binary-ops.cpp:50-137). */
int b200_binary(int op, const float * a, const int64_t * nea, const int64_t * nba,
                const float * b, const int64_t * neb, const int64_t * nbb,
                float * dst, const int64_t * nbd, void * stream);

/* SCALE (ops.cpp:3840) and GELU via the F16 lookup table (vec.h:443-457) on contiguous f32. */
int b200_scale(const float * x, float * y, int64_t n, float s, void * stream);
int b200_gelu(const float * x, float * y, int64_t n, void * stream);

/* CPY / DUP / CONT (ops.cpp:26-1183): f32->f32, f32->f16, f16->f16, f16->f32, any strides,
 * same element count, element order = row-major over ne. */
int b200_cpy(const void * src, int src_type, const int64_t * nes, const int64_t * nbs,
             void * dst, int dst_type, const int64_t * ned, const int64_t * nbd, void * stream);

/* GET_ROWS (ops.cpp:4146-4313): rows selected by i32 ids from a Q5_0/Q8_0 (planes), F16 or F32
 * table [ne00, n_table_rows] -> f32 [ne00, n_ids] contiguous. */
int b200_get_rows(int type, const void * table, int64_t nb_total_or_row_stride, int64_t ne00,
                  const int32_t * ids, int64_t n_ids, float * dst, void * stream);

/* Side output for the host sampler (whisper_process_logits / whisper_sample_token / whisper_sample_token_topk,
 * src/whisper.cpp:5015-5430, which scan a full row of n_vocab logits per decoder and step): per row of n values the k
 * largest with their indices (ties: lower index first, as the reference's forward scan with `>` resolves them), the
 * maximum and log(sum(exp(x - max))) + max.  rows[i] / out[i] are device pointers, at most 64 rows per call. */
#define B200_TOPK_MAX 8
typedef struct { int32_t n, k; float max, logsumexp; int32_t ids[B200_TOPK_MAX]; float vals[B200_TOPK_MAX]; } b200_topk_result;
int b200_topk_rows(const float * const * rows, b200_topk_result * const * out, int n_rows, int64_t n, int k, void * stream);

/* ---- beam search on the device, on a paged key/value cache ------------------------------------------------------
 * whisper's beam search samples, sorts and copies caches on the host (whisper_sample_token_topk, whisper_full_with_state,
 * src/whisper.cpp:5230-5430, 5880-6010: one decoder per beam, whisper_kv_cache_seq_cp for the caches).  The entry points
 * below do the same work next to the logits.  They are defined by their formulas, not by a reference kernel: sums, softmax
 * statistics and scores are held in 32 bits or more, and every result is independent of the order in which blocks run.
 * None of them allocates, synchronises or keeps anything between calls; all may be captured into a graph.  Scratch memory
 * comes from the caller (16-byte aligned); two calls that may overlap on the device need a scratch area each.  How much a call
 * needs depends on how its work is dealt out: a smaller call can need more than a larger one, so ask for every size that is used
 * (b200_paged_attn: an area of 21 MB serves every call). */

/* The next beams of every sequence.  Row r = sequence * n_beam + beam has n_vocab logits x (F32, F16 or BF16; nb_row bytes
 * between rows) and an accumulated score.  Candidates are
 *   of a live beam b   every token v that is not banned:  score[b] + x[v] - max(x) - log(sum(exp(x - max(x))))
 *   of a done beam b   the one token eos, with score[b]
 * and the n_beam best become the new beams, best first, ties towards the lower b * n_vocab + v.  Banned tokens (bit v of word
 * v / 32; banned_stride words between the rows' masks, 0 = one mask for all) and NaN count as -inf logits; where a row has logits of +inf,
 * they share it (-log of their number each) and its other tokens are none.  A candidate of
 * score -inf or NaN is none, and of a row whose score is that, or that is done, the logits do not matter; with a score of +inf a row's candidates are equal.
 * The new beam is done when its parent
 * was or its token is eos.  Where candidates run out: score -inf, token and parent -1, done 1
 * (b200_beam_reorder leaves such a beam as it is; for b200_pages_update, which counts rows over all sequences, it is row_parent = the row itself with
 * keep = n_new = 0, and never sequence * n_beam - 1, the row before the sequence).
 * score_out / done_out may be score / done.  n_beam <= B200_BEAM_MAX, n_beam * n_vocab < 2^31, n_beam * ceil(n_vocab / 8192) <= 32768, any
 * alignment of the rows that suits their type.  done, banned may be NULL.  Rules that weigh tokens against each other (whisper's timestamps against text)
 * are no mask: they change the logits before this call. */
#define B200_BEAM_MAX 32
typedef struct {
    const void * logits; int type; int64_t nb_row; int64_t n_vocab; int n_seq, n_beam;
    const float * score; const uint8_t * done; int32_t eos;
    const uint32_t * banned; int64_t banned_stride;
    float * score_out; int32_t * token_out; int32_t * parent_out; uint8_t * done_out;    /* [n_seq * n_beam] each */
    void * workspace; int64_t workspace_bytes;
} b200_beam_select_args;
int64_t b200_beam_select_workspace(int n_seq, int n_beam, int64_t n_vocab);
int b200_beam_select(const b200_beam_select_args * a, void * stream);

/* State that is kept per beam follows its parent, in place: for every outer index o of every block, the row_bytes bytes at
 * base + o * nb_outer + (sequence * n_beam + b) * nb_row become those of row parent[sequence * n_beam + b] of the same
 * sequence (any value outside 0..n_beam-1 leaves the row as it is).  Caches of all layers, token histories, any state with a
 * row per beam.  Any alignment (16-byte aligned base and strides are fastest); rows must not overlap; at most 8 blocks. */
typedef struct { void * base; int64_t n_outer, nb_outer, nb_row, row_bytes; } b200_beam_block;
int b200_beam_reorder(const b200_beam_block * blocks, int n_blocks, const int32_t * parent, int n_seq, int n_beam, void * stream);

/* A paged key/value cache.  The value of token t (0..page_size-1), head h, dimension i of page p in layer l lies at
 * base + l * nb_layer + p * nb_page + t * nb_tok + h * nb_head + 2 * i  (bytes; F16 or BF16; all strides and both bases
 * multiples of 16, so token-major and head-major pages are both possible).  head_dim is 64 or 128, page_size 1 .. 2^20, n_head_kv at most 1024,
 * a page less than 32 GB. */
typedef struct {
    void * k; void * v; int type, n_layer, n_pages, page_size, n_head_kv, head_dim;
    int64_t nb_layer, nb_page, nb_tok, nb_head;
} b200_page_pool;
/* Who uses the pages: row i (a sequence, or a beam of one) holds lens[i] tokens in pages tables[i * table_stride + 0 ..
 * ceil(lens[i] / page_size) - 1]; refs[p] counts the holders of page p over all rows (plus any holder of the caller's own),
 * 0 = free.  At most 8192 rows and 2^30 pages; table_stride * page_size < 2^31, table_stride * n_rows < 2^30. */
typedef struct { int32_t * tables; int32_t * lens; int32_t * refs; int64_t n_rows, table_stride; } b200_page_state;
int64_t b200_pages_workspace(int64_t n_rows, int64_t n_pages);

/* Row i becomes the first keep[i] tokens of row parent[i], with room for n_new[i] more - fork (parent != i), truncate
 * (keep < length), free (keep = n_new = 0), grow (n_new > 0), in any mix.  `from` is read, `to` (same n_rows and table_stride) is written;
 * neither its arrays nor status nor the workspace may overlap one another or an input (a program keeps two states and swaps them).  Whole pages are shared.  A partly filled last page that will be written
 * (n_new > 0) stays where it is for one row only: if nobody else holds it, or, among several such rows and no other holder, for
 * the first of them; the others get a new page with a copy of its keep[i] % page_size tokens, in every layer of the pool.  New
 * pages are those free in `from`, lowest number first, row by row (within a row: first the copy, then the following pages);
 * pages that become free here can be taken by the next call.  Table entries behind a row's last page are set to -1.
 * parent NULL: every row is its own parent.  pool NULL: tables only; b200_pages_copy then makes the copies, for as many
 * pools as the caller has (n_pages and page_size are needed, so they come with pool: pass k = v = NULL for tables only).
 * status[0] (device): 0; the number of pages that are missing; or -1 (a parent, keep, n_new or table entry out of range, or
 * a used entry on a free page: a row cannot keep more than its parent holds, nor grow beyond table_stride pages).  If it is not 0, `to` is a copy of `from` and
 * nothing else happened.  status[1]: pages copied. */
int b200_pages_update(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, const int32_t * parent,
                      const int32_t * keep, const int32_t * n_new, int32_t * status, void * workspace, int64_t workspace_bytes, void * stream);

/* With L pages in use, the i-th used page numbered L or more moves to the i-th free page below L.  `to` receives tables, lens
 * and refs in the new numbers, remap[p] the new number of page p (-1: free) for holders that the tables do not show.  What is written
 * must not overlap itself or `from`; the pages themselves move within the pool.  status as above ([0]: 0, or -1 for a table entry out of
 * range or on a free page; [1]: pages moved). */
int b200_pages_compact(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, int32_t * remap,
                       int32_t * status, void * workspace, int64_t workspace_bytes, void * stream);

/* Repeats the page copies of the last b200_pages_update / b200_pages_compact that used this workspace (same n_rows,
 * n_pages and page_size) in another pool: one pool per layer, or a draft model's cache beside the main one. */
int b200_pages_copy(const b200_page_pool * pool, int64_t n_rows, const void * workspace, int64_t workspace_bytes, void * stream);

/* Attention of a chunk of new tokens over the paged cache, one token per sequence included (the single-token step).
 * Sequence s has the query tokens q_start[s] .. q_start[s+1]-1 (n_new of them) and lens[s] tokens in its pages, the new ones
 * last: query t stands at position p = lens[s] - n_new + t and attends to positions 0..p (causal), or to all lens[s] (causal
 * = 0).  Query head h reads key/value head h / (n_head / n_head_kv).  q is F16 or BF16 like the pool, or F32; dst has q's type:
 *   dst[tok][h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q.k_j - m),   lse[tok][h] = m + log(sum_j w_j)   (lse may be NULL)
 * Scores and sums are 32-bit; for 16-bit q the weights w_j are rounded to the pool's type before the product with V, which
 * adds at most half a step of that type relative to each weight, the size of the output's own rounding (F16: for weights below 2^-25 of the
 * largest, at most 2^-36 of the largest instead), and the tensor pipe truncates its 32-bit sums instead of rounding them.  For F32 q the products take q
 * and the weights with the pool's type in two parts (F16: 22 bits, but no finer than 2^-36 of a row's largest |q| and 2^-50 of the largest weight) or
 * three (BF16: 24 bits), and their sums are rounded.  A query
 * without a key gives zeros and lse -inf; a NaN or infinite value in a position that a query does not attend to has no effect on it.
 * A NaN or infinite value in one that it does attend to leaves the dimensions that it enters infinite or NaN.
 * k_new / v_new (type of q, [n_tok][n_head_kv][head_dim] with strides nb_new_tok, nb_new_head) are first stored at their positions,
 * rounded to the pool's type; NULL (both) if the pages hold them already.  nb_* in bytes, multiples of 16, and 16-byte
 * aligned pointers.  max_new and max_len bound n_new and lens from above (device values beyond them, or beyond the tables, are cut
 * off, and the new tokens then replace the last ones below the cut); n_tok = q_start[n_seq].  Limits: n_seq 65535, n_head 4096, max_len 2^30 - 1, table_stride below 2^31, new tokens (min(max_new, n_tok)) and
 * rows (that * n_head / n_head_kv) of a sequence below 2^30.  A table entry outside the pool reads as keys and values of zero and stores nothing.
 * status (device, may be NULL): that of the b200_pages_update that made the state.  Where status[0] is not 0 there is no room for the new tokens - the state
 * is the old one, and its last tokens would be taken for them - so that nothing is stored and no row of dst and lse written.  Without it the status
 * has to be looked at before any attention or store with k_new.  For the same reason q_start has to give a sequence as many tokens as the update's n_new did
 * (none where that was 0). */
typedef struct {
    const void * q; int q_type; int64_t nb_q_tok, nb_q_head;
    void * dst; int64_t nb_dst_tok, nb_dst_head;
    const void * k_new; const void * v_new; int64_t nb_new_tok, nb_new_head;
    int layer;
    const int32_t * tables; int64_t table_stride; const int32_t * lens; const int32_t * q_start;
    int64_t n_tok; int n_seq, n_head; int64_t max_new, max_len; int causal; float scale;
    float * lse;
    void * workspace; int64_t workspace_bytes;
    const int32_t * status;
} b200_paged_attn_args;
int64_t b200_paged_attn_workspace(const b200_page_pool * pool, const b200_paged_attn_args * a);
int b200_paged_attn(const b200_page_pool * pool, const b200_paged_attn_args * a, void * stream);
/* 0, or the code of the first device-side wait that ran out on the current device since the code was last asked for (its launch left rows unfinished, although
 * the call had returned 0).  Waits for all work on the device; not while a stream is being captured.  With launches by several threads the code does not
 * tell whose it was. */
int b200_paged_attn_status(void);
/* The store alone (prompts whose attention runs elsewhere, caches filled from another source); uses of *a: k_new .. q_start,
 * n_tok, n_seq, max_new, max_len, status, and q_type as the type of k_new / v_new. */
int b200_paged_store(const b200_page_pool * pool, const b200_paged_attn_args * a, void * stream);

/* IM2COL 1-D, F16 output (ops.cpp:5784-5855): x f32 [IW, IC] (row stride bytes) ->
 * dst f16 [IC*KW, OW]. */
int b200_im2col_1d_f16(const float * x, int64_t x_stride_bytes, int64_t IW, int64_t IC, int64_t KW,
                       int64_t OW, int s0, int p0, int d0, void * dst, void * stream);

/* SOFT_MAX with optional mask and scale (ops.cpp:4641-4737, max_bias = 0): rows of ne00 f32. */
int b200_soft_max(const float * x, const void * mask, int mask_type, int64_t mask_nb1, int64_t mask_ne1,
                  float * y, int64_t ne00, int64_t nrows, int64_t ne01, float scale, void * stream);

/* CONCAT along dim (ops.cpp:2403-2604), f32, contiguous dst. */
int b200_concat(const float * a, const int64_t * nea, const int64_t * nba,
                const float * b, const int64_t * neb, const int64_t * nbb,
                float * dst, const int64_t * ned, const int64_t * nbd, int dim, void * stream);

/* log_mel_spectrogram (src/whisper.cpp:3008-3271): 16 kHz mono f32 PCM -> log-mel [n_mel][n_len]
 * on the device; out_host receives n_mel*n_len floats (n_len = (n_samples + 480000 padding)/160).
 * The result feeds whisper_set_mel_with_state (include/whisper.h:278-293). */
int b200_log_mel(int device, const float * pcm_host, int64_t n_samples, const float * filters_host,
                 int n_mel, float * out_host, int64_t out_capacity, int * n_len, int * n_len_org);

/* Same front-end with persistent device buffers, tables and a private stream, for repeated use
 * (one plan per host thread).  b200_mel_compute is synchronous: on return out_host holds
 * [n_mel][n_len] floats.  No counterpart in the reference (its mel runs on host threads). */
void * b200_mel_create(int device, const float * filters_host, int n_mel);
int    b200_mel_compute(void * plan, const float * pcm_host, int64_t n_samples, float * out_host, int64_t out_capacity,
                        int * n_len, int * n_len_org);
void   b200_mel_destroy(void * plan);

/* ---- optional entry points of the plugin (libggml-b200.so), obtained with
 * ggml_backend_reg_get_proc_address(ggml_backend_reg_by_name("B200"), name)  (ggml/include/ggml-backend.h:190):
 *
 *   void b200_logits_side_output(int top_k, int skip_readback)
 *       top_k > 0: after every decoder graph (its last node is the logits product, src/whisper.cpp:2830) the plugin also
 *       leaves b200_topk_rows of every logits row in a small device buffer of the backend instance that ran the graph.
 *       skip_readback != 0: ggml_backend_tensor_get on a logits tensor returns at once without copying - for callers
 *       that sample from the side output only; whisper_get_logits() then holds stale data.  Default: off, off.
 *   int b200_last_topk(int row, b200_topk_result * out)
 *       side output of logits row `row` of the last decoder graph computed on the CALLING thread (whisper_decode is
 *       synchronous, so that is the state the thread just stepped); waits for that graph, copies one result to the host.
 *       Returns 0, or B200_ERR_ARG when there is no such row.
 * No counterpart in the reference, which samples from the full row on the host.
 *
 * A plain exported symbol of the plugin for tests (no device work, needs no GPU):
 *   int b200_plan_probe(struct ggml_cgraph * plan_graph, struct ggml_cgraph * candidate)
 *       builds the fused execution plan of plan_graph and checks candidate against it the way a cached plan is checked
 *       before reuse: -1 when the two graphs' signatures differ, else bit 0 = candidate may run on the plan, bit 1 = the
 *       plan fuses at least one pair of nodes. */

/* Library info: number of kernel launches issued so far by this process (all entry points). */
int64_t b200_launch_count(void);
const char * b200_version(void);

#ifdef __cplusplus
}
#endif
#endif /* B200_WHISPER_H */
