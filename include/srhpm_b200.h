/* srhpm_b200: B200 (sm_100a) kernels for SR-HPM's speculative-verification hot path, behind a plain C ABI.
 *
 * The path verifies 1 + k drafted tokens against a quantized dense decoder in one pass:
 *   - small-batch quantized matmul (ggml_mul_mat with ne[1] = 1..16 on Q4_K / Q5_K / Q6_K / Q3_K / IQ4_XS / Q8_0)
 *   - multi-query attention over an f16 or q8_0 KV cache (ggml_flash_attn_ext with 1..16 query rows)
 *   - greedy longest-prefix acceptance over the target logits
 * and, for a batch of sequences over a paged KV cache (f16, q8_0 or q4_0), plans the pages of a step, stores into them,
 * attends over them, applies penalties, biases and token masks to the logits and accepts drafted tokens by sampling; between
 * steps it forks sequences, gives pages back and moves them together.
 *
 * Conventions (all entry points):
 *   - tensors are ggml-shaped views (srhpm_tensor: type, ne[4] in elements, nb[4] in bytes, data) of DEVICE memory,
 *     unless an argument says otherwise; the caller owns every buffer, including the work buffer (wdata) whose size
 *     the matching *_work_size call returns.
 *   - calls are asynchronous and ordered on `stream` (a cudaStream_t; NULL = the legacy default stream).
 *   - errors are returned as srhpm_status codes, never by aborting. SRHPM_UNSUPPORTED means "not handled here, run
 *     the stock path", as the reference's compute_forward returning false does.
 *   - one srhpm_ctx per device; a context may be used from several host threads only with external serialisation, but for
 *     the calls of a batch over a paged KV cache (srhpm_page_plan to srhpm_adjust_logits), which may come at once.
 */
#ifndef SRHPM_B200_H
#define SRHPM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ggml_type numbering (GGUF) */
enum srhpm_type {
    SRHPM_TYPE_F32    = 0,
    SRHPM_TYPE_F16    = 1,
    SRHPM_TYPE_Q4_0   = 2,  /* of paged caches only */
    SRHPM_TYPE_Q8_0   = 8,
    SRHPM_TYPE_Q3_K   = 11,
    SRHPM_TYPE_Q4_K   = 12,
    SRHPM_TYPE_Q5_K   = 13,
    SRHPM_TYPE_Q6_K   = 14,
    SRHPM_TYPE_Q8_K   = 15,
    SRHPM_TYPE_IQ4_XS = 23,
    SRHPM_TYPE_I32    = 26,
};

enum srhpm_status {
    SRHPM_OK             = 0,
    SRHPM_UNSUPPORTED    = 1,  /* shape / type outside this path: use the stock path */
    SRHPM_ERR_INVALID    = -1, /* inconsistent arguments */
    SRHPM_ERR_ALIGN      = -2, /* a pointer or stride misses its required alignment */
    SRHPM_ERR_WORKSPACE  = -3, /* wdata missing or smaller than *_work_size */
    SRHPM_ERR_CUDA       = -4, /* a CUDA runtime call failed (srhpm_last_cuda_error has the code) */
    SRHPM_ERR_DEVICE     = -5, /* a kernel reported an error through the context's status word */
    SRHPM_ERR_TOO_LARGE  = -6, /* the product needs more scratch than srhpm_mul_mat_static's fixed buffer holds */
};

/* q8_0 activation quantizer used for Q8_0 weights and for Q against a q8_0 KV cache (the upstream ggml-cpu quantizer
 * is not in the reference; both variants are provided). SIMD: id = 127/amax, round half to even (ggml-cpu's x86
 * path, the default). REF: id = 1/d, roundf (ggml's quantize_row_q8_0_ref). */
enum srhpm_q8_0_act_mode { SRHPM_Q8_0_ACT_SIMD = 0, SRHPM_Q8_0_ACT_REF = 1 };

typedef struct srhpm_tensor {
    int32_t type;   /* enum srhpm_type */
    int64_t ne[4];  /* elements per dimension, ggml order (ne[0] innermost) */
    size_t  nb[4];  /* bytes per step in each dimension */
    void *  data;   /* device pointer */
} srhpm_tensor;

typedef struct srhpm_ctx srhpm_ctx;

/* Context of one device: options, a device status word for bounded-wait errors, launch counters.
 * Replaces dgpu_init (dgpu/dgpu.cu:17-25); srhpm_ctx_destroy has no counterpart there. */
int  srhpm_ctx_create(int device, srhpm_ctx ** out);
int  srhpm_ctx_destroy(srhpm_ctx * ctx);
int  srhpm_ctx_set_q8_0_act_mode(srhpm_ctx * ctx, int mode);
/* kernels this context launched since creation (or the last reset) */
int64_t srhpm_ctx_launch_count(const srhpm_ctx * ctx, int reset);
/* reads (synchronously) and clears the device status word; SRHPM_ERR_DEVICE when a kernel reported an error */
int  srhpm_ctx_check(srhpm_ctx * ctx, int32_t * device_code);
int  srhpm_last_cuda_error(void);
const char * srhpm_status_str(int status);

/* ggml type facts (ggml_blck_size / ggml_type_size / ggml_row_size) */
int    srhpm_blck_size(int type);
size_t srhpm_type_size(int type);
size_t srhpm_row_size(int type, int64_t n);

/* ---- small-batch quantized matmul ------------------------------------------------------------------------------
 * Y = W X in ggml_mul_mat semantics: W = src0 [K, rows] of a quantized type (rows contiguous, nb[1] = row size,
 * data 16-byte aligned), X = src1 f32 [K, N] (any row stride, multiple of 4), Y = dst f32 [rows, N] (any row
 * stride). 1 <= N <= 16, K a multiple of 256. Activations are quantized per row and 256 columns to int8 (bit-identical
 * to the reference's srv_quantize_row, patch/srhpm.patch:5518-5575) or, for Q8_0 weights, to q8_0; each super-block
 * is decoded once for all N rows and reduced with exact int32 sums on the tensor cores.
 * Replaces tensor_traits_srv::work_size / compute_forward (patch/srhpm.patch:6366-6374, :6400-6611) and the dGPU's
 * dgpu_launch + dgpu_collect (dgpu/dgpu.cu:244-312). A row range of W (a view with fewer rows and Y a matching view)
 * is the reference's CPU/GPU row split (patch/srhpm.patch:6497-6529). */
int srhpm_mul_mat_work_size(const srhpm_tensor * W, const srhpm_tensor * X, size_t * size);
int srhpm_mul_mat(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * X, srhpm_tensor * Y, void * wdata,
                  size_t wsize, void * stream);

/* srhpm_mul_mat in ONE kernel launch: the matmul grid quantizes its own activations (every consumer warp of the grid
 * takes a share of the (super-block, row) pairs) and meets at an arrival counter before any CTA loads the records;
 * the same records, so the output is bit-identical to srhpm_mul_mat's. Same work buffer (srhpm_mul_mat_work_size).
 * Faster after a small kernel that leaves the SMs free (attention output -> its projection: the grid is resident
 * early and the activations sit in L2), slower right after another large matmul (the grid becomes resident piecewise
 * as that one drains and the meet waits for its last CTA): measured on a B200, -0.13 ms per 27B-class verify step
 * as the attention output projection, +1.5 us per product in a sweep of back-to-back products. The counter is kept by
 * the context, one per work buffer: calls through one context on several streams need separate work buffers (as
 * their activation records already do). Products whose grid would get more than two quantization jobs per warp
 * fall back to the separate quantizer. No reference counterpart (the reference quantizes on its CPU threads before
 * the barrier, patch/srhpm.patch:6455-6461). */
int srhpm_mul_mat_fused_quant(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * X, srhpm_tensor * Y,
                              void * wdata, size_t wsize, void * stream);

/* The integer part of srhpm_mul_mat, for bit-exact checks: per (token t, row r, block j) the int32 sum of
 * (integer block scale) x (code . activation) over block j (super-block of 256, or the 32-block for Q8_0), written to
 * isum[(t * rows + r) * nblk + j], and for Q4_K / Q5_K the sum of (integer min) x (activation sum) to imin (same
 * layout; may be NULL otherwise). Same kernels and decoders as srhpm_mul_mat. No reference counterpart (test hook). */
int srhpm_mul_mat_isums(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * X, int32_t * isum,
                        int32_t * imin, void * wdata, size_t wsize, void * stream);

/* srhpm_mul_mat without a work buffer, for callers that cannot allocate device memory: a host framework that hands
 * out only the tensors it owns (no scratch per operation), or a latency-critical decode loop where a cudaMalloc
 * would synchronise the device. The scratch is a fixed 1 MiB array inside the library on every device that loads
 * it, kept until the process exits; products are not split along K here. Limit: the activation records and row-block
 * counters of the product must fit 1 MiB (for K up to 32768 and N up to 16 that leaves room for 6 million weight
 * rows); beyond that the call returns SRHPM_ERR_TOO_LARGE and does nothing. The first call on a device looks up the array's device address
 * (make it before any stream capture). All calls share the array: calls whose work overlaps on the GPU race. The
 * context's device must be the calling thread's current device (else SRHPM_ERR_INVALID). Allocates nothing. No
 * counterpart in the reference. */
int srhpm_mul_mat_static(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * X, srhpm_tensor * Y,
                         void * stream);

/* Activation quantizer, row by row: X f32 [K, N] -> q int8 [N][K], d f32 [N][K/256], bsum32 int16 [N][K/32],
 * bsum16 int16 [N][K/16] (dense, device; bsum pointers may be NULL). Bit-identical to srv_quantize_row
 * (patch/srhpm.patch:5518-5575), which equals ggml's quantize_row_q8_K. */
int srhpm_quantize_rows_q8_K(srhpm_ctx * ctx, const srhpm_tensor * X, int8_t * q, float * d, int16_t * bsum32,
                             int16_t * bsum16, void * stream);
/* X f32 [K, N] -> N rows of K/32 q8_0 blocks (34 bytes each, GGUF layout), with the context's q8_0 mode.
 * ggml-cpu from_float of GGML_TYPE_Q8_0 (upstream; used by the reference at patch/srhpm.patch:670-673). */
int srhpm_quantize_rows_q8_0(srhpm_ctx * ctx, const srhpm_tensor * X, void * blocks, void * stream);

/* ---- multi-query attention -------------------------------------------------------------------------------------
 * dst = softmax(scale * Q K^T [softcap] + slope * mask [+ sink]) V in ggml_flash_attn_ext semantics, for the few query
 * tokens of a verification pass: q f32 [DK, N, H] (token stride nb[1], head stride nb[2]), k / v [256, L, Hkv] of type
 * q8_0 or f16 (DK = DV = 256; token stride nb[1] and KV-head stride nb[2] multiples of 16 bytes, data 16-byte aligned, so
 * both the [Hkv][L] layout and llama.cpp's [L][Hkv] cache view are accepted), mask f16 [>= L, >= N, ne2] applied to
 * head h from slice h % ne2 (may be NULL), sinks f32 [H] (may be NULL), dst f32 [DV, H, N] (dst row of head h and
 * token t at h * nb[1] + t * nb[2]). H a multiple of Hkv, 1 <= N <= 16. Q is quantized per row to q8_0 with the
 * context's q8_0 mode and Q.K is the exact q8_0 integer dot product, as the reference's grouped path computes it;
 * with an f16 cache Q stays f32 (split into two f16 parts on the tensor cores). Other types / head sizes:
 * SRHPM_UNSUPPORTED. wdata: srhpm_flash_attn_ext_work_size bytes (0 when the KV range is
 * not split), ordered on `stream` like every call.
 * Replaces ggml_fa_gqa_small_work_size / ggml_compute_forward_flash_attn_ext_gqa_small (patch/srhpm.patch:555-824)
 * behind the gate at patch/srhpm.patch:833-841. */
int srhpm_flash_attn_ext_work_size(const srhpm_ctx * ctx, const srhpm_tensor * q, const srhpm_tensor * k,
                                   const srhpm_tensor * v, size_t * size);
int srhpm_flash_attn_ext(srhpm_ctx * ctx, const srhpm_tensor * q, const srhpm_tensor * k, const srhpm_tensor * v,
                         const srhpm_tensor * mask, const srhpm_tensor * sinks, float scale, float max_bias,
                         float softcap, srhpm_tensor * dst, void * wdata, size_t wsize, void * stream);

/* ---- attention split over the KV range across devices ----------------------------------------------------------
 * Each device holds a range of the cache's tokens: k / v views (and the mask's columns) start at the range's first
 * token and k->ne[1] = its token count (0 for an empty range; no work buffer then). srhpm_flash_attn_ext_partial
 * takes the arguments of srhpm_flash_attn_ext except sinks and dst and writes the range's record set into `part`
 * (srhpm_flash_attn_part_size(H, N) bytes, 16-byte aligned; wdata: srhpm_flash_attn_ext_work_size of the range's
 * views): for row r = h * N + t, float {max, sum} pairs [H * N] (max of the scaled scores in base-2 units; sum = 0 for
 * a range without a finite score), zero-padded to a multiple of 16 bytes, then float acc[H * N][256] (the row's output
 * times its sum, not normalized).
 * srhpm_flash_attn_merge combines n_parts (<= 256) such sets stored one after another (for example gathered from all
 * devices in KV order), adds the sinks (f32 [H] or NULL) and writes dst f32 [256, H, N] as srhpm_flash_attn_ext would
 * for the whole range. The reference splits the KV range into chunks over its CPU threads and merges their
 * (max, sum, acc) records the same way (patch/srhpm.patch:555-579, 779-823); here the devices are the chunks. */
size_t srhpm_flash_attn_part_size(int64_t n_head, int64_t n_tokens);
int    srhpm_flash_attn_ext_partial(srhpm_ctx * ctx, const srhpm_tensor * q, const srhpm_tensor * k,
                                    const srhpm_tensor * v, const srhpm_tensor * mask, float scale, float max_bias,
                                    float softcap, void * part, void * wdata, size_t wsize, void * stream);
int    srhpm_flash_attn_merge(srhpm_ctx * ctx, const void * parts, int n_parts, const srhpm_tensor * sinks,
                              srhpm_tensor * dst, void * stream);
/* The same merge without a collective: every rank's record set sits at the start of its own buffer of
 * srhpm_flash_attn_peer_buffer_size(H, N) bytes, zeroed once and mapped on every rank (peer_buffers[j] = rank j's
 * buffer as this rank addresses it: symmetric memory), written there by srhpm_flash_attn_ext_partial. Per row, the
 * call sends its record row to every rank's buffer as 8-byte (value, epoch) words, waits (bounded: 2 s, then an error
 * status) until every rank's words in its own buffer carry the epoch, merges them in rank order, adds the sinks and
 * writes dst as srhpm_flash_attn_merge does (the same arithmetic, so the same result). epochs: u32 [H * N] on this
 * device, zero at the start, counted per call identically on every rank; two receive slots alternate, so a rank's
 * next call never overwrites words a peer still reads. Every rank must make the same calls in the same order;
 * world <= 8. No counterpart in the reference (one device). */
size_t srhpm_flash_attn_peer_buffer_size(int64_t n_head, int64_t n_tokens);
int    srhpm_flash_attn_merge_peers(srhpm_ctx * ctx, const uint64_t * peer_buffers, int world, int rank,
                                    uint32_t * epochs, const srhpm_tensor * sinks, srhpm_tensor * dst, void * stream);

/* ---- greedy acceptance -----------------------------------------------------------------------------------------
 * Target logits f32 [n_vocab, >= n_draft + 1] (row i scores the token after draft position i; row stride nb[1]) and
 * the drafted ids int32 [n_draft] (device): for i < n_draft, id_i = argmax of row i (the first maximum, as the
 * sequential greedy scan finds it); with relax > 0 a drafted token whose logit is within relax of row i's maximum is
 * taken instead; id_i is emitted and the scan stops at the first id_i != draft[i]; when all n_draft tokens are
 * accepted, the argmax of row n_draft is emitted as well. out_ids int32 [n_draft + 1] and out_n int32 (device) receive
 * the emitted ids and their count (accepted drafted tokens + 1; n_rollback = n_draft + 1 - out_n). 0 <= n_draft <= 16.
 * Replaces common_sampler_sample_and_accept_n with a greedy sampler (upstream) and the reference's relaxed acceptance
 * (patch/srhpm.patch:9-35). wdata: srhpm_verify_accept_work_size bytes. */
int srhpm_verify_accept_work_size(const srhpm_ctx * ctx, const srhpm_tensor * logits, size_t * size);
int srhpm_verify_accept(srhpm_ctx * ctx, const srhpm_tensor * logits, const int32_t * draft, int n_draft, float relax,
                        int32_t * out_ids, int32_t * out_n, void * wdata, size_t wsize, void * stream);

/* Acceptance over a vocabulary sharded across devices: each shard (logits [shard size, n_rows], global ids starting
 * at vocab_offset) writes one record per row with srhpm_argmax_shard; srhpm_accept_merge takes the records of all
 * shards ([n_shards][n_rows], in vocabulary order, gathered to one device) and emits what srhpm_verify_accept would
 * for the whole vocabulary. imax = -1 marks a shard that starts the vocabulary with a NaN logit (argmax 0), -2 a row
 * of the shard without a non-NaN value. No counterpart in the reference (its head is not sharded). */
typedef struct srhpm_argmax_record {
    float   vmax;       /* maximum over the shard's non-NaN logits of the row */
    int32_t imax;       /* its first (global) index */
    float   vdraft;     /* logit of the drafted token of this row, when the shard holds it */
    int32_t has_draft;  /* 1 when it does */
} srhpm_argmax_record;
int srhpm_argmax_shard(srhpm_ctx * ctx, const srhpm_tensor * logits, int64_t vocab_offset, const int32_t * draft,
                       int n_draft, srhpm_argmax_record * out, void * wdata, size_t wsize, void * stream);
int srhpm_accept_merge(srhpm_ctx * ctx, const srhpm_argmax_record * recs, int n_shards, int n_rows,
                       const int32_t * draft, int n_draft, float relax, int32_t * out_ids, int32_t * out_n,
                       void * stream);

/* ---- the element-wise operators of a dense decoder verify step (ggml semantics) ------------------------------------
 * Device pointers, rows of d contiguous values, n <= 16 rows. These surround the verify GEMMs in a full model step
 * (the 27B-class benchmark); the reference runs them as stock ggml operators.
 *   srhpm_get_rows: out[i] = table row ids[i] (f16 or f32 table [d, n_rows] with row stride nb[1]) as f32
 *   srhpm_add_rms_norm: x += delta (delta may be NULL), then y = x / sqrt(mean(x^2) + eps) * w     (x, y [n][d])
 *   srhpm_rope_kv: qkv rows [n][ld] = n_head query heads | n_head_kv key heads | n_head_kv value heads of head_dim;
 *       NeoX rotary embedding (pairs (j, j + head_dim/2), theta_j = pos * theta_base^(-2j/head_dim)) of the query and
 *       key heads in place, then the keys and values are stored into the caches at token pos[t] (views as for
 *       srhpm_flash_attn_ext: [head_dim, capacity, n_head_kv], f16 or q8_0 with the context's q8_0 mode)
 *   srhpm_swiglu: out[t][j] = silu(gate[t][j]) * up[t][j] for n rows of n_ff values (input row stride ld_in, output
 *       ld_out, in floats; gate and up may be the two halves of one fused gate|up GEMM output) */
int srhpm_get_rows(srhpm_ctx * ctx, const srhpm_tensor * table, const int32_t * ids, int n, float * out, void * stream);
int srhpm_add_rms_norm(srhpm_ctx * ctx, float * x, const float * delta, const float * w, float eps, float * y, int n,
                       int64_t d, void * stream);
/* Residual add + RMSNorm fused with the activation quantization of the GEMM that consumes y (a fused GEMM
 * prologue): x += delta (delta may be NULL), y = x / sqrt(mean(x^2) + eps) * w as srhpm_add_rms_norm, and the
 * activation records of y for the product with W_next (its type, rows and K = d: ne = [d, rows]) are written into
 * wdata (sized by srhpm_mul_mat_work_size(W_next, X[d, n])), bit-identical to what srhpm_mul_mat's own quantizer
 * would write; srhpm_mul_mat_prequantized(W_next, X, Y, same wdata) then runs the product on them (X's data is not
 * read, only its shape). K-quant and IQ4_XS weights (Q8_0: SRHPM_UNSUPPORTED, use srhpm_mul_mat). n <= 16,
 * d <= 16384; x, delta, w, y 16-byte aligned. */
int srhpm_add_rms_norm_quant(srhpm_ctx * ctx, float * x, const float * delta, const float * w, float eps, float * y,
                             int n, const srhpm_tensor * W_next, void * wdata, size_t wsize, void * stream);
int srhpm_mul_mat_prequantized(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * X, srhpm_tensor * Y,
                               void * wdata, size_t wsize, void * stream);
/* SwiGLU fused the same way: out = silu(gate) * up as srhpm_swiglu (rows of ld_in / ld_out floats, n_ff = W_next's
 * K columns), and the activation records of out for the product with W_next written into wdata for
 * srhpm_mul_mat_prequantized. */
int srhpm_swiglu_quant(srhpm_ctx * ctx, const float * gate, const float * up, int64_t ld_in, float * out,
                       int64_t ld_out, int n, const srhpm_tensor * W_next, void * wdata, size_t wsize, void * stream);
/* The FFN down projection with the SwiGLU in its own prologue: Y = W . h for h = silu(gate) * up (silu(g) =
 * g / (1 + exp(-g)), as srhpm_swiglu), gate and up f32 views of the same shape and row stride (ne[0] = K, ne[1] = n).
 * The GEMM grid computes h for its activation super-blocks and quantizes it into the records, as
 * srhpm_mul_mat_fused_quant does for X: the work of srhpm_swiglu_quant + srhpm_mul_mat_prequantized in one launch,
 * h itself not stored (when the grid is too small for the prologue, the SwiGLU record kernel runs first). The records
 * are the same bytes, so Y is bit-identical to that pair. K-quant and IQ4_XS W (Q8_0: SRHPM_UNSUPPORTED); wdata of
 * srhpm_mul_mat_work_size(W, gate) bytes. */
int srhpm_mul_mat_swiglu(srhpm_ctx * ctx, const srhpm_tensor * W, const srhpm_tensor * gate, const srhpm_tensor * up,
                         srhpm_tensor * Y, void * wdata, size_t wsize, void * stream);

/* Tensor-parallel residual add + RMSNorm with the all-reduce inside (row-parallel GEMM -> next norm):
 * every rank's row-parallel GEMM (attention output, FFN down) writes its partial sum [n][d] f32 into slot `slot`
 * (0 or 1) of its own symmetric buffer of srhpm_allreduce_buffer_size(d) bytes, zeroed once before first use and
 * mapped on every rank (peer_buffers: a DEVICE array of `world` addresses, this rank's own at [rank]; IPC / symmetric
 * memory set up by the caller). srhpm_add_rms_norm_allreduce then, per row: sends each of its partial values with a
 * per-(slot, row) epoch, as one 8-byte word, into the receive area of every rank's buffer, waits (bounded: 2 s, then
 * SRHPM_ERR_DEVICE through srhpm_ctx_check) until every word it receives carries the epoch, sums the ranks' values in
 * rank order (identical on every rank), adds the sum to x and writes y = x / sqrt(mean(x^2) + eps) * w. epochs: this rank's uint32 [2][16] counters, zeroed once. n <= 16, world <= 8,
 * d a multiple of 4 and <= 16384; x, w, y 16-byte aligned. The two slots alternate (O, down): a slot is rewritten only
 * after the other slot's barrier has passed on every rank. Every rank must make the same sequence of calls. No
 * counterpart in the reference (it runs on one device): the tensor-parallel decoder's all-reduce after O and down. */
size_t srhpm_allreduce_buffer_size(int64_t d);
int srhpm_add_rms_norm_allreduce(srhpm_ctx * ctx, float * x, const uint64_t * peer_buffers, int world, int rank,
                                 int slot, uint32_t * epochs, const float * w, float eps, float * y, int n, int64_t d,
                                 void * stream);
/* srhpm_add_rms_norm_allreduce fused with the activation quantization of the GEMM that consumes y, as
 * srhpm_add_rms_norm_quant is for srhpm_add_rms_norm: the same exchange and rank-order sum of the ranks' slot
 * `slot` rows, the residual add and the norm, and W_next's activation records written into wdata for
 * srhpm_mul_mat_prequantized. One launch instead of the norm plus srhpm_mul_mat's own quantizer; each row is spread
 * over a cluster of 8 CTAs (each sends and sums a share of the columns), with results bit-identical to one CTA per
 * row. Same limits as both (K-quant and IQ4_XS W_next, n <= 16, d <= 16384, world <= 8). No counterpart in the
 * reference (one device). */
int srhpm_add_rms_norm_allreduce_quant(srhpm_ctx * ctx, float * x, const uint64_t * peer_buffers, int world,
                                       int rank, int slot, uint32_t * epochs, const float * w, float eps, float * y,
                                       int n, const srhpm_tensor * W_next, void * wdata, size_t wsize, void * stream);
int srhpm_rope_kv(srhpm_ctx * ctx, float * qkv, int64_t ld, int n, int n_head, int n_head_kv, int head_dim,
                  const int32_t * pos, float theta_base, const srhpm_tensor * k_cache, const srhpm_tensor * v_cache,
                  void * stream);
int srhpm_swiglu(srhpm_ctx * ctx, const float * gate, const float * up, int64_t ld_in, float * out, int64_t ld_out,
                 int n, int64_t n_ff, void * stream);

/* ---- a batch of sequences over a paged KV cache ----------------------------------------------------------------
 * One step of a batch: the new token rows of n_seqs sequences stand one sequence after another in row buffers of T
 * rows; sequence s has rows q_start[s] .. q_start[s + 1] - 1 (any number, 0 too), and rows behind the last sequence
 * are padding. The caches are pools of pages: k / v views with ne = [head_dim, page_size, n_head_kv, n_pages] and
 * strides nb[1] (token), nb[2] (KV head), nb[3] (page), type f16, q8_0 or q4_0 (ggml's blocks of 32 values: the step d as
 * f16, then 16 bytes of which byte j holds number j in its low and number j + 16 in its high half; value d * (number - 8)). A sequence's position p sits in slot p %
 * page_size of the page that entry p / page_size of its block table row names (block_table: i32, ne = [entries,
 * n_seqs], row stride nb[1]); a slot number is page * page_size + p % page_size. All lengths, tables and slots are
 * read on the device, so a step can be captured once and replayed with new ones. A verify step calls, in this
 * order: srhpm_page_plan, then per layer srhpm_rope_kv_paged and srhpm_flash_attn_paged, and srhpm_verify_sample on
 * the logits of the rows to be scored (all of a draft, the last one of a prompt, none of a refused sequence), with
 * starts of their own. No counterpart in the reference (one sequence, a contiguous cache, greedy acceptance). */

/* srhpm_page_plan: the step's block table entries, row starts, cache lengths, positions and slots, from the
 * sequences' lengths: n_past[s] tokens in the cache (its first ceil(n_past / page_size) table entries name their
 * pages) and n_new[s] >= 0 new ones (i32 [n_seqs] both). n_held i32 [n_seqs] or NULL: table entries that name a
 * sequence's pages already, where they are more than its cache fills (after rejected tokens: max(n_held, ceil(kv_len
 * / page_size)) of the step before; without n_held those pages are taken anew). A sequence that needs pages takes
 * them, in order of sequences, from free_pages[*free_head ..] (free_head NULL: 0; n_free entries in all), written
 * behind its entries; n_taken i32 [1] receives how many were taken (the next step's head is *free_head + *n_taken).
 * Outputs: q_start i32 [n_seqs + 1]; kv_len i32 [n_seqs] = n_past + n_new; per row pos i32 [n_rows] and slots i64
 * [n_rows] (padding rows: 0 and -1); status i32 [n_seqs], one of srhpm_page_status. A refused sequence takes no page
 * and its kv_len is 0; its rows keep their place in q_start, with the pos and slots of padding (they store nothing
 * and attend to nothing, but srhpm_verify_sample would score them); one that finds no free page refuses every later
 * one that needs a page too. A negative table entry of a page in the cache gives slot -1. Nothing else of the table
 * is written. 1 <= n_seqs <= 8192; page_size >= 1; free_pages, pos and slots may be NULL where n_free or n_rows is 0.
 * No output may share memory with an input (kv_len with the next step's n_past, say: SRHPM_ERR_INVALID); the table
 * with neither. */
enum srhpm_page_status {
    SRHPM_PAGES_OK         = 0,
    SRHPM_PAGES_TABLE_FULL = 1, /* more pages than the table row has entries */
    SRHPM_PAGES_NONE_FREE  = 2, /* the free list is used up */
    SRHPM_PAGES_BAD_LENGTH = 3, /* a negative length */
    SRHPM_PAGES_NO_ROWS    = 4, /* its rows end behind n_rows */
};
int srhpm_page_plan(srhpm_ctx * ctx, const int32_t * n_past, const int32_t * n_new, const int32_t * n_held, int n_seqs,
                    int page_size, const srhpm_tensor * block_table, const int32_t * free_pages, int n_free, const int32_t * free_head,
                    int n_rows, int32_t * q_start, int32_t * kv_len, int32_t * pos, int64_t * slots, int32_t * status,
                    int32_t * n_taken, void * stream);

/* srhpm_rope_kv_paged: qkv f32 rows, ne = [(n_head + 2 n_head_kv) * head_dim, n] (query heads | key heads | value
 * heads; only read): NeoX rotary embedding of the query and key heads at pos[t] (as srhpm_rope_kv, the angles in 64
 * bits), the turned queries written to q_out (f32 or f16, ne = [head_dim, n, n_head], the query view of
 * srhpm_flash_attn_paged), the turned keys and the values into the cache rows of slots[t] (i64; a slot outside the
 * cache, -1 of a padding row among them, stores nothing; two rows with one slot leave either's values there). f16
 * values round to nearest, q8_0 uses the context's q8_0 mode, q4_0 ggml's reference rounding (d = -m / 8 for the value m of
 * largest size, the first of equals; number = min(15, trunc(x * (1 / d) + 8.5)) in f32; a key's block is
 * turned in 64 bits where a value is next to the border of two numbers, or where two values of unlike signs are nearly of
 * the largest size). q_out shares no memory with qkv or the caches. head_dim 64, 128 or 256; qkv and q_out 16-byte
 * aligned with row strides multiples of 16; cache strides multiples of 16 (f16) or 2 (q8_0, q4_0). */
int srhpm_rope_kv_paged(srhpm_ctx * ctx, const srhpm_tensor * qkv, int n_head, int n_head_kv, const int32_t * pos,
                        const int64_t * slots, float theta_base, const srhpm_tensor * q_out,
                        const srhpm_tensor * k_cache, const srhpm_tensor * v_cache, void * stream);

/* srhpm_flash_attn_paged: row i of sequence s, at position p = kv_len[s] - (rows of s) + i, attends to the cached
 * positions j <= p, and j > p - window where window > 0: dst = softmax(scale * q k [softcap * tanh(. / softcap)] [+
 * sink]) v. q: ne = [head_dim, T, n_head], f32 or f16 (token stride nb[1], head stride nb[2]); dst of the same type,
 * ne = [head_dim, n_head, T] (head stride nb[1], token stride nb[2], as in srhpm_flash_attn_ext); head h reads KV
 * head h / (n_head / n_head_kv); sinks f32 [n_head], finite or -inf, or NULL. A row that sees nothing is 0; padding
 * rows of dst stay as they are. f16 rows: probabilities are rounded to f16 for the product with v, sums are kept in
 * f32. f32 rows: q and the probabilities are taken as sums of two f16 parts: off by at most 2^-22 of themselves, or
 * 2^-25 (q) and 2^-32 of the row's largest (probabilities) where that is more, beside f32 sums. A q8_0 or q4_0
 * cache is read as d * q or d * (q - 8) rounded to f16 (2^-11 of each value), with f32 rows too. head_dim 64, 128 or 256
 * (q8_0: 256); page_size a multiple of 16; cache data aligned to 16 bytes and its strides multiples of 16 (q4_0: both of
 * head_dim / 16 bytes, which rows side by side always have); q and dst 16-byte aligned with strides
 * multiples of 16. Cache slots behind a sequence's kv_len and before its window may hold anything, and pages wholly
 * before the window may be given away (their entries are not read). A table entry that is not a page of the cache
 * reads as zeros and raises the context's device status; positions behind the table's entries are not seen. Where the
 * scores of a row hold a NaN, its result is NaN; a value of the cache that is infinite or NaN reaches every row of
 * its sequence if one of them sees it. f32 q: finite in f16's range. dst overlaps neither q nor the caches. n_seqs <=
 * 8192, and (T * n_head / n_head_kv / 56 + 1) * (entries * page_size / 64 + 1) < 2^31, over q4_0 with 8 and 16 in place of 56
 * and 64 (else SRHPM_UNSUPPORTED).
 * wdata: srhpm_flash_attn_paged_work_size bytes, of the call alone until it is done; for f16 rows of prompts over a q4_0 cache (more
 * than 1.5 head_dim rows per sequence and KV head, padding included) the pools as f16 are among them, up to 1 GiB. */
int srhpm_flash_attn_paged_work_size(const srhpm_ctx * ctx, const srhpm_tensor * q, const srhpm_tensor * k_cache,
                                     int n_seqs, size_t * size);
int srhpm_flash_attn_paged(srhpm_ctx * ctx, const srhpm_tensor * q, const srhpm_tensor * k_cache,
                           const srhpm_tensor * v_cache, const srhpm_tensor * block_table, const int32_t * q_start,
                           const int32_t * kv_len, const srhpm_tensor * sinks, float scale, float softcap, int window,
                           srhpm_tensor * dst, void * wdata, size_t wsize, void * stream);

/* srhpm_verify_sample: acceptance of drafted tokens that keeps the target's distribution, from given random numbers.
 * logits f32 [n_vocab, T]; ids i32 [T] are the rows' input tokens: row r of a sequence scores the token behind
 * ids[r], so its drafted token is x = ids[r + 1] (none for the sequence's last row). Every row but the last is taken
 * for a draft's: of a prompt, whose tokens are given, only the last row belongs here, and no row of a sequence that
 * srhpm_page_plan refused; q_start i32 [n_seqs + 1] are the starts of these rows. p_r = softmax(logits_r /
 * temperature[s]) (temperature NULL: 1; <= 0: all on the row's first maximum); q_r the drafter's distribution
 * (draft_probs f32 [n_vocab, >= T], >= 0; NULL: all on x). Rows are scanned in order: x is accepted when u_accept[r]
 * * q_r(x) < p_r(x); the first row whose x is not accepted emits a token drawn from max(p_r - q_r, 0), and when all
 * are accepted the last row emits one drawn from p_r: the first j whose inclusive sum of weights is above u_sample[s]
 * times their total (a total of 0: the row's first maximum). NaN logits count as -inf. out_ids i32 [T]: the emitted
 * ids in the sequence's rows, -1 in the rest of them; out_n i32 [n_seqs]: their count (accepted + 1; 0 for a sequence
 * without rows); p_draft f32 [T] or NULL: p_r(x) of each row with a drafted token, 0 for a last row. Padding rows of
 * out_ids and p_draft stay as they are. u_accept f32 [T], u_sample f32 [n_seqs], in [0, 1). p_r(x) of the acceptance
 * and of p_draft has its sum in 32 bits: it is off by less than 2^-16 of itself (2^-22 mostly). The weights of a
 * drawn token and their sums are kept in 64 bits, each exponential to 2^-39 of itself, so the token does not hang on
 * the order of summation and one whose weight is 0 is never drawn (an exponential below e^-690 of the row's largest,
 * a border taken in f32, counts as 0). out_ids, out_n and p_draft share no memory with the other vectors
 * (SRHPM_ERR_INVALID). n_vocab <= 2^29; T and n_seqs <= 2^24. wdata: srhpm_verify_sample_work_size bytes, of the call
 * alone until it is done. */
int srhpm_verify_sample_work_size(const srhpm_ctx * ctx, const srhpm_tensor * logits, int n_seqs, size_t * size);
int srhpm_verify_sample(srhpm_ctx * ctx, const srhpm_tensor * logits, const int32_t * ids, const int32_t * q_start,
                        int n_seqs, const srhpm_tensor * draft_probs, const float * temperature,
                        const float * u_accept, const float * u_sample, int32_t * out_ids, int32_t * out_n,
                        float * p_draft, void * wdata, size_t wsize, void * stream);

/* srhpm_page_fork: n_forks new sequences that begin with the first n_keep[i] >= 0 tokens of others: block table row child[i]
 * gets the first ceil(n_keep / page_size) entries of row parent[i]. Whole pages are shared: page_refs i32 [n_pages] (zeros at
 * the start, kept by these calls) counts a page's holders beyond the first. A partly filled last page is replaced by one
 * taken from free_pages, in order of forks, as srhpm_page_plan takes them (free_head, n_taken), and its copy is left to
 * srhpm_page_copy: src[i], dst[i] (i32 [n_forks]; -1 and -1 where there is nothing to copy). The child's n_past is n_keep[i]. status i32
 * [n_forks], of srhpm_page_status: a refused fork writes no entry and takes nothing; SRHPM_PAGES_BAD_LENGTH also for a row
 * that the table lacks and for parent = child. An entry that is no page is handed on uncounted; if it is the partly filled
 * one's, a page is taken and nothing copied. No two forks have one child, and no child is a parent of the same call (the rows
 * then hold either's entries). The child's row names no page before that is not given up elsewhere. Nothing else of the table
 * is written. Shared pages are not written to as long as neither sequence's n_past falls below n_keep[i] (below it, it
 * would write into what the other reads). n_forks <= 8192. No output shares memory with an input
 * or another output (SRHPM_ERR_INVALID). Not before n_keep[i] tokens of the parent are stored: calls are ordered on the
 * stream. */
int srhpm_page_fork(srhpm_ctx * ctx, const int32_t * parent, const int32_t * child, const int32_t * n_keep, int n_forks,
                    int page_size, const srhpm_tensor * block_table, int32_t * page_refs, int n_pages,
                    const int32_t * free_pages, int n_free, const int32_t * free_head, int32_t * src, int32_t * dst,
                    int32_t * status, int32_t * n_taken, void * stream);

/* srhpm_page_copy: page src[i] copied to page dst[i], i < n (i32 [n]; where either is not a page, nothing), in each of
 * n_caches pools (an array of views in HOST memory: K and V of every layer, say), in one launch per 256 of them. The pools
 * have one type (f16, q8_0 or q4_0), shape and strides (any multiples of 2). n_moves i32 [1] or NULL: only the first
 * *n_moves. No dst stands twice or is a src of the same call (its page then holds either's bytes). */
int srhpm_page_copy(srhpm_ctx * ctx, const srhpm_tensor * caches, int n_caches, const int32_t * src, const int32_t * dst, int n,
                    const int32_t * n_moves, void * stream);

/* srhpm_page_free: entries begin[i] .. end[i] - 1 (i32 [n]; begin NULL: 0) of block table rows rows[i] are given up: they
 * become -1, each page's count of holders goes down, and the pages without one are written in front of *free_head into
 * free_pages (i32 [n_free]), in the order of their numbers; n_freed i32 [1] receives how many (the next step's head is
 * *free_head - *n_freed). For sequences that are done (0, entries held), and for pages behind a cache or before a window. An
 * entry given up twice counts once; rows that the table lacks and entries that are no page are passed over. Pages that find
 * no room in front of the head (more than were taken from the list) are lost, and the context's device status is raised.
 * n_pages <= 2^22. No output shares memory with an input or another output (SRHPM_ERR_INVALID). */
int srhpm_page_free(srhpm_ctx * ctx, const int32_t * rows, const int32_t * begin, const int32_t * end, int n,
                    const srhpm_tensor * block_table, int32_t * page_refs, int n_pages, int32_t * free_pages, int n_free,
                    const int32_t * free_head, int32_t * n_freed, void * stream);

/* srhpm_page_compact: the pages in use (named by the first n_held[s] entries of the block table's rows; i32 [n_seqs]) get the
 * lowest numbers, so that the pool's end can be given away: with n_used of them, the k-th page in use from n_used on goes to
 * the k-th number below n_used that is not. The table's entries and page_refs follow, free_pages (i32 [n_pages]) becomes the
 * number i at place i for n_used <= i < n_pages (its head is n_used from here on; the places before it stay), and src, dst
 * (i32 [n_pages / 2]), n_moves, n_used (i32 [1]) say what srhpm_page_copy has to move; entries behind n_moves stay as they
 * are. n_pages <= 2^22.
 * No output shares memory with an input or another output (SRHPM_ERR_INVALID). */
int srhpm_page_compact(srhpm_ctx * ctx, const srhpm_tensor * block_table, const int32_t * n_held, int32_t * page_refs, int n_pages,
                       int32_t * free_pages, int32_t * src, int32_t * dst, int32_t * n_moves, int32_t * n_used, void * stream);

/* srhpm_adjust_logits: rules on the logits f32 [n_vocab, T] of the rows that a step scores, before srhpm_verify_sample (ids
 * and q_start as there). For the tokens x of row r of sequence s, in this order:
 *   bias        l += bias[j] where bias_ids[j] = x for a j in bias_start[s] .. bias_start[s + 1] - 1 (the last such j; i32
 *               [n_seqs + 1], i32 and f32 [n_bias]; n_bias 0: none)
 *   penalties   where x stands c > 0 times in the row's window: l = l / repeat[s] if l > 0, else l * repeat[s]; then l -= c *
 *               frequency[s] + presence[s] (f32 [n_seqs] each, repeat > 0; NULL: 1, 0 and 0). The window is the last
 *               last_n[s] (i32 [n_seqs]; negative, or NULL: all) tokens of the sequence's history (i32, ne = [capacity,
 *               n_seqs], n_history[s] of them: those before its first row here; or NULL) followed by ids[q_start[s]] ..
 *               ids[r], so a drafted token counts in the rows behind it
 *   mask        l = -inf where bit x % 32 of word x / 32 is 0 in the row's mask (mask i32, ne = [>= ceil(n_vocab / 32),
 *               masks], or NULL): mask_row[r] (i32 [T]; outside the masks: none), or r where mask_row is NULL
 * each operation rounded to f32 by itself (c * frequency, then + presence, then l minus that). out f32 [n_vocab, T]:
 * the logits themselves (rows without a mask are then touched only where a rule changes them), or memory that shares
 * nothing with them; padding rows of out stay as they are. Tokens outside the vocabulary are passed over. A row whose
 * mask leaves nothing is all -inf (srhpm_verify_sample then emits token 0). T and n_seqs <= 2^24, n_vocab <= 2^29,
 * max(T, n_seqs) * ceil(n_vocab / 4096) < 2^31 (else SRHPM_UNSUPPORTED). */
int srhpm_adjust_logits(srhpm_ctx * ctx, const srhpm_tensor * logits, const int32_t * ids, const int32_t * q_start, int n_seqs,
                        const srhpm_tensor * history, const int32_t * n_history, const int32_t * last_n, const float * repeat,
                        const float * frequency, const float * presence, const int32_t * bias_start, const int32_t * bias_ids,
                        const float * bias, int n_bias, const srhpm_tensor * mask, const int32_t * mask_row,
                        const srhpm_tensor * out, void * stream);

/* ---- host-side weight quantizer (CPU) -------------------------------------------------------------------------
 * f32 rows -> GGUF blocks of `type` (Q4_K, Q5_K, Q6_K, Q3_K, IQ4_XS, Q8_0, F16). Host pointers. Returns the bytes
 * written. ggml_quantize_chunk's contract (upstream); imatrix is accepted and ignored (uniform importance). */
size_t srhpm_quantize_chunk(int type, const float * src, void * dst, int64_t start, int64_t nrows, int64_t n_per_row,
                            const float * imatrix);

#ifdef __cplusplus
}
#endif
#endif /* SRHPM_B200_H */
