/* C ABI of the MuNet MI355X (gfx950) HIP backend: libmunet_hip.so.
 *
 * Every entry point takes plain device pointers, sizes and an optional HIP
 * stream (`stream` = NULL means the HIP null stream), returns 0 on success and
 * a non-zero status otherwise; mh_last_error() gives the message of the last
 * failure on the calling thread.  No entry point allocates on the hot path
 * except where noted ("workspace"): those grow a per-device scratch buffer
 * on first use and must not be called under stream capture.
 *
 * Storage dtypes (MuNet DataType, reference src/types.hpp:16):
 *   0 = float32, 1 = float16, 2 = bfloat16, 3 = int32.
 * fp16 rounding is round-half-away (src/types.hpp:239-278), bf16 is RNE
 * without a NaN case (src/types.hpp:311-317), exactly as MuNet's codecs.
 *
 * Each declaration names the reference interface it replaces. */
#ifndef MUNET_HIP_H
#define MUNET_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MH_F32 0
#define MH_F16 1
#define MH_BF16 2
#define MH_I32 3

#define MH_DEVICE_CPU 0
#define MH_DEVICE_HIP 1

#define MH_ACT_NONE 0
#define MH_ACT_RELU 1
#define MH_ACT_GELU 2

/* ---- status / runtime --------------------------------------------------- */
/* Message of the last failed call on this thread ("" if none). */
const char *mh_last_error(void);
/* Library version string. */
const char *mh_version(void);
/* Number of visible HIP devices (BackendRegistry probe,
 * src/backend/backend_manager.cpp:21-42). */
int mh_device_count(int *count);
/* Select `device` for the calling thread and create its state. */
int mh_init(int device);
/* Backend::query_support (src/core/backend.hpp:411-425): whether this backend
 * runs `feature` on storages of `dtype`, the fallback policy when it does
 * not, and the accumulation dtype it prefers.  Feature codes 0-12 are the
 * reference's BackendFeature values in its order (src/core/backend.hpp:
 * 16-30); codes from 100 are the path's functions that have no reference
 * capability.  Policy codes follow BackendFallbackPolicy (:32-36): nothing
 * falls back to the CPU here, so the policy is always ExplicitUnsupported.
 * An unknown feature is unavailable (the reference's default); an unknown
 * dtype code is an error.  Needs no device. */
#define MH_FEATURE_ELEMENTWISE_BINARY 0
#define MH_FEATURE_BROADCAST_ROW 1
#define MH_FEATURE_MATMUL 2
#define MH_FEATURE_UNARY_ACTIVATION 3
#define MH_FEATURE_SOFTMAX 4
#define MH_FEATURE_CONCAT 5
#define MH_FEATURE_LOSS 6
#define MH_FEATURE_CONVOLUTION 7
#define MH_FEATURE_POOLING 8
#define MH_FEATURE_BATCH_NORM 9
#define MH_FEATURE_OPTIMIZER_STEP 10
#define MH_FEATURE_RANDOM_FILL 11
#define MH_FEATURE_REDUCTION 12
#define MH_FEATURE_TO_CONTIGUOUS 100
#define MH_FEATURE_LAYER_NORM 101
#define MH_FEATURE_ATTENTION 102
#define MH_FEATURE_EMBEDDING 103
#define MH_FEATURE_MASKED_FILL 104
#define MH_POLICY_EXPLICIT_UNSUPPORTED 0
#define MH_POLICY_CPU_FALLBACK 1
#define MH_POLICY_CONVERSION_FALLBACK 2
int mh_query_support(int feature, int dtype, int *available, int *fallback_policy, int *accumulation_dtype);
/* Poll and clear device-side error flags (embedding ids out of range, pages
 * and slots of the paged KV cache); synchronises the device.  Returns non-zero
 * with a message that names all kinds of error that were set. */
int mh_check_device_errors(void);

/* ---- BackendAllocationTransferCapability (src/core/backend.hpp:190-205) --- */
int mh_allocate(void **ptr, size_t bytes);                    /* :193 allocate */
int mh_deallocate(void *ptr);                                 /* :194 deallocate */
int mh_memset(void *ptr, int value, size_t bytes, void *stream); /* :195 memset */
/* :196-197 copy(src, dst, bytes, src_dev, dst_dev); devices MH_DEVICE_*.
 * Device-to-host copies complete before returning (MuNet copies are
 * synchronous, src/backend/cpu_backend.hpp:212-232). */
int mh_copy(const void *src, void *dst, size_t bytes, int src_dev, int dst_dev, void *stream);
int mh_synchronize(void *stream);                             /* :198 synchronize */
/* :200-201 get_last_kernel_time_us: GPU time of the last timed region. */
double mh_get_last_kernel_time_us(void);
/* :202-204 to_contiguous(src, dst, shape, strides, offset): strided gather. */
int mh_to_contiguous(int dt, const void *src, void *dst, int ndim, const int *shape, const int64_t *strides,
                     int64_t offset, void *stream);

/* ---- BackendElementwiseCapability (src/core/backend.hpp:207-238) --------- */
/* :210-217 add/sub/mul/div(a, b, out, BroadcastInfo): out_shape and the
 * per-operand element strides of compute_broadcast (src/types.hpp:436-478). */
int mh_add(int dt, const void *a, const void *b, void *out, int ndim, const int *out_shape,
           const int64_t *strides_a, const int64_t *strides_b, void *stream);
int mh_sub(int dt, const void *a, const void *b, void *out, int ndim, const int *out_shape,
           const int64_t *strides_a, const int64_t *strides_b, void *stream);
int mh_mul(int dt, const void *a, const void *b, void *out, int ndim, const int *out_shape,
           const int64_t *strides_a, const int64_t *strides_b, void *stream);
int mh_div(int dt, const void *a, const void *b, void *out, int ndim, const int *out_shape,
           const int64_t *strides_a, const int64_t *strides_b, void *stream);
int mh_relu(int dt, const void *in, void *out, size_t n, void *stream);    /* :220 */
int mh_sigmoid(int dt, const void *in, void *out, size_t n, void *stream); /* :222 */
int mh_exp(int dt, const void *in, void *out, size_t n, void *stream);     /* :226 */
int mh_log(int dt, const void *in, void *out, size_t n, void *stream);     /* :227 */
int mh_sqrt(int dt, const void *in, void *out, size_t n, void *stream);    /* :228 */
int mh_rsqrt(int dt, const void *in, void *out, size_t n, void *stream);   /* :229 */
int mh_sin(int dt, const void *in, void *out, size_t n, void *stream);     /* :230 */
int mh_cos(int dt, const void *in, void *out, size_t n, void *stream);     /* :231 */
/* :233-234 softmax(in, out, batch_size, num_classes): last-dim softmax. */
int mh_softmax(int dt, const void *in, void *out, int batch_size, int num_classes, void *stream);

/* ---- op-layer functions with no backend hook in the reference ------------ */
/* nn::GELU (src/nn/activations.hpp:31-38): x*sigmoid(x*1.702), three rounded ops. */
int mh_gelu(int dt, const void *in, void *out, size_t n, void *stream);
/* ops::masked_fill (src/core/ops/elementwise.cpp:8-53), int32 mask. */
int mh_masked_fill(int dt, const void *x, const int32_t *mask, void *out, size_t n, double value, void *stream);
/* ops::layer_norm (src/core/ops/normalization.cpp:125-224) over the last dim. */
int mh_layer_norm(int dt, const void *x, const void *weight, const void *bias, void *out, int rows, int cols,
                  float eps, void *stream);
/* nn::Embedding gather path (src/nn/linear.hpp:92-128): ids [n] int32,
 * weight [V, D].  Out-of-range ids write zeros and raise the device error
 * flag reported by mh_check_device_errors. */
int mh_embedding(int dt, const int32_t *ids, const void *weight, void *out, int n, int V, int D, void *stream);
/* Fused token + position embedding: out[r] = tok_w[ids[r]] + pos_w[r % T]
 * (two nn::Embedding gathers and ops::add, one rounding). */
int mh_embedding_pos(int dt, const int32_t *ids, const void *tok_w, const void *pos_w, void *out, int n, int V,
                     int D, int T, void *stream);
/* Tensor::to(DataType) (src/tensor.cpp:249-284) on device memory. */
int mh_convert(int src_dt, const void *in, int dst_dt, void *out, size_t n, void *stream);
/* No counterpart in the reference: a self-check of the kernels' fast fp16
 * rounding (zero and the normal half range by a bit trick, the rest by the
 * full codec that mh_convert uses) against that codec over all 2^32 float
 * bit patterns; *mismatches receives the count of patterns that differ in any
 * bit (0 when the fast path is exact).  Synchronises `stream`. */
int mh_check_f16_rounding(unsigned long long *mismatches, void *stream);
/* Row argmax, first index of the maximum (the demos' np.argmax). */
int mh_argmax(int dt, const void *x, int32_t *out, int rows, int cols, void *stream);
/* Measured matrix-core peak of this GPU in FLOP/s: a full grid of waves
 * issuing independent 16x16x32 bf16 (dt MH_BF16) or fp16 MFMAs on registers,
 * `iters` loop trips of 8 per wave, timed with HIP events on `stream` (the
 * call synchronises it).  No counterpart in the reference: the measured peak
 * that the roofline reports beside the datasheet one. */
int mh_measure_mfma_peak(int dt, int iters, double *flops_per_s, void *stream);
/* Measured HBM read rate in bytes/s: a full grid streams the caller's device
 * buffer `buf` (16-byte aligned, `bytes` >= 1 MiB; make it several times the
 * 256 MB last-level cache) `reps` times with 16-byte loads, timed with HIP
 * events on `stream` (the call synchronises it).  No counterpart in the
 * reference: the measured read peak the roofline reports beside the
 * datasheet HBM figure. */
int mh_measure_hbm_read(const void *buf, size_t bytes, int reps, double *bytes_per_s, void *stream);

/* ---- BackendBlasCapability (src/core/backend.hpp:250-260) ---------------- */
/* :253-254 matmul(a, b, out, M, K, N, transA, transB) on raw row-major storage.
 * Uses the workspace when transA or !transB. */
int mh_matmul(int dt, const void *a, const void *b, void *out, int M, int K, int N, int transA, int transB,
              void *stream);
/* No counterpart in the reference: mh_matmul for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  Same arguments and results as mh_matmul,
 * but the transposed operands it stages (A when transA, B when !transB) go to
 * a fixed 64 MiB per-device scratch array inside the library instead of the
 * growable workspace; a call needing more fails with a message and enqueues
 * nothing.  No hipMalloc/hipFree on any path.  The array's device address is
 * resolved by mh_init (or on the first call on a device).  Every call on one
 * GPU shares that GPU's array: calls that overlap on one GPU (two streams,
 * two threads) race and must be serialised by the caller. */
int mh_matmul_noalloc(int dt, const void *a, const void *b, void *out, int M, int K, int N, int transA, int transB,
                      void *stream);
/* :255-259 batched_matmul(..., stride_a, stride_b, stride_out); stride_b = 0
 * broadcasts one right operand.  Workspace as mh_matmul. */
int mh_batched_matmul(int dt, const void *a, const void *b, void *out, int batch, int M, int K, int N, int transA,
                      int transB, int64_t stride_a, int64_t stride_b, int64_t stride_out, void *stream);
/* nn::Linear forward (src/nn/linear.hpp:28-34) with the weight pre-packed as
 * w_t [N, K] (mh_pack_linear_weight): out = act(x*W + bias) (+ resid), with
 * the reference's rounding after the matmul, the bias add, each GELU op and
 * the residual add.  bias / resid may be NULL; act is MH_ACT_*. */
int mh_linear(int dt, const void *x, const void *w_t, const void *bias, void *out, int M, int K, int N, int act,
              const void *resid, void *stream);
/* Repack a Linear weight [in, out] (MuNet layout, src/nn/linear.hpp:14) to
 * the K-contiguous [out, in] panel the MFMA GEMM reads. */
int mh_pack_linear_weight(int dt, const void *w, void *w_t, int in_features, int out_features, void *stream);
/* The q/k/v projections of nn::MultiHeadAttention with their permute to
 * [B, H, T, hd] (src/nn/attention.hpp:47-62) as one GEMM: wqkv_t [3E, E]
 * (rows q, k, v), bqkv [3E]; q/k/v outputs [B*H*T*hd]. */
int mh_qkv_projection(int dt, const void *x, const void *wqkv_t, const void *bqkv, void *q, void *k, void *v, int B,
                      int T, int E, int H, void *stream);

/* ---- fused attention (src/nn/attention.hpp:64-99) ------------------------- */
/* q, k, v in [B*H, T, hd] (permuted, contiguous); k is read as MuNet reads it:
 * its buffer viewed as a row-major [hd, B*H*T] matrix.  ctx is written merged
 * as [B, T, H*hd].  Scale = 1/sqrt(hd) rounded to dt. */
int mh_attention(int dt, const void *q, const void *k, const void *v, void *ctx, int B, int H, int T, int hd,
                 int causal, void *stream);
/* No counterpart in the reference (its attention has no per-position keys,
 * so it cannot be decoded incrementally): the same rounding steps with key j
 * of head (b, h) read as row (b*H + h)*T + j of k, like v.  The attention of
 * the KV-cache decode (mh_decoder_*) and of DecoderLM configs with
 * "attention": "textbook". */
int mh_attention_textbook(int dt, const void *q, const void *k, const void *v, void *ctx, int B, int H, int T,
                          int hd, int causal, void *stream);

/* ---- paged 8-bit KV cache --------------------------------------------------
 * No counterpart in the reference: keys and values of many requests in one
 * pool of pages, read by ragged batches of queries (one token, a prompt, or a
 * chunk of a prompt behind a cached prefix each).
 *
 * A page holds `page` tokens (16, 32, 64, 128 or 256) of every key/value head,
 * in 8-bit floating point (e4m3: largest value 448, one NaN, no infinity) with
 * one float scale per page and head for keys and one for values:
 *   k_cache [n_pages][Hkv][page][hd], v_cache [n_pages][Hkv][hd][page] (a
 *   page's values are stored transposed), k_scale, v_scale [n_pages][Hkv].
 * An element stands for its e4m3 value times its scale.  Scales are positive;
 * those that mh_kv_store_paged writes are powers of two.  A slot is
 * page number * page + place.  A request's pages are its row of the block
 * table [B][width]: token t lies in page table[t / page], place t % page.
 * hd is a multiple of 16, at most 256; n_pages * page is below 2^31, width * page
 * at most 2^31 - 4096.  Caches are 16-byte aligned.
 * Device-side data that cannot be checked on the host never leads outside the
 * buffers: what is done instead is said below, and mh_check_device_errors
 * reports it.  None of these calls allocates; all may be captured into graphs
 * (after mh_init). */

/* Where a step's new tokens go.  Request b has lens[b] tokens in the cache and
 * gets new_lens[b] more (negative counts as 0).  The pages that it needs beyond the
 * ceil(lens[b] / page) it holds are taken from free_pages [n_free] in order, request
 * after request, and written into its row of `tables` (other entries stay).
 * Outputs: total_lens [B] = lens + new_lens; cu [B + 1], the running sum of
 * new_lens from 0; slots [n_slots], the slot of each new token, request after
 * request, -1 behind the last; positions [n_slots] (may be NULL), its position,
 * 0 behind the last; used [1], pages taken (above n_free: so many were
 * needed).  A token whose page does not exist (the free pages or the table's
 * width are exhausted, a held entry lies outside the pool) gets slot -1, a page
 * that could not be had the entry -1, tokens past n_slots are left out (cu stops
 * there), and the error flag is raised.  Outputs overlap no input and no other
 * output.  Nothing is done for B = 0; B is at most 2^20 (above some 10^4 requests
 * the time grows with B^2). */
int mh_page_plan(const int32_t *lens, const int32_t *new_lens, const int32_t *free_pages, int32_t *tables,
                 int32_t *total_lens, int32_t *cu, int32_t *slots, int32_t *positions, int32_t *used, int B, int n_free,
                 int width, int page, int n_pages, int n_slots, void *stream);
/* Keys and values of n tokens into their slots.  k, v: token rows of Hkv * hd
 * values of `dt`, ldk / ldv values apart (multiples of 16 bytes, as are the
 * pointers).  Tokens of one page follow each other, in the order of their
 * places, as mh_page_plan lists them: two separate stretches of one page in one call
 * leave that page's contents and scales unspecified.  Slots of -1 are skipped, slots
 * outside the pool too, raising the error flag.
 * For each page and head: e is the least power of two (from 2^-100) whose
 * 448-fold holds the new values' largest magnitude; the scale becomes e where the
 * page's first token is among them, else the larger of e and the scale held,
 * and if it grows the page's earlier tokens are rounded to it; values are
 * rounded to the nearest e4m3, ties to even.  Infinities and NaN become NaN and do not
 * count towards the magnitude.  n is at most 2^27, Hkv 65535. */
int mh_kv_store_paged(int dt, const void *k, const void *v, int64_t ldk, int64_t ldv, const int32_t *slots,
                      void *k_cache, void *v_cache, float *k_scale, float *v_scale, int n, int Hkv, int hd, int page,
                      int n_pages, void *stream);
/* Attention of ragged queries over the cache.  Request b's queries are token
 * rows cu[b] .. cu[b+1]-1 of q and out (Hq * hd values of `dt`, ldq / ldo values
 * apart, multiples of 16 bytes, as are the pointers; cu does not decrease), the
 * last of its lens[b] tokens: query i stands at position
 * p = lens[b] - (cu[b+1] - cu[b]) + i.  Head h reads key/value head
 * h / (Hq / Hkv).  It sees keys j < lens[b]; with `causal` only j <= p, with
 * window > 0 only j > p - window.  out = softmax(scale q k) v over those, zeros
 * for a query that sees none; scale 0 means 1 / sqrt(hd), and |scale| is at most
 * 2^127.  Rows of no request are left as they are.  Scores, softmax and sums are
 * fp32; a probability times its page's value scale enters the product with the
 * values as fp16 (for float32 as two fp16 parts, as does q), relative to the
 * row's largest.
 * max_q and max_len bound the requests' query and key counts; they size the
 * launch (larger ones on the device are still served, more slowly).  B * Hkv is
 * below 2^23, n_rows * Hq at most 2^30.
 * Table entries outside the pool hold no keys, and lengths past width * page
 * are cut there, raising the error flag; an entry none of whose keys a query of
 * the request sees (behind the window) may be anything.
 * workspace: mh_attention_paged_workspace bytes, 16-byte aligned, in use until the
 * call's work on the stream has ended; calls that may overlap need one each.  out
 * may not overlap another operand. */
int mh_attention_paged_workspace(int dt, int B, int n_rows, int Hq, int Hkv, int hd, int max_q, int max_len, int window,
                                 size_t *bytes);
int mh_attention_paged(int dt, const void *q, int64_t ldq, const void *k_cache, const void *v_cache, const float *k_scale,
                       const float *v_scale, const int32_t *tables, const int32_t *lens, const int32_t *cu, void *out,
                       int64_t ldo, int B, int n_rows, int Hq, int Hkv, int hd, int page, int n_pages, int width, int max_q,
                       int max_len, int causal, int window, float scale, void *workspace, size_t workspace_bytes,
                       void *stream);

/* ---- rotary positions ----------------------------------------------------------
 * No counterpart in the reference, whose positions are learned vectors
 * (mh_embedding_pos).  A head's first 2 * half values are `half` pairs, each turned
 * by position * frequency: pair j is (x_j, x_{j + half}), or with `interleaved`
 * (x_2j, x_{2j + 1}); what lies behind them stays.  The angles of a step's tokens
 * are worked out once (mh_rotary_table) and read by every layer.  None of the calls
 * on a stream allocates; all may be captured. */

/* Frequencies of a rotation of `rot` values (even) of each head, on the host: freq
 * [rot / 2] gets base^(-2 j / rot), changed for contexts longer than the trained:
 *   MH_ROTARY_PLAIN   as they are;
 *   MH_ROTARY_LINEAR  divided by `factor` (positions drawn together);
 *   MH_ROTARY_BASE    of the base times factor^(rot / (rot - 2)) (rot from 4 on): the
 *                     fastest stays, the slowest is divided by factor;
 *   MH_ROTARY_TURNS   by the turns r = original freq / (2 pi) that a pair makes over
 *                     the `original` trained positions: from `high` turns on as it
 *                     is, up to `low` divided by factor, between in proportion
 *                     (g f + (1 - g) f / factor, g = (r - low) / (high - low)).
 * *magnitude (may be NULL) gets 1 + 0.1 ln(factor) for MH_ROTARY_TURNS with a factor
 * above 1, else 1: what tables are to be multiplied by in models that were trained
 * so.  Others that blend by turns take the frequencies and a table of magnitude 1.
 * Frequencies that are no longer finite are refused. */
#define MH_ROTARY_PLAIN 0
#define MH_ROTARY_LINEAR 1
#define MH_ROTARY_BASE 2
#define MH_ROTARY_TURNS 3
int mh_rotary_frequencies(double *freq, double *magnitude, int rot, double base, int scaling, double factor, double original,
                          double low, double high);
/* table [n][half][2] = magnitude * (cos a, sin a), a = positions[t] * freq[j] (device
 * arrays; a exact to about 2^-50 behind its whole turns, at any int32 position).
 * table is 16-byte aligned and overlaps neither of them. */
int mh_rotary_table(const int32_t *positions, const double *freq, float *table, int n, int half, double magnitude, void *stream);
/* out = x with its pairs (a, b) turned to (a c - b s, a s + b c); with `inverse` s
 * counts negative, which is also the gradient.  x, out: n token rows of heads * hd
 * values of `dt`, ldx / ldo values apart; table [n][half][2], 2 half <= hd.  out is
 * x (with ldo = ldx) or does not overlap it, nor the table.  heads * hd is at most 2^30. */
int mh_rotary(int dt, const void *x, int64_t ldx, const float *table, void *out, int64_t ldo, int n, int heads, int hd, int half,
              int interleaved, int inverse, void *stream);
/* mh_kv_store_paged of keys that are rotated on the way (the cache's 8 bits are
 * their only rounding; mh_kv_store_paged has the other arguments and what is
 * written), and beside them q [n][Hq * hd] (rows ldq values apart) rotated
 * into q_out (ldqo apart; q itself, or not overlapping q, k, v, table or slots).  q NULL: none.
 * The caches and scales overlap neither each other nor any other operand.
 * Rows of q whose slot is -1 or outside the pool are left as they are in q_out.
 * Rows of q and q_out are multiples of 16 bytes apart, as are the pointers. */
int mh_kv_store_rotary_paged(int dt, const void *k, const void *v, int64_t ldk, int64_t ldv, const float *table,
                             const int32_t *slots, void *k_cache, void *v_cache, float *k_scale, float *v_scale, int n, int Hkv,
                             int hd, int half, int interleaved, int page, int n_pages, const void *q, int64_t ldq, void *q_out,
                             int64_t ldqo, int Hq, void *stream);

/* ---- products in 8-bit integers --------------------------------------------------
 * No counterpart in the reference.  Rows of values (a token's activations, an output
 * channel's weights) as int8 with one float scale each, and nn::Linear on them.
 * None of these calls allocates; all may be captured. */

/* q = the whole numbers nearest to 127 x / a (ties to even), scale = a / 127, a the
 * row's largest magnitude, at least 127 * 2^-126.  A row with NaN or infinities
 * gets the scale NaN (and q = 0): what is computed from it is NaN.  x [rows][cols]
 * of `dt`, rows ldx values apart, q ldq apart, of any alignment; q may not overlap
 * x, nor scale either of them. */
int mh_quantize_rows(int dt, const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int rows, int cols, void *stream);
/* out = q * scale of its row, rounded to `dt`; out overlaps neither. */
int mh_dequantize_rows(int dt, const int8_t *q, int64_t ldq, const float *scale, void *out, int64_t ldo, int rows, int cols,
                       void *stream);
/* out[m][n] = act(x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]) + resid[m][n]:
 * mh_linear with both operands in int8, [M][K] rows ldx and [N][K] rows ldw apart, of
 * any alignment (K, spacings and addresses that are all multiples of 16 are up to
 * twice as fast, K = 4090 in rows of 4096 is not; of others whole 4-byte words that
 * hold a value are read).  bias (may be NULL), resid (may be
 * NULL; rows ldr apart) and out (ldo apart) are of `dt`; act is MH_ACT_*, GELU
 * x * sigmoid(1.702 x).  The sum is exact in int32 (K is at most 2^17 - 1), the rest
 * in fp32, rounded once.  out may be resid (with ldo = ldr), else it overlaps
 * neither it nor any other operand. */
int mh_linear_i8(int dt, const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw, const float *w_scale,
                 const void *bias, const void *resid, int64_t ldr, void *out, int64_t ldo, int M, int N, int K, int act,
                 void *stream);

/* ---- sampling ----------------------------------------------------------------
 * No counterpart in the reference (its demos take np.argmax, mh_argmax here):
 * one token per row of logits [rows][cols] (rows ld values apart), drawn with
 * the given uniform numbers u [rows] in [0, 1).  Per row, from device arrays (NULL:
 * off): temperature T (1; 0 and below, and NaN: the row's argmax), top_k (off
 * at 0 and below), top_p (off at 1 and above), min_p (off at 0 and below).
 * Tokens in the order of their logits, ties by index; w = e^((x - max) / T).  Kept
 * are the first n: the least of top_k, of the fewest whose w reach top_p of the sum
 * over the first top_k, and of the count with w >= min_p; one at least.  The draw is
 * the first kept token, in index order, at which the running sum of kept w
 * exceeds u times their sum.  Sums are whole 64-bit numbers: results do not vary
 * from run to run.  NaN logits count as -inf; a row of nothing else gives -1.
 * logprob [rows] (may be NULL): log of the drawn token's share of the kept w
 * (-inf with -1).  rows is below 2^22, cols at most 2^31 - 2^21.  workspace:
 * mh_sample_workspace bytes, as in mh_attention_paged (0, whatever the size: no
 * row needs one yet). */
int mh_sample_workspace(int dt, int rows, int cols, size_t *bytes);
int mh_sample(int dt, const void *logits, int64_t ld, int rows, int cols, const float *u, const float *temperature,
              const int32_t *top_k, const float *top_p, const float *min_p, int32_t *out, float *logprob, void *workspace,
              size_t workspace_bytes, void *stream);

/* ---- BackendShapeCapability (src/core/backend.hpp:263-271) --------------- */
/* :266-267 concat(inputs, out, dim, shapes): `count` contiguous inputs of rank
 * ndim, shapes row-major count x ndim. */
int mh_concat(int dt, const void *const *inputs, int count, void *out, int dim, int ndim, const int *shapes,
              void *stream);
/* out[b][c][r] = in[b][r][c] for batch slices of rows x cols. */
int mh_transpose2d(int dt, const void *in, void *out, int batch, int rows, int cols, void *stream);

/* ---- BackendSpatialCapability (src/core/backend.hpp:291-311) ------------- */
/* :294-296 conv2d(in, weight, bias, out, B, iC, iH, iW, oC, kH, kW, s, p):
 * NCHW / OIHW, bias may be NULL.  Workspace (layout change to NHWC). */
int mh_conv2d(int dt, const void *in, const void *weight, const void *bias, void *out, int B, int iC, int iH, int iW,
              int oC, int kH, int kW, int s, int p, void *stream);
/* Channels-last conv with OHWI weights (mh_pack_conv_weight); act fused. */
int mh_conv2d_nhwc(int dt, const void *x, const void *w_ohwi, const void *bias, void *out, int B, int iC, int iH,
                   int iW, int oC, int kH, int kW, int s, int p, int act, void *stream);
/* OIHW -> OHWI repack. */
int mh_pack_conv_weight(int dt, const void *w_oihw, void *w_ohwi, int oC, int iC, int kH, int kW, void *stream);
/* Transposed conv with kernel == stride (no overlap), NHWC in/out; weight
 * packed [k*k*oC, iC] by mh_pack_convt_weight; out row stride ldc >= oC lets
 * the result land inside a channel-concat buffer. */
int mh_conv_transpose2d_nhwc(int dt, const void *x, const void *w_packed, const void *bias, void *out, int B, int iC,
                             int iH, int iW, int oC, int k, int64_t ldc, void *stream);
/* [iC, oC, k, k] -> [k, k, oC, iC]. */
int mh_pack_convt_weight(int dt, const void *w, void *w_packed, int iC, int oC, int k, void *stream);
/* :302-303 max_pool2d(in, out, B, C, iH, iW, k, s, p), NCHW. */
int mh_max_pool2d(int dt, const void *in, void *out, int B, int C, int iH, int iW, int k, int s, int p, void *stream);
int mh_max_pool2d_nhwc(int dt, const void *in, void *out, int B, int C, int iH, int iW, int k, int s, int p,
                       void *stream);
/* :307-308 upsample2d(in, out, B, C, iH, iW, scale), nearest, NCHW. */
int mh_upsample2d(int dt, const void *in, void *out, int B, int C, int iH, int iW, int scale, void *stream);
int mh_upsample2d_nhwc(int dt, const void *in, void *out, int B, int C, int iH, int iW, int scale, void *stream);
/* Layout change between NCHW and NHWC. */
int mh_nchw_to_nhwc(int dt, const void *in, void *out, int B, int C, int HW, void *stream);
int mh_nhwc_to_nchw(int dt, const void *in, void *out, int B, int C, int HW, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MUNET_HIP_H */
