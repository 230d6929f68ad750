/*
 * ct_b200.h -- C ABI of the B200 (sm_100a) attention hot path.
 *
 * Every entry point takes caller-owned device pointers, explicit element
 * strides and sizes, and a cudaStream_t passed as `void*` (NULL = legacy
 * default stream).  Nothing here allocates device memory: operations that need
 * scratch space take a `workspace` pointer whose minimum size is reported by
 * the matching *_workspace_size() query.  All launches are asynchronous on the
 * given stream; the return value reports argument validation and launch
 * errors only.  Device-side watchdog failures (a bounded wait that ran out)
 * are recorded in a per-device status word read by ct_device_status().
 *
 * Tensors are FP32 unless a declaration takes a CT_DTYPE_*.  Four-dimensional attention tensors are indexed
 * [batch, head, seq, head_dim]; strides are in elements.  Outputs are written
 * densely (contiguous) exactly as the reference launchers allocate them.
 *
 * Each declaration names the reference interface it replaces
 * (AnshSachinkumarArora/CUDA_Transformer, path:line).
 */
#ifndef CT_B200_H
#define CT_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
enum {
  CT_OK = 0,
  CT_ERR_INVALID_ARGUMENT = 1,     /* null pointer, negative size, size mismatch        */
  CT_ERR_UNSUPPORTED_HEAD_DIM = 2, /* FA2 head_dim not in {32, 64, 128}                 */
  CT_ERR_UNSUPPORTED_LAYOUT = 3,   /* strides the selected kernel cannot address (TMA)  */
  CT_ERR_LAUNCH_FAILED = 4,        /* cudaGetLastError() after a launch                 */
  CT_ERR_DEVICE_TIMEOUT = 5,       /* a device-side bounded wait expired                */
  CT_ERR_CUDA = 6,                 /* any other CUDA runtime error                      */
  CT_ERR_UNSUPPORTED_DEVICE = 7,   /* not an sm_100 device                              */
  CT_ERR_WORKSPACE_TOO_SMALL = 8   /* workspace_bytes below the *_workspace_size()      */
};

/* ---- precision modes for the tensor-core kernels ----------------------- */
enum {
  CT_PRECISION_3XTF32 = 0, /* FP32-accurate: hi/lo TF32 split, three MMAs per product   */
  CT_PRECISION_TF32 = 1,   /* one TF32 MMA per product (looser tolerance)               */
  CT_PRECISION_FP32 = 2    /* CUDA-core FP32 FFMA kernels (no tensor cores)             */
};

const char* ct_status_string(int status);
int ct_version(void);

/* Reads (and optionally clears) the device watchdog word of `device`.
 * *flag_out is 0 when no bounded wait has expired since the last clear.
 * While the word is non-zero, the tensor-core kernels of this library (FA2
 * forward, dQ, dK/dV, linear layer, tree attention) return at entry without
 * writing their outputs: a failed wait stops the device's queue of tensor-core work until
 * the caller has seen the failure and cleared the word.  No reference
 * counterpart: the reference kernels have no failure detection. */
int ct_device_status(int device, int clear, unsigned int* flag_out);

/* Limit of every bounded device-side wait (barrier phases, split-K ordering)
 * on `device`, in nanoseconds; 2 s by default.  Legitimate waits last
 * microseconds, so the limit only decides how long a stuck kernel takes to
 * give up, report CT_DEVSTAT_TIMEOUT and tear down.  Accepted range
 * [CT_WAIT_LIMIT_MIN_NS, CT_WAIT_LIMIT_MAX_NS].  The setter copies
 * synchronously; set it while no kernel of this library runs on the device.
 * No reference counterpart. */
#define CT_WAIT_LIMIT_MIN_NS 100000ull         /* 0.1 ms */
#define CT_WAIT_LIMIT_MAX_NS 60000000000ull    /* 60 s   */
int ct_set_wait_limit_ns(int device, unsigned long long limit_ns);
int ct_get_wait_limit_ns(int device, unsigned long long* limit_ns);

/* Failure-detection self-test: launches, on the current device and `stream`,
 * one CTA whose warps wait on a barrier phase that nothing ever completes.
 * The waits run out after the device's wait limit and the CTA takes the same
 * abort teardown as the attention and GEMM kernels (MMA commit and bounded
 * drain, TMEM release); the kernel then returns, leaving CT_DEVSTAT_TIMEOUT
 * in the device's status word for ct_device_status to report.  Set a short
 * limit first (ct_set_wait_limit_ns) and clear the word afterwards.  No
 * reference counterpart. */
int ct_watchdog_selftest(void* stream);

/* ======================================================================== */
/* FlashAttention-2                                                          */
/* ======================================================================== */

/* Forward: O = softmax(Q K^T / sqrt(D) [causal mask q >= k]) V and
 * LSE = rowmax + ln(rowsum) (natural log, scaled-score domain).
 * O is written contiguous [B,H,T,D]; lse contiguous [B,H,T].
 * Replaces cuda_transformer::flash_attention_fwd
 * (Transformer_launchers/flash_attn_launcher.cu:22-65) and the kernel
 * flash_attention_fwd_kernel (Transformer_kernels/flash_attention.cuh:27-170). */
int ct_fa2_fwd(const float* q, const int64_t q_stride[4],
               const float* k, const int64_t k_stride[4],
               const float* v, const int64_t v_stride[4],
               float* o, float* lse,
               int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
               int causal, int precision, void* stream);

/* delta[b,h,t] = sum_d O[b,h,t,d] * dO[b,h,t,d]; delta contiguous [B,H,T].
 * Replaces flash_attention_bwd_delta (Transformer_kernels/flash_attention.cuh:175-213). */
int ct_fa2_bwd_delta(const float* o, const int64_t o_stride[4],
                     const float* d_o, const int64_t do_stride[4],
                     float* delta,
                     int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                     void* stream);

/* dQ = sum_j dS_ij K_j / sqrt(D) with P = exp(S - L), dS = P * (dP - delta).
 * lse_stride has three entries ([B,H,T]); delta is contiguous [B,H,T].
 * Replaces flash_attention_bwd_dq (Transformer_kernels/flash_attention.cuh:216-354). */
int ct_fa2_bwd_dq(const float* q, const int64_t q_stride[4],
                  const float* k, const int64_t k_stride[4],
                  const float* v, const int64_t v_stride[4],
                  const float* d_o, const int64_t do_stride[4],
                  const float* lse, const int64_t lse_stride[3],
                  const float* delta, float* dq,
                  int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                  int causal, int precision, void* stream);

/* dV = sum_i P_ij^T dO_i ; dK = sum_i dS_ij^T Q_i / sqrt(D).
 * Replaces flash_attention_bwd_dk_dv (Transformer_kernels/flash_attention.cuh:357-504);
 * unlike the reference it skips fully masked causal tiles. */
int ct_fa2_bwd_dkdv(const float* q, const int64_t q_stride[4],
                    const float* k, const int64_t k_stride[4],
                    const float* v, const int64_t v_stride[4],
                    const float* d_o, const int64_t do_stride[4],
                    const float* lse, const int64_t lse_stride[3],
                    const float* delta, float* dk, float* dv,
                    int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                    int causal, int precision, void* stream);

/* Bytes of workspace ct_fa2_bwd and ct_fa2_bwd_fused need: the delta vector,
 * then (from a 256-byte boundary) the one-kernel backward's ordering counters
 * and launch tickets. */
size_t ct_fa2_bwd_workspace_size(int64_t batch, int64_t heads, int64_t seq_len,
                                 int64_t head_dim);

/* Full backward: delta, dQ, dK, dV (three launches on `stream`).
 * Replaces cuda_transformer::flash_attention_bwd
 * (Transformer_launchers/flash_attn_launcher.cu:67-142), which allocates delta
 * itself; here delta lives in the caller's workspace. */
int ct_fa2_bwd(const float* q, const int64_t q_stride[4],
               const float* k, const int64_t k_stride[4],
               const float* v, const int64_t v_stride[4],
               const float* o, const int64_t o_stride[4],
               const float* d_o, const int64_t do_stride[4],
               const float* lse, const int64_t lse_stride[3],
               float* dq, float* dk, float* dv,
               void* workspace, size_t workspace_bytes,
               int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
               int causal, int precision, void* stream);

/* The same backward as ct_fa2_bwd in one key/value-stationary kernel after
 * delta: P and dS are formed once per (key tile, query tile) and each CTA adds
 * its dQ contribution into dQ in a fixed order of key tiles (per-tile counters
 * in the workspace; bit-identical run to run).  TF32 precision and head dim 64
 * only (CT_ERR_INVALID_ARGUMENT / CT_ERR_UNSUPPORTED_HEAD_DIM otherwise).  Not
 * the default: on B200 it measures slower than ct_fa2_bwd's two kernels.  No
 * reference counterpart (the reference's backward is two atomics-free kernels,
 * Transformer_kernels/flash_attention.cuh:216-504). */
int ct_fa2_bwd_fused(const float* q, const int64_t q_stride[4],
                     const float* k, const int64_t k_stride[4],
                     const float* v, const int64_t v_stride[4],
                     const float* o, const int64_t o_stride[4],
                     const float* d_o, const int64_t do_stride[4],
                     const float* lse, const int64_t lse_stride[3],
                     float* dq, float* dk, float* dv,
                     void* workspace, size_t workspace_bytes,
                     int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                     int causal, int precision, void* stream);

/* Largest batch * heads * seq_len ct_fa2_bwd_noalloc accepts. */
#define CT_FA2_BWD_NOALLOC_MAX_ROWS 2097152

/* The full backward of ct_fa2_bwd for callers that cannot allocate device
 * memory (for example a plugin given only tensor pointers by a host whose
 * allocator it cannot reach, or a service that allows no cudaMalloc after
 * start-up).  This entry point has no counterpart in the reference, whose
 * launcher allocates the delta temporary with torch::empty.  Delta lives in a
 * fixed array inside this library (8 MiB held on every GPU that loads it
 * until the process exits); the call itself allocates nothing.  Returns
 * CT_ERR_WORKSPACE_TOO_SMALL when batch * heads * seq_len exceeds
 * CT_FA2_BWD_NOALLOC_MAX_ROWS.  The first call on a device looks up the
 * array's device address, so make it before any stream capture.  All calls
 * share the array: calls that overlap on the GPU race, so order them on one
 * stream (or with events). */
int ct_fa2_bwd_noalloc(const float* q, const int64_t q_stride[4],
                       const float* k, const int64_t k_stride[4],
                       const float* v, const int64_t v_stride[4],
                       const float* o, const int64_t o_stride[4],
                       const float* d_o, const int64_t do_stride[4],
                       const float* lse, const int64_t lse_stride[3],
                       float* dq, float* dk, float* dv,
                       int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                       int causal, int precision, void* stream);

/* ======================================================================== */
/* Linear layer                                                              */
/* ======================================================================== */

/* out[b] = x[b] @ W[w_batch == 1 ? 0 : b] + bias, out contiguous [batch,m,n].
 * x is [batch,m,k] with strides x_stride; W is [w_batch,k,n] with strides
 * w_stride (w_stride[0] ignored when w_batch == 1); bias is [n] with stride
 * bias_stride.  Replaces cuda_transformer::cuda_fma
 * (Transformer_launchers/linear_layer.cu:28-70) and fused_multiply_add
 * (Transformer_kernels/fused_multiply_add.cuh:10-93). */
int ct_linear_fwd(const float* x, const int64_t x_stride[3],
                  const float* w, const int64_t w_stride[3],
                  const float* bias, int64_t bias_stride,
                  float* out,
                  int64_t batch, int64_t m, int64_t k, int64_t n, int64_t w_batch,
                  int precision, void* stream);

/* Device workspace (bytes, possibly 0) that ct_linear_fwd_ws may use to split
 * the K reduction across SMs when the output has few tiles (the weight
 * gradient x^T dy over batch*seq rows). */
size_t ct_linear_workspace_size(int64_t batch, int64_t m, int64_t k, int64_t n);

/* ct_linear_fwd with a caller-owned device workspace of workspace_bytes
 * (>= ct_linear_workspace_size for the split-K schedule; smaller or NULL
 * disables it).  The slices of a split reduction are added in a fixed order,
 * so results are deterministic.  The workspace must not be used by another
 * call that can run concurrently.  Same reference counterpart as
 * ct_linear_fwd (Transformer_launchers/linear_layer.cu:28-70). */
int ct_linear_fwd_ws(const float* x, const int64_t x_stride[3],
                     const float* w, const int64_t w_stride[3],
                     const float* bias, int64_t bias_stride,
                     float* out,
                     int64_t batch, int64_t m, int64_t k, int64_t n, int64_t w_batch,
                     int precision, void* workspace, size_t workspace_bytes, void* stream);

/* Fused epilogues of ct_linear_fwd_ex. */
enum {
  CT_EPILOGUE_NONE = 0,      /* out = x W + bias                                        */
  CT_EPILOGUE_GELU = 1,      /* out = x W + bias and act_out = gelu(out) (erf form)     */
  CT_EPILOGUE_GELU_GRAD = 2  /* out = (x W + bias) * gelu'(act_in), act_in [batch,m,n]  */
};

/* ct_linear_fwd_ws with the linear layer's neighbours fused in:
 *  - `epilogue` applies GELU (gelu/gelu_bwd of Transformer_kernels/GeLU.cuh:7-29)
 *    to the GEMM's output tile before it leaves the chip: CT_EPILOGUE_GELU
 *    also writes act_out = gelu(out) (the MLP's fc1 and activation,
 *    gpt/gpt.py:134-135), CT_EPILOGUE_GELU_GRAD multiplies by the GELU
 *    derivative at act_in (the fc2 input gradient times gelu', the same
 *    MLP's backward);
 *  - `w_colsum` (batch == 1), when not NULL, receives the column sums of the
 *    W operand over the reduction index: with W = dY this is the bias
 *    gradient db, formed from the dY tiles the weight-gradient GEMM
 *    dW = x^T dY already stages (cuda_autograd_fns/cuda_linear_layer.py:25-27,
 *    Transformer_kernels/warp_sum_kernel.cuh:13-51);
 *  - `accumulate` != 0 adds into out (and w_colsum) instead of storing
 *    (CT_EPILOGUE_NONE only).
 * On the tensor cores w_colsum needs workspace_bytes >= ct_linear_workspace_size
 * (CT_ERR_WORKSPACE_TOO_SMALL otherwise): the units that share a tile column
 * add their partial sums in a fixed order through counters kept there.
 * Deterministic: split-K slices and the column sums add in a fixed order.
 * Same reference counterpart as ct_linear_fwd (linear_layer.cu:28-70). */
int ct_linear_fwd_ex(const float* x, const int64_t x_stride[3],
                     const float* w, const int64_t w_stride[3],
                     const float* bias, int64_t bias_stride,
                     float* out,
                     int64_t batch, int64_t m, int64_t k, int64_t n, int64_t w_batch,
                     int precision, int epilogue, float* act_out, const float* act_in,
                     float* w_colsum, int accumulate,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of workspace ct_bias_grad needs. */
size_t ct_bias_grad_workspace_size(int64_t batch, int64_t m, int64_t n);

/* db[j] = sum_{b,i} dy[b,i,j].  Replaces cuda_transformer::db_calculation
 * (Transformer_launchers/linear_layer.cu:74-97) and warp_sum_kernel
 * (Transformer_kernels/warp_sum_kernel.cuh:13-51).  Deterministic two-stage
 * column reduction; the partial sums live in `workspace`. */
int ct_bias_grad(const float* dy, const int64_t dy_stride[3], float* db,
                 int64_t batch, int64_t m, int64_t n,
                 void* workspace, size_t workspace_bytes, void* stream);

/* ======================================================================== */
/* Row-wise kernels                                                          */
/* ======================================================================== */

/* y = softmax(x) along the last dimension of a contiguous [rows, n] tensor.
 * Replaces cuda_transformer::cuda_softmax (Transformer_launchers/softmax_layer.cu:22-50)
 * and naive_softmax (Transformer_kernels/softmax.cuh:25-106). */
int ct_softmax_fwd(const float* x, float* y, int64_t rows, int64_t n, void* stream);

/* dx = p * (dp - sum(p * dp)) per row.  Replaces cuda_softmax_bwd
 * (Transformer_launchers/softmax_layer.cu:52-80) and naive_softmax_bwd
 * (Transformer_kernels/softmax.cuh:108-159). */
int ct_softmax_bwd(const float* p, const float* dp, float* dx, int64_t rows, int64_t n,
                   void* stream);

/* Exact (erf) GELU y = x * Phi(x).  Replaces gelu_activation
 * (Transformer_launchers/gelu_activation.cu:22-47) and gelu (Transformer_kernels/GeLU.cuh:7-16). */
int ct_gelu_fwd(const float* x, float* y, int64_t numel, void* stream);

/* dx = dy * (Phi(x) + x * phi(x)).  Replaces gelu_activation_bwd
 * (Transformer_launchers/gelu_activation.cu:49-77) and gelu_bwd (Transformer_kernels/GeLU.cuh:19-29). */
int ct_gelu_bwd(const float* x, const float* dy, float* dx, int64_t numel, void* stream);

/* LayerNorm over the last dimension of a contiguous [rows, n] tensor:
 * y = (x - mean) / sqrt(var_biased + eps) * gamma + beta (n <= 8192); mean and rstd
 * ([rows], may be NULL) are saved for the backward.  The reference has no
 * CUDA LayerNorm: this restates the PyTorch module in gpt/gpt.py:47-59. */
int ct_layernorm_fwd(const float* x, const float* gamma, const float* beta,
                     float* y, float* mean, float* rstd,
                     int64_t rows, int64_t n, float eps, void* stream);

size_t ct_layernorm_bwd_workspace_size(int64_t rows, int64_t n);

/* Gradients of ct_layernorm_fwd: dx [rows,n], dgamma [n], dbeta [n]
 * (autograd of gpt/gpt.py:55-58).  Column sums are reduced
 * deterministically through `workspace`. */
int ct_layernorm_bwd(const float* x, const float* gamma, const float* mean,
                     const float* rstd, const float* dy,
                     float* dx, float* dgamma, float* dbeta,
                     int64_t rows, int64_t n,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Cross entropy of `rows` logit rows of length `vocab` (row stride ld),
 * forward and backward together:
 *   loss_rows[r] = logsumexp(logits[r]) - logits[r][targets[r]]
 *   logits[r][:] <- softmax(logits[r]) - onehot(targets[r])   (in place)
 * A target equal to ignore_index gives loss 0 and a zero gradient row; one
 * outside [0, vocab) gives NaN for that row.  With mean reduction the caller
 * divides the summed loss and the gradient by the number of counted rows.
 * The reference applies torch's F.cross_entropy to the lm_head logits
 * (gpt/gpt.py:167-175); this lets the lm_head GEMM and the loss run chunk by
 * chunk without materialising every row of logits. */
int ct_cross_entropy_fwd_bwd(float* logits, int64_t ld, int64_t rows, int64_t vocab,
                             const int64_t* targets, int64_t ignore_index, float* loss_rows,
                             void* stream);

/* ======================================================================== */
/* Token generation: paged key/value cache, one-token attention, logits       */
/* ======================================================================== */

/* Element types of the generation operators.  Activations (q, k, v, outputs)
 * are FP32, or of the cache's type. */
enum { CT_DTYPE_F32 = 0, CT_DTYPE_BF16 = 1, CT_DTYPE_F16 = 2 };

/* A paged cache is a pool of `pages` pages of `page_size` token slots:
 * k_cache and v_cache are indexed [page, kv_head, slot, head_dim] through
 * their element strides (any order of the first three; unit stride along
 * head_dim, no negative strides; those of dimensions of one element are not
 * looked at).  Row s of block_table ([batch, max_pages]
 * int32, row stride table_stride) lists the pages of sequence s in order:
 * its token j lives in page block_table[s][j / page_size], slot
 * j % page_size.  head_dim in {32, 64, 128};
 * max_pages * page_size <= 2^30 - 256. */

/* Appends `tokens` new keys and values (k, v indexed [token, kv_head,
 * head_dim] through their strides) to the cache: token t goes to position
 * positions[t] of sequence seq_ids[t] (NULL: sequence t).  With rot_dim > 0
 * (even, <= head_dim) the first rot_dim elements of each key are turned by the
 * position's angles on the way: cos and sin are dense [max_positions,
 * rot_dim / 2] FP32 tables, and element i pairs with i + rot_dim / 2, or
 * 2i with 2i + 1 when `interleaved`.  q (NULL when q_heads is 0), indexed
 * [token, q_head, head_dim], is turned the same way into q_out; k_out, when
 * not NULL, also receives the turned keys.  Both are dense and of the
 * activations' type; they may not overlap the inputs.  A token with a negative position is
 * padding: nothing is appended and its q_out and k_out rows are zero.  A token
 * with no place (sequence, page table entry or angle row out of range) is not
 * appended and its q_out and k_out rows are NaN.  Values beyond an f16 cache's
 * range become infinite in it (ct_paged_attention says what follows).  Two
 * tokens with the same place leave a mix of both there.  No reference counterpart
 * (the reference keeps no cache). */
int ct_kv_append(const void* q, const int64_t q_stride[3],
                 const void* k, const int64_t k_stride[3],
                 const void* v, const int64_t v_stride[3],
                 void* q_out, void* k_out, const float* cos, const float* sin,
                 void* k_cache, const int64_t kc_stride[4],
                 void* v_cache, const int64_t vc_stride[4],
                 const int32_t* block_table, int64_t table_stride,
                 const int32_t* seq_ids, const int32_t* positions,
                 int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                 int64_t rot_dim, int interleaved, int64_t max_positions,
                 int64_t batch, int64_t pages, int64_t page_size, int64_t max_pages,
                 int act_dtype, int cache_dtype, void* stream);

/* ct_kv_append with the angles of other positions than the slots': token t is
 * turned by the angles of rotary_positions[t] (NULL: positions[t]) and still
 * written to positions[t].  A drafted token of a tree has the angles of its
 * depth and the slot of its number.  One without a row in the tables of angles
 * has no place, unless it is padding by positions[t].  No reference counterpart. */
int ct_kv_append_ex(const void* q, const int64_t q_stride[3],
                    const void* k, const int64_t k_stride[3],
                    const void* v, const int64_t v_stride[3],
                    void* q_out, void* k_out, const float* cos, const float* sin,
                    void* k_cache, const int64_t kc_stride[4],
                    void* v_cache, const int64_t vc_stride[4],
                    const int32_t* block_table, int64_t table_stride,
                    const int32_t* seq_ids, const int32_t* positions,
                    const int32_t* rotary_positions,
                    int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                    int64_t rot_dim, int interleaved, int64_t max_positions,
                    int64_t batch, int64_t pages, int64_t page_size, int64_t max_pages,
                    int act_dtype, int cache_dtype, void* stream);

/* Bytes of workspace ct_paged_attention needs; they do not depend on the batch
 * or the lengths. */
size_t ct_paged_attention_workspace_size(int64_t q_heads, int64_t kv_heads, int64_t head_dim);

/* Attention of one new token per sequence over the paged cache:
 *   O = sum_j softmax_j(scale q . k_j) v_j,  LSE = ln sum_j exp(scale q . k_j)
 * over the first seq_lens[b] cached tokens of sequence b.  q is indexed
 * [batch, q_head, head_dim] through its strides; q_heads is a multiple of
 * kv_heads and query head h reads key/value head h / (q_heads / kv_heads);
 * batch * q_heads < 2^31, and times (max_pages * page_size / 8 + 16) < 2^52.
 * out is dense [batch, q_heads, head_dim] of q's type; lse (may be NULL) dense
 * [batch, q_heads].  A length of zero or below gives O = 0 and LSE = -inf; one
 * beyond max_pages * page_size, or a page out of range, gives NaN.  Slots past
 * the length are not read.  Cached values that are not finite follow the
 * formula: a key with a score of -inf has no weight, a score of +inf or NaN makes
 * its head NaN, an infinite value makes its element of O infinite, or NaN where
 * its key has no weight.  (Weights below 2^-120 of the largest count as none, and
 * with more than one head a key/value head of an f16 cache those below 2^-30;
 * there, elements of an FP32 q below 2^-38 of their head's largest count as 0.)  The cache's base and strides must be multiples of
 * 16 bytes (CT_ERR_UNSUPPORTED_LAYOUT otherwise).
 * The first CT_PAGED_ATTENTION_COUNTER_BYTES of the workspace must be zero
 * before its first use; every call leaves them so, ready for the next call of
 * whatever sizes.  The workspace must be 16-byte aligned and not be used by
 * another call that can run concurrently.  Deterministic.  No reference counterpart
 * (the reference keeps no cache). */
#define CT_PAGED_ATTENTION_COUNTER_BYTES 8192
int ct_paged_attention(const void* q, const int64_t q_stride[3],
                       const void* k_cache, const int64_t kc_stride[4],
                       const void* v_cache, const int64_t vc_stride[4],
                       const int32_t* block_table, int64_t table_stride,
                       const int32_t* seq_lens, void* out, float* lse,
                       int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                       int64_t pages, int64_t page_size, int64_t max_pages, float scale,
                       int act_dtype, int cache_dtype,
                       void* workspace, size_t workspace_bytes, void* stream);

/* Sampling penalties, biases and a grammar mask on `rows` rows of logits of
 * length `vocab` (type `dtype`, row stride ld), into FP32 out (row stride
 * out_ld).  With h = tokens[r][0 .. lens[r]) (lens NULL: max_len; clamped to
 * [0, max_len]), of which the first prompt_lens[r] (NULL: 0) are the prompt,
 * and count(i) the occurrences of token i in the rest of h:
 *   x = logit(i);  where i occurs in h: x = x > 0 ? x / repetition : x * repetition
 *   x -= frequency * count(i) + presence * (count(i) > 0)
 *   x += bias_values of the row's entries with bias_ids == i, one by one
 *   x = -inf where bit i % 32 of mask[r][i / 32] is 0
 * tokens NULL: no penalties; repetition, frequency and presence are FP32
 * [rows], NULL: 1, 0 and 0; bias_n entries a row (0: none); mask NULL: none.
 * Ids outside [0, vocab) are ignored.  out may be logits itself when dtype is
 * CT_DTYPE_F32 and out_ld == ld; any other overlap is not allowed.
 * Deterministic.  The reference's GPT.generate samples from the plain softmax of
 * the logits (gpt/gpt.py:184). */
int ct_logits_process(const void* logits, int64_t ld, int dtype, float* out, int64_t out_ld,
                      int64_t rows, int64_t vocab,
                      const int64_t* tokens, int64_t tokens_ld, int64_t max_len,
                      const int32_t* lens, const int32_t* prompt_lens,
                      const float* repetition, const float* frequency, const float* presence,
                      const int64_t* bias_ids, int64_t bias_ids_ld,
                      const float* bias_values, int64_t bias_values_ld, int64_t bias_n,
                      const int32_t* mask, int64_t mask_ld, void* stream);

/* ======================================================================== */
/* Speculative decoding: drafted tokens over the paged cache                  */
/* ======================================================================== */

/* Bytes of workspace ct_tree_attention needs; they do not depend on the batch
 * or the lengths (0: arguments out of range). */
size_t ct_tree_attention_workspace_size(int64_t drafts, int64_t q_heads, int64_t kv_heads,
                                        int64_t head_dim);

/* Attention of up to `drafts` new tokens per sequence over the paged cache.
 * Sequence b has context_lens[b] tokens before them; its draft_lens[b] new ones
 * (NULL: `drafts`; clamped to [0, drafts]) are in the cache behind those, token i
 * at position context_lens[b] + i.  New token i sees the tokens before the draft
 * and the new tokens j whose bit j % 32 of the word mask[b][i][j / 32] is set
 * (mask strides in words, unit stride along the last; bits from draft_lens[b] on
 * are not looked at), or those with j <= i when mask is NULL:
 *   O = sum_j softmax_j(scale q_i . k_j) v_j,  LSE = ln sum_j exp(scale q_i . k_j)
 * q is indexed [batch, draft, q_head, head_dim] through its strides; heads are
 * shared and the cache is laid out as in ct_paged_attention, with its limits on
 * layout and types; drafts <= CT_TREE_ATTENTION_MAX_DRAFTS, batch * drafts *
 * q_heads < 2^31, and times (max_pages * page_size / 8 + 16) < 2^52.  out is dense
 * [batch, drafts, q_heads, head_dim] of q's type; lse (may be NULL) dense [batch,
 * drafts, q_heads].  Rows from draft_lens[b] on, rows that see nothing, and all
 * rows of a sequence with a negative context_lens[b] (it takes no part) give O = 0
 * and LSE = -inf; a length beyond max_pages * page_size, or a page out of range,
 * gives NaN in the rows that are there.  What slots past the last new token hold
 * has no effect (they may be fetched with the others of their page).  Cached values
 * that are not finite reach the rows that see their token, by the formula: a key
 * with a score of -inf has no weight, a score of +inf or NaN makes its row NaN, an
 * infinite value makes its element of O infinite, or NaN where its key has no
 * weight.  (Weights below 2^-100 of the largest may count as none, those over an
 * f16 cache below 2^-22.)
 * The workspace (16-byte aligned) needs no clearing and must not be used by
 * another call that can run concurrently.  Deterministic.  No reference
 * counterpart (the reference keeps no cache). */
#define CT_TREE_ATTENTION_MAX_DRAFTS 16384
int ct_tree_attention(const void* q, const int64_t q_stride[4],
                      const void* k_cache, const int64_t kc_stride[4],
                      const void* v_cache, const int64_t vc_stride[4],
                      const int32_t* block_table, int64_t table_stride,
                      const int32_t* context_lens, const int32_t* draft_lens,
                      const int32_t* mask, const int64_t mask_stride[2],
                      void* out, float* lse,
                      int64_t batch, int64_t drafts, int64_t q_heads, int64_t kv_heads,
                      int64_t head_dim, int64_t pages, int64_t page_size, int64_t max_pages,
                      float scale, int act_dtype, int cache_dtype,
                      void* workspace, size_t workspace_bytes, void* stream);

/* Which drafted tokens are kept, and the token after them.  The draft of a
 * sequence is a tree of draft_lens[b] nodes (NULL: `drafts`; clamped to [0,
 * drafts]; 1 <= drafts <= CT_VERIFY_DRAFTS_MAX; vocab < 2^30): node 0 is the last
 * token that is certain, node i > 0 proposes tokens[b][i] after its parent parents[b][i] < i
 * (parents NULL: i - 1).  target ([batch, node, vocab] through its strides, unit
 * along vocab, of type `dtype`) holds the target's probabilities of the token after
 * each node; draft_probs (NULL: proposals are certain, each the only one that its
 * drafter could make) those that the proposals after each node were drawn from, one
 * by one; uniform[b][i] are numbers in [0, 1).
 * From node 0 on, the children of the last kept node are tried in the order of
 * their numbers.  With r the target's row of that node, q the drafter's and Z = 1:
 *   child i with token x is kept when uniform[b][i] q(x) Z < r(x)
 *   else r <- max(r / Z - q, 0), Z <- sum r        (when that sum is positive)
 * and for certain proposals q(x) counts as 1, r(x) <- 0 and Z <- Z - r(x).  When no
 * child is kept, the token after the path is the first t with
 *   sum_{s <= t} r(s) > uniform[b][0] sum_s r(s)
 * (-1 when the sum is not positive), so that the tokens are distributed as the
 * target's own.  uniform NULL (draft_probs NULL too): target holds scores, a child
 * is kept when it is the best token (the lowest of equal ones), which is also the
 * token after the path; -1 for a row of -inf or with a NaN.  A child whose token is
 * outside the vocabulary is not tried.
 * counts[b]: nodes of the path, node 0 among them (0 without nodes); path
 * ([batch, drafts], dense): their numbers, then -1; new_tokens (likewise): the
 * tokens after each node of the path, then -1.  Sums and products are formed in
 * 64 bits.  Deterministic.  The reference's GPT.generate draws one token a step
 * (gpt/gpt.py:177-190). */
#define CT_VERIFY_DRAFTS_MAX 1024
int ct_verify_drafts(const void* target, const int64_t target_stride[2],
                     const void* draft_probs, const int64_t draft_stride[2], int dtype,
                     const int64_t* tokens, int64_t tokens_ld,
                     const int32_t* parents, int64_t parents_ld, const int32_t* draft_lens,
                     const float* uniform, int64_t uniform_ld,
                     int64_t* new_tokens, int32_t* path, int32_t* counts,
                     int64_t batch, int64_t drafts, int64_t vocab, void* stream);

/* The kept ones of the last tokens move up: in each of caches_n caches (of one
 * shape and type, [page, kv_head, slot, head_dim] with 4 strides each in
 * cache_strides; keys and values of all layers, any head_dim up to 65536) the
 * values at position context_lens[b] + keep[b][j] of sequence b go to position
 * context_lens[b] + j, for j < counts[b] (clamped to [0, drafts]).  keep[b][0] <
 * keep[b][1] < ... (ct_verify_drafts' path); a move is left out when its page is
 * out of range, and when keep[b][j] <= j (it is in its place).  Where they do not
 * ascend, the moved rows' values mean nothing.  Two sequences must not share the
 * pages that are written; no cache may overlap another (the same one twice is
 * refused).  No reference counterpart. */
int ct_kv_compact(void* const* caches, const int64_t* cache_strides, int64_t caches_n,
                  const int32_t* block_table, int64_t table_stride,
                  const int32_t* context_lens, const int32_t* keep, int64_t keep_ld,
                  const int32_t* counts, int64_t batch, int64_t drafts,
                  int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size,
                  int64_t max_pages, int cache_dtype, void* stream);

/* Copies page src[i] to page dst[i], i < count, in each of caches_n caches (as
 * in ct_kv_compact).  A pair with a page out of range is left out.  No dst may
 * be a src or another dst.  No reference counterpart. */
int ct_kv_copy_pages(void* const* caches, const int64_t* cache_strides, int64_t caches_n,
                     const int32_t* src, const int32_t* dst, int64_t count,
                     int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size,
                     int cache_dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CT_B200_H */
