// ct_internal.h -- host-side declarations shared by the kernel translation
// units and the C-ABI layer (capi.cu).  No torch types anywhere.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/ct_b200.h"

namespace ct {

// Per-device state, created on first use with the device current.
struct DeviceInfo {
  int device = -1;
  int sm_count = 0;
  int cc_major = 0, cc_minor = 0;
  uint32_t* status = nullptr;  // device address of the watchdog word
};

// Returns the state of the current device (initialising it on first use), or
// nullptr with *err set on failure.
const DeviceInfo* current_device(int* err);

// Encodes a TMA descriptor for an FP32 tensor of rank 3 or 4 with a 32-float
// (128-byte) inner box.  `mn_major` selects CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B
// (tiles the tensor core reads MN-major) instead of CU_TENSOR_MAP_SWIZZLE_128B
// (tiles read K-major).  dims[0] is the contiguous dimension; strides_bytes[i]
// is the stride of dims[i + 1].  Returns CT_OK or CT_ERR_UNSUPPORTED_LAYOUT
// when TMA cannot address the tensor.
int make_tmap_f32(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
                  const uint64_t* strides_bytes, const uint32_t* box, bool mn_major = false);

// Encodes a TMA descriptor for the pages of a cache: [page, kv_head, slot, dim]
// of a CT_DTYPE_*, read in boxes of 128 bytes of a row (64 of a shorter row)
// times `rows` slots times `box_heads` heads of one page, swizzled over that many
// bytes.  strides are in elements; those of single-element dimensions are not looked at.
int make_tmap_pages(CUtensorMap* map, const void* base, int dtype, int64_t pages, int64_t heads,
                    int64_t page_size, int64_t head_dim, const int64_t strides[3], int rows,
                    int box_heads = 1);

// True when a float tensor with these element strides (innermost first
// omitted) can be described by a TMA map: unit inner stride, 16-byte aligned
// base and outer strides.
bool tma_compatible(const void* base, int64_t inner_stride, const int64_t* outer, int n_outer);

inline int check_launch() {
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CT_OK : CT_ERR_LAUNCH_FAILED;
}

// ---------------------------------------------------------------- FA2 args
struct Fa2Problem {
  int64_t B, H, T, D;
  bool causal;
  int precision;
};
struct Strided4 {
  const float* ptr;
  int64_t s[4];  // batch, head, seq, dim (elements)
};

// ------------------------------------------ FA2 entry-point validation / dispatch
// Shared by every FA2 entry point of the C ABI (capi.cu, fa2_bwd_noalloc.cu).
// Shape check without any CUDA call: sizes non-negative, head_dim positive,
// T < 2^31 and B*H < 2^31 (each factor bounded before the product is formed,
// so the product cannot overflow).  After it, B*H*T < 2^62.
bool fa2_shape_ok(int64_t B, int64_t H, int64_t T, int64_t D);
bool valid_precision(int p);
// fa2_shape_ok + precision + head dim in {32, 64, 128} (status, no CUDA call).
int fa2_validate(int64_t B, int64_t H, int64_t T, int64_t D, int precision);
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline Strided4 s4(const float* p, const int64_t* s) {
  Strided4 t;
  t.ptr = p;
  for (int i = 0; i < 4; ++i) t.s[i] = s[i];
  return t;
}
// dQ / dK-dV launch on the tensor cores when they cover the problem, else on
// the FP32 CUDA-core kernels.
int fa2_dq_dispatch(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 g,
                    const float* lse, const int64_t* ls, const float* delta, float* dq,
                    const DeviceInfo& dev, cudaStream_t st);
int fa2_dkdv_dispatch(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 g,
                      const float* lse, const int64_t* ls, const float* delta, float* dk,
                      float* dv, const DeviceInfo& dev, cudaStream_t st);

// Kernel launchers (one translation unit each).  All return a ct status.
int launch_fa2_fwd_tc(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, float* o,
                      float* lse, const DeviceInfo& dev, cudaStream_t st);
int launch_fa2_bwd_dq_tc(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 dO,
                         const float* lse, const int64_t lse_s[3], const float* delta, float* dq,
                         const DeviceInfo& dev, cudaStream_t st);
int launch_fa2_bwd_dkdv_tc(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 dO,
                           const float* lse, const int64_t lse_s[3], const float* delta,
                           float* dk, float* dv, const DeviceInfo& dev, cudaStream_t st);
// The one-kernel backward (TF32, head dim 64): dQ, dK and dV from one
// key/value-stationary pass, dQ added in a fixed key-tile order.  sync_words:
// fa2_bwd_fused_sync_words(B, H, T) 32-bit words of device scratch (ordering
// counters and per-launch tickets), zeroed by the launcher on `st`.
int launch_fa2_bwd_fused_tc(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 dO,
                            const float* lse, const int64_t lse_s[3], const float* delta,
                            float* dq, float* dk, float* dv, uint32_t* sync_words,
                            const DeviceInfo& dev, cudaStream_t st);
size_t fa2_bwd_fused_sync_words(int64_t B, int64_t H, int64_t T);
// dK/dV on CTA pairs (TF32, head dim 64; fa2_bwd_pair.cu): the default for
// that case unless CT_FA2_PAIR_DKDV=0.
int launch_fa2_bwd_dkdv_pair(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v,
                             Strided4 dO, const float* lse, const int64_t lse_s[3],
                             const float* delta, float* dk, float* dv, const DeviceInfo& dev,
                             cudaStream_t st);
bool fa2_bwd_pair_supported(const Fa2Problem& p);
// Persistent dQ (TF32, head dim 64; fa2_bwd_dq_persist.cu): the default for
// that case unless CT_FA2_PERSIST_DQ=0.
int launch_fa2_bwd_dq_persist(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v,
                              Strided4 dO, const float* lse, const int64_t lse_s[3],
                              const float* delta, float* dq, const DeviceInfo& dev,
                              cudaStream_t st);
bool fa2_bwd_dq_persist_supported(const Fa2Problem& p);
// Whether the tensor-core kernels cover this problem (head dim / precision).
bool fa2_fwd_tc_supported(const Fa2Problem& p);
bool fa2_bwd_tc_supported(const Fa2Problem& p);
bool fa2_bwd_fused_supported(const Fa2Problem& p);

// CUDA-core FP32 kernels: any strides, head_dim in {32, 64, 128}.
int launch_fa2_fwd_simt(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, float* o,
                        float* lse, cudaStream_t st);
int launch_fa2_bwd_dq_simt(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v, Strided4 dO,
                           const float* lse, const int64_t lse_s[3], const float* delta,
                           float* dq, cudaStream_t st);
int launch_fa2_bwd_dkdv_simt(const Fa2Problem& p, Strided4 q, Strided4 k, Strided4 v,
                             Strided4 dO, const float* lse, const int64_t lse_s[3],
                             const float* delta, float* dk, float* dv, cudaStream_t st);
int launch_fa2_delta(const Fa2Problem& p, Strided4 o, Strided4 dO, float* delta, cudaStream_t st);

// ------------------------------------------------------------- GEMM args
struct GemmProblem {
  int64_t batch, m, k, n;
  const float* x;
  int64_t xs[3];  // batch, row (m), col (k)
  const float* w;
  int64_t ws[3];  // batch (0 = shared), row (k), col (n)
  const float* bias;
  int64_t bias_s;
  float* out;     // contiguous [batch, m, n]
  int precision;
  // Fused epilogues (CT_EPILOGUE_*): GELU writes gelu(out) to out_act as well;
  // GELU_GRAD multiplies out by gelu'(act_in) (act_in dense [batch, m, n]).
  int epilogue = CT_EPILOGUE_NONE;
  float* out_act = nullptr;
  const float* act_in = nullptr;
  // Column sums of the W operand over the batch and reduction indices, [n]
  // (the bias gradient when W is dY); batch == 1.
  float* w_colsum = nullptr;
  bool accumulate = false;  // out (and w_colsum) += instead of =
};
// ws / ws_bytes: optional per-tile counters that enable the split-K schedule.
int launch_linear_tc(const GemmProblem& g, void* ws, size_t ws_bytes, const DeviceInfo& dev,
                     cudaStream_t st);
size_t linear_workspace_bytes(int64_t batch, int64_t m, int64_t n);
bool linear_tc_supported(const GemmProblem& g);
int launch_linear_simt(const GemmProblem& g, cudaStream_t st);
// w_colsum of a GemmProblem on the CUDA cores (fallback path).
int launch_w_colsum_simt(const GemmProblem& g, cudaStream_t st);

// -------------------------------------------------------- row-wise kernels
size_t bias_grad_workspace(int64_t rows, int64_t n);
int launch_bias_grad(const float* dy, const int64_t s[3], float* db, int64_t batch, int64_t m,
                     int64_t n, float* ws, cudaStream_t st);
int launch_softmax_fwd(const float* x, float* y, int64_t rows, int64_t n, cudaStream_t st);
int launch_softmax_bwd(const float* p, const float* dp, float* dx, int64_t rows, int64_t n,
                       cudaStream_t st);
int launch_gelu_fwd(const float* x, float* y, int64_t numel, cudaStream_t st);
int launch_gelu_bwd(const float* x, const float* dy, float* dx, int64_t numel, cudaStream_t st);
// Widest LayerNorm row: one warp per row up to 1024 columns, one CTA per row above.
constexpr int64_t kLayerNormMaxCols = 8192;
int launch_layernorm_fwd(const float* x, const float* g, const float* b, float* y, float* mean,
                         float* rstd, int64_t rows, int64_t n, float eps, cudaStream_t st);
size_t layernorm_bwd_workspace(int64_t rows, int64_t n);
int launch_layernorm_bwd(const float* x, const float* g, const float* mean, const float* rstd,
                         const float* dy, float* dx, float* dg, float* db, int64_t rows,
                         int64_t n, float* ws, cudaStream_t st);

// Cross entropy of logit rows (loss per row; gradient written over the logits).
int launch_cross_entropy(float* x, int64_t ld, int64_t rows, int64_t vocab, const int64_t* targets,
                         int64_t ignore, float* loss_rows, cudaStream_t st);

// -------------------------------------------------- token generation (decode)
// A paged cache: [page, kv_head, slot, head_dim], unit stride along head_dim.
struct PagedKv {
  void* k;
  void* v;
  int64_t ks[3], vs[3];  // page, head, slot strides (elements)
  const int32_t* table;  // [batch, max_pages]
  int64_t table_s;
  int64_t pages, max_pages;
  int page_size;
  int dtype;  // CT_DTYPE_*
};
struct KvAppend {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // token, head, dim
  void *q_out, *k_out;
  const float *cos, *sin;
  PagedKv kv;
  const int32_t *seq_ids, *positions;
  const int32_t* rotary_positions;  // nullptr: positions
  int64_t tokens, q_heads, kv_heads, batch, max_positions;
  int head_dim, rot_dim, act_dtype;
  bool interleaved;
};
int launch_kv_append(const KvAppend& p, const DeviceInfo& dev, cudaStream_t st);
struct PagedAttention {
  const void* q;
  int64_t qs[3];  // sequence, head, dim
  PagedKv kv;
  const int32_t* seq_lens;
  void* out;
  float* lse;
  int64_t batch, q_heads, kv_heads;
  int head_dim, act_dtype;
  float scale;
  void* ws;
};
size_t paged_attention_workspace(int64_t head_dim);
int launch_paged_attention(const PagedAttention& p, const DeviceInfo& dev, cudaStream_t st);
struct LogitsProcess {
  const void* logits;
  float* out;
  int64_t ld, out_ld, rows, vocab;
  const int64_t* tokens;
  int64_t tokens_ld, max_len;
  const int32_t *lens, *prompt_lens;
  const float *repetition, *frequency, *presence;
  const int64_t* bias_ids;
  const float* bias_values;
  int64_t bias_ld, bias_values_ld, bias_n;
  const uint32_t* mask;
  int64_t mask_ld;
  int dtype;
};
int launch_logits_process(const LogitsProcess& p, const DeviceInfo& dev, cudaStream_t st);

// ------------------------------------- speculative decoding (drafted tokens)
struct TreeAttention {
  const void* q;
  int64_t qs[4];  // sequence, drafted token, head, dim
  PagedKv kv;
  const int32_t *context_lens, *draft_lens;
  const uint32_t* mask;
  int64_t ms[2];  // sequence, drafted token
  void* out;
  float* lse;
  int64_t batch, drafts, q_heads, kv_heads;
  int head_dim, act_dtype;
  float scale;
  void* ws;
};
size_t tree_attention_workspace(int64_t drafts, int64_t q_heads, int64_t kv_heads,
                                int64_t head_dim);
int launch_tree_attention(const TreeAttention& p, const DeviceInfo& dev, cudaStream_t st);
struct VerifyDrafts {
  const void *target, *draft_probs;
  int64_t ts[2], ds[2];  // sequence, node
  const int64_t* tokens;
  int64_t tokens_ld;
  const int32_t* parents;
  int64_t parents_ld;
  const int32_t* draft_lens;
  const float* uniform;
  int64_t uniform_ld;
  int64_t* new_tokens;
  int32_t *path, *counts;
  int64_t batch, drafts, vocab;
  int dtype;
};
int launch_verify_drafts(const VerifyDrafts& p, const DeviceInfo& dev, cudaStream_t st);
// Several caches of one shape, [page, kv_head, slot, head_dim]; the most that
// one launch takes.
constexpr int kMostCaches = 64;
struct CacheList {
  int n;
  void* base[kMostCaches];
  int64_t s[kMostCaches][3];  // page, head, slot strides (elements)
};
struct KvCompact {
  CacheList caches;
  const int32_t* table;
  int64_t table_s, batch, kv_heads, pages, max_pages, drafts;
  const int32_t *context_lens, *keep, *counts;
  int64_t keep_ld;
  int page_size, head_dim, dtype;
};
int launch_kv_compact(const KvCompact& p, const DeviceInfo& dev, cudaStream_t st);
struct KvCopyPages {
  CacheList caches;
  const int32_t *src, *dst;
  int64_t count, kv_heads, pages;
  int page_size, head_dim, dtype;
};
int launch_kv_copy_pages(const KvCopyPages& p, const DeviceInfo& dev, cudaStream_t st);

// ------------------------------------------------------------ watchdog
// One CTA whose waits on a barrier phase that nothing completes run out after
// the device's wait limit, followed by the kernels' abort teardown.
int launch_watchdog_selftest(const DeviceInfo& dev, cudaStream_t st);

}  // namespace ct
