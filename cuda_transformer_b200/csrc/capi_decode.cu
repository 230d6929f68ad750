// capi_decode.cu -- the extern "C" entry points of the token-generation
// operators: argument validation and dispatch to the kernel launchers.
#include "decode_common.cuh"

using namespace ct;

namespace {

constexpr int64_t kLim = 1ll << 31;
// longest sequence: the tiles of 32 are counted in 32 bits
constexpr int64_t kMaxTokens = (1ll << 30) - 256;

// tiles (of 8 keys at least) of all items, with 16 for each item's ends: times
// the CTAs, fewer than 2^9, they stay below 2^62
constexpr int64_t kMaxTiles = 1ll << 52;

bool in_range(int64_t v, int64_t low) { return v >= low && v < kLim; }

bool valid_types(int act, int cache) {
  return (cache == CT_DTYPE_F32 || cache == CT_DTYPE_BF16 || cache == CT_DTYPE_F16) &&
         (act == cache || act == CT_DTYPE_F32);
}

// Sizes of a paged cache (status, no CUDA call).
int check_cache(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t pages,
                int64_t page_size, int64_t max_pages, int act, int cache) {
  if (!in_range(batch, 0) || !in_range(q_heads, 0) || !in_range(kv_heads, 1) ||
      !in_range(pages, 0) || !in_range(page_size, 1) || !in_range(max_pages, 0) ||
      max_pages * page_size > kMaxTokens || !valid_types(act, cache))
    return CT_ERR_INVALID_ARGUMENT;
  if (!(head_dim == 32 || head_dim == 64 || head_dim == 128)) return CT_ERR_UNSUPPORTED_HEAD_DIM;
  return CT_OK;
}

// The stride of a dimension of `size` elements: that of a single one says
// nothing (imported tensors have any value there).
int64_t stride_of(int64_t size, int64_t stride) { return size > 1 ? stride : 0; }

int fill_cache(PagedKv* kv, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
               const int32_t* table, int64_t table_s, int64_t batch, int64_t kv_heads,
               int64_t pages, int64_t page_size, int64_t max_pages, int dtype) {
  if (!ks || !vs || (pages > 0 && (!k || !v)) || (batch > 0 && max_pages > 0 && !table))
    return CT_ERR_INVALID_ARGUMENT;
  if (ks[3] != 1 || vs[3] != 1) return CT_ERR_UNSUPPORTED_LAYOUT;
  const int64_t sizes[3] = {pages, kv_heads, page_size};
  kv->k = const_cast<void*>(k);
  kv->v = const_cast<void*>(v);
  for (int i = 0; i < 3; ++i) {
    kv->ks[i] = stride_of(sizes[i], ks[i]);
    kv->vs[i] = stride_of(sizes[i], vs[i]);
    if (kv->ks[i] < 0 || kv->vs[i] < 0) return CT_ERR_UNSUPPORTED_LAYOUT;
  }
  kv->table = table;
  kv->table_s = table_s;
  kv->pages = pages;
  kv->max_pages = max_pages;
  kv->page_size = (int)page_size;
  kv->dtype = dtype;
  return CT_OK;
}

}  // namespace

extern "C" {

int ct_kv_append(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                 const void* v, const int64_t v_stride[3], void* q_out, void* k_out,
                 const float* cos, const float* sin, void* k_cache, const int64_t kc_stride[4],
                 void* v_cache, const int64_t vc_stride[4], const int32_t* block_table,
                 int64_t table_stride, const int32_t* seq_ids, const int32_t* positions,
                 int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                 int64_t rot_dim, int interleaved, int64_t max_positions, int64_t batch,
                 int64_t pages, int64_t page_size, int64_t max_pages, int act_dtype,
                 int cache_dtype, void* stream) {
  int rc = check_cache(batch, q_heads, kv_heads, head_dim, pages, page_size, max_pages, act_dtype,
                       cache_dtype);
  if (rc != CT_OK) return rc;
  if (!in_range(tokens, 0) || q_heads + 2 * kv_heads > 65536 || rot_dim < 0 || rot_dim % 2 != 0 ||
      rot_dim > head_dim || (rot_dim > 0 && max_positions < 0) || (q_heads > 0 && !q_stride) ||
      !k_stride || !v_stride)
    return CT_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return CT_OK;
  if (!k || !v || !positions || (q_heads > 0 && (!q || !q_out)) ||
      (rot_dim > 0 && max_positions > 0 && (!cos || !sin)))
    return CT_ERR_INVALID_ARGUMENT;
  KvAppend p{};
  rc = fill_cache(&p.kv, k_cache, kc_stride, v_cache, vc_stride, block_table, table_stride, batch,
                  kv_heads, pages, page_size, max_pages, cache_dtype);
  if (rc != CT_OK) return rc;
  p.q = q;
  p.k = k;
  p.v = v;
  for (int i = 0; i < 3; ++i) {
    const int64_t size = i == 0 ? tokens : i == 1 ? kv_heads : head_dim;
    p.qs[i] = q_heads > 0 ? stride_of(i == 1 ? q_heads : size, q_stride[i]) : 0;
    p.ks[i] = stride_of(size, k_stride[i]);
    p.vs[i] = stride_of(size, v_stride[i]);
  }
  if ((q_heads > 0 && p.qs[2] != 1) || p.ks[2] != 1 || p.vs[2] != 1)
    return CT_ERR_UNSUPPORTED_LAYOUT;
  p.q_out = q_out;
  p.k_out = k_out;
  p.cos = cos;
  p.sin = sin;
  p.seq_ids = seq_ids;
  p.positions = positions;
  p.tokens = tokens;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.batch = batch;
  p.max_positions = rot_dim > 0 ? max_positions : kLim;
  p.head_dim = (int)head_dim;
  p.rot_dim = (int)rot_dim;
  p.act_dtype = act_dtype;
  p.interleaved = interleaved != 0;
  const DeviceInfo* dev = current_device(&rc);
  if (rc != CT_OK) return rc;
  return launch_kv_append(p, *dev, reinterpret_cast<cudaStream_t>(stream));
}

size_t ct_paged_attention_workspace_size(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  if (!in_range(q_heads, 0) || !in_range(kv_heads, 1) || !in_range(head_dim, 1)) return 0;
  return paged_attention_workspace(head_dim);
}

int ct_paged_attention(const void* q, const int64_t q_stride[3], const void* k_cache,
                       const int64_t kc_stride[4], const void* v_cache, const int64_t vc_stride[4],
                       const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens,
                       void* out, float* lse, int64_t batch, int64_t q_heads, int64_t kv_heads,
                       int64_t head_dim, int64_t pages, int64_t page_size, int64_t max_pages,
                       float scale, int act_dtype, int cache_dtype, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int rc = check_cache(batch, q_heads, kv_heads, head_dim, pages, page_size, max_pages, act_dtype,
                       cache_dtype);
  if (rc != CT_OK) return rc;
  if (q_heads % kv_heads != 0 || batch * q_heads >= kLim ||
      batch * q_heads * (max_pages * page_size / 8 + 16) >= kMaxTiles)
    return CT_ERR_INVALID_ARGUMENT;
  if (batch * q_heads == 0) return CT_OK;
  if (!q || !q_stride || !seq_lens || !out || !aligned16(out)) return CT_ERR_INVALID_ARGUMENT;
  PagedAttention p{};
  rc = fill_cache(&p.kv, k_cache, kc_stride, v_cache, vc_stride, block_table, table_stride, batch,
                  kv_heads, pages, page_size, max_pages, cache_dtype);
  if (rc != CT_OK) return rc;
  const int64_t align = 16 / dtype_bytes(cache_dtype);
  bool ok = aligned16(k_cache) && aligned16(v_cache);
  for (int i = 0; i < 3; ++i) ok = ok && p.kv.ks[i] % align == 0 && p.kv.vs[i] % align == 0;
  if (!ok) return CT_ERR_UNSUPPORTED_LAYOUT;
  if (workspace_bytes < paged_attention_workspace(head_dim) ||
      (workspace_bytes > 0 && !workspace))
    return CT_ERR_WORKSPACE_TOO_SMALL;
  if (!aligned16(workspace)) return CT_ERR_INVALID_ARGUMENT;
  p.q = q;
  p.qs[0] = stride_of(batch, q_stride[0]);
  p.qs[1] = stride_of(q_heads, q_stride[1]);
  p.qs[2] = q_stride[2];
  p.seq_lens = seq_lens;
  p.out = out;
  p.lse = lse;
  p.batch = batch;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.head_dim = (int)head_dim;
  p.act_dtype = act_dtype;
  p.scale = scale;
  p.ws = workspace;
  const DeviceInfo* dev = current_device(&rc);
  if (rc != CT_OK) return rc;
  return launch_paged_attention(p, *dev, reinterpret_cast<cudaStream_t>(stream));
}

int ct_logits_process(const void* logits, int64_t ld, int dtype, float* out, int64_t out_ld,
                      int64_t rows, int64_t vocab, const int64_t* tokens, int64_t tokens_ld,
                      int64_t max_len, const int32_t* lens, const int32_t* prompt_lens,
                      const float* repetition, const float* frequency, const float* presence,
                      const int64_t* bias_ids, int64_t bias_ids_ld, const float* bias_values,
                      int64_t bias_values_ld, int64_t bias_n, const int32_t* mask, int64_t mask_ld,
                      void* stream) {
  if (!in_range(rows, 0) || !in_range(vocab, 1) || ld < vocab || out_ld < vocab ||
      !(dtype == CT_DTYPE_F32 || dtype == CT_DTYPE_BF16 || dtype == CT_DTYPE_F16) ||
      (tokens && (!in_range(max_len, 0) || tokens_ld < 0)) || !in_range(bias_n, 0) ||
      (bias_n > 0 && (!bias_ids || !bias_values || bias_ids_ld < 0 || bias_values_ld < 0)) ||
      (mask && mask_ld < 0))
    return CT_ERR_INVALID_ARGUMENT;
  if (rows == 0) return CT_OK;
  if (!logits || !out || (logits == out && (dtype != CT_DTYPE_F32 || ld != out_ld)))
    return CT_ERR_INVALID_ARGUMENT;
  LogitsProcess p{};
  p.logits = logits;
  p.out = out;
  p.ld = ld;
  p.out_ld = out_ld;
  p.rows = rows;
  p.vocab = vocab;
  p.tokens = tokens;
  p.tokens_ld = tokens_ld;
  p.max_len = max_len;
  p.lens = lens;
  p.prompt_lens = prompt_lens;
  p.repetition = repetition;
  p.frequency = frequency;
  p.presence = presence;
  p.bias_ids = bias_ids;
  p.bias_values = bias_values;
  p.bias_ld = bias_ids_ld;
  p.bias_values_ld = bias_values_ld;
  p.bias_n = bias_n;
  p.mask = reinterpret_cast<const uint32_t*>(mask);
  p.mask_ld = mask_ld;
  p.dtype = dtype;
  int rc = CT_OK;
  const DeviceInfo* dev = current_device(&rc);
  if (rc != CT_OK) return rc;
  return launch_logits_process(p, *dev, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
