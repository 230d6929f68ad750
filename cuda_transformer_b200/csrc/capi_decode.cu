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

// Sizes of a list of caches that are only moved about: any head size (status,
// no CUDA call).
int check_sizes(int64_t caches_n, int64_t kv_heads, int64_t head_dim, int64_t pages,
                int64_t page_size, int cache) {
  const bool ok = in_range(caches_n, 0) && in_range(kv_heads, 1) && kv_heads <= 65536 &&
                  in_range(head_dim, 1) && head_dim <= 65536 && in_range(pages, 0) &&
                  in_range(page_size, 1) && page_size <= kMaxTokens &&
                  kv_heads * head_dim < kLim && valid_types(cache, cache);
  return ok ? CT_OK : CT_ERR_INVALID_ARGUMENT;
}

// Calls `launch` for the caches, as many at a time as a launch takes.  All are
// checked before the first; distinct: one that is there twice is refused.
template <class P, class F>
int for_caches(P& p, void* const* caches, const int64_t* strides, int64_t n, int64_t kv_heads,
               int64_t head_dim, int64_t pages, int64_t page_size, bool distinct, F&& launch) {
  const int64_t sizes[3] = {pages, kv_heads, page_size};
  for (int64_t c = 0; c < n; ++c) {
    if (pages > 0 && !caches[c]) return CT_ERR_INVALID_ARGUMENT;
    if (head_dim > 1 && strides[4 * c + 3] != 1) return CT_ERR_UNSUPPORTED_LAYOUT;
    for (int i = 0; i < 3; ++i)
      if (stride_of(sizes[i], strides[4 * c + i]) < 0) return CT_ERR_UNSUPPORTED_LAYOUT;
  }
  if (pages == 0) return CT_OK;  // no place to read or write
  for (int64_t c = 1; distinct && c < n; ++c)
    for (int64_t d = 0; d < c; ++d)
      if (caches[c] == caches[d]) return CT_ERR_INVALID_ARGUMENT;
  int rc = CT_OK;
  const DeviceInfo* dev = current_device(&rc);
  for (int64_t c = 0; c < n && rc == CT_OK; c += kMostCaches) {
    p.caches.n = (int)(n - c < kMostCaches ? n - c : kMostCaches);
    for (int j = 0; j < p.caches.n; ++j) {
      p.caches.base[j] = caches[c + j];
      for (int i = 0; i < 3; ++i)
        p.caches.s[j][i] = stride_of(sizes[i], strides[4 * (c + j) + i]);
    }
    rc = launch(*dev);
  }
  return rc;
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
  return ct_kv_append_ex(q, q_stride, k, k_stride, v, v_stride, q_out, k_out, cos, sin, k_cache,
                         kc_stride, v_cache, vc_stride, block_table, table_stride, seq_ids,
                         positions, nullptr, tokens, q_heads, kv_heads, head_dim, rot_dim,
                         interleaved, max_positions, batch, pages, page_size, max_pages, act_dtype,
                         cache_dtype, stream);
}

int ct_kv_append_ex(const void* q, const int64_t q_stride[3], const void* k,
                    const int64_t k_stride[3], const void* v, const int64_t v_stride[3],
                    void* q_out, void* k_out, const float* cos, const float* sin, void* k_cache,
                    const int64_t kc_stride[4], void* v_cache, const int64_t vc_stride[4],
                    const int32_t* block_table, int64_t table_stride, const int32_t* seq_ids,
                    const int32_t* positions, const int32_t* rotary_positions, int64_t tokens,
                    int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t rot_dim,
                    int interleaved, int64_t max_positions, int64_t batch, int64_t pages,
                    int64_t page_size, int64_t max_pages, int act_dtype, int cache_dtype,
                    void* stream) {
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
  // (without a rotation they are not looked at)
  p.rotary_positions = rot_dim > 0 ? rotary_positions : nullptr;
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

size_t ct_tree_attention_workspace_size(int64_t drafts, int64_t q_heads, int64_t kv_heads,
                                        int64_t head_dim) {
  if (!in_range(drafts, 0) || !in_range(q_heads, 0) || !in_range(kv_heads, 1) ||
      q_heads % kv_heads != 0 || !in_range(head_dim, 1))
    return 0;
  return tree_attention_workspace(drafts, q_heads, kv_heads, head_dim);
}

int ct_tree_attention(const void* q, const int64_t q_stride[4], const void* k_cache,
                      const int64_t kc_stride[4], const void* v_cache, const int64_t vc_stride[4],
                      const int32_t* block_table, int64_t table_stride,
                      const int32_t* context_lens, const int32_t* draft_lens, const int32_t* mask,
                      const int64_t mask_stride[2], void* out, float* lse, int64_t batch,
                      int64_t drafts, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                      int64_t pages, int64_t page_size, int64_t max_pages, float scale,
                      int act_dtype, int cache_dtype, void* workspace, size_t workspace_bytes,
                      void* stream) {
  int rc = check_cache(batch, q_heads, kv_heads, head_dim, pages, page_size, max_pages, act_dtype,
                       cache_dtype);
  if (rc != CT_OK) return rc;
  // (each product is formed of bounded factors: no overflow)
  if (q_heads % kv_heads != 0 || !in_range(drafts, 0) || drafts > CT_TREE_ATTENTION_MAX_DRAFTS ||
      q_heads > 65536 || batch * q_heads >= kLim || batch * q_heads * drafts >= kLim ||
      batch * q_heads * drafts * (max_pages * page_size / 8 + 16) >= kMaxTiles)
    return CT_ERR_INVALID_ARGUMENT;
  if (batch * q_heads * drafts == 0) return CT_OK;
  if (!q || !q_stride || !context_lens || !out || !aligned16(out) || (mask && !mask_stride))
    return CT_ERR_INVALID_ARGUMENT;
  TreeAttention p{};
  rc = fill_cache(&p.kv, k_cache, kc_stride, v_cache, vc_stride, block_table, table_stride, batch,
                  kv_heads, pages, page_size, max_pages, cache_dtype);
  if (rc != CT_OK) return rc;
  const int64_t align = 16 / dtype_bytes(cache_dtype);
  bool ok = aligned16(k_cache) && aligned16(v_cache);
  for (int i = 0; i < 3; ++i) ok = ok && p.kv.ks[i] % align == 0 && p.kv.vs[i] % align == 0;
  if (!ok) return CT_ERR_UNSUPPORTED_LAYOUT;
  if (workspace_bytes < tree_attention_workspace(drafts, q_heads, kv_heads, head_dim) ||
      (workspace_bytes > 0 && !workspace))
    return CT_ERR_WORKSPACE_TOO_SMALL;
  if (!aligned16(workspace)) return CT_ERR_INVALID_ARGUMENT;
  p.q = q;
  p.qs[0] = stride_of(batch, q_stride[0]);
  p.qs[1] = stride_of(drafts, q_stride[1]);
  p.qs[2] = stride_of(q_heads, q_stride[2]);
  p.qs[3] = q_stride[3];
  p.context_lens = context_lens;
  p.draft_lens = draft_lens;
  p.mask = reinterpret_cast<const uint32_t*>(mask);
  if (mask) {
    p.ms[0] = stride_of(batch, mask_stride[0]);
    p.ms[1] = stride_of(drafts, mask_stride[1]);
  }
  p.out = out;
  p.lse = lse;
  p.batch = batch;
  p.drafts = drafts;
  p.q_heads = q_heads;
  p.kv_heads = kv_heads;
  p.head_dim = (int)head_dim;
  p.act_dtype = act_dtype;
  p.scale = scale;
  p.ws = workspace;
  const DeviceInfo* dev = current_device(&rc);
  if (rc != CT_OK) return rc;
  return launch_tree_attention(p, *dev, reinterpret_cast<cudaStream_t>(stream));
}

int ct_verify_drafts(const void* target, const int64_t target_stride[2], const void* draft_probs,
                     const int64_t draft_stride[2], int dtype, const int64_t* tokens,
                     int64_t tokens_ld, const int32_t* parents, int64_t parents_ld,
                     const int32_t* draft_lens, const float* uniform, int64_t uniform_ld,
                     int64_t* new_tokens, int32_t* path, int32_t* counts, int64_t batch,
                     int64_t drafts, int64_t vocab, void* stream) {
  if (!in_range(batch, 0) || !in_range(drafts, 1) || drafts > CT_VERIFY_DRAFTS_MAX ||
      !in_range(vocab, 1) || vocab >= kLim / 2 ||
      !(dtype == CT_DTYPE_F32 || dtype == CT_DTYPE_BF16 || dtype == CT_DTYPE_F16) ||
      tokens_ld < 0 || (parents && parents_ld < 0) || (uniform && uniform_ld < 0) ||
      (draft_probs && (!uniform || !draft_stride)))
    return CT_ERR_INVALID_ARGUMENT;
  if (batch == 0) return CT_OK;
  if (!target || !target_stride || !tokens || !new_tokens || !path || !counts)
    return CT_ERR_INVALID_ARGUMENT;
  VerifyDrafts p{};
  p.target = target;
  p.draft_probs = draft_probs;
  p.ts[0] = stride_of(batch, target_stride[0]);
  p.ts[1] = stride_of(drafts, target_stride[1]);
  if (draft_probs) {
    p.ds[0] = stride_of(batch, draft_stride[0]);
    p.ds[1] = stride_of(drafts, draft_stride[1]);
  }
  if (p.ts[0] < 0 || p.ts[1] < 0 || p.ds[0] < 0 || p.ds[1] < 0) return CT_ERR_UNSUPPORTED_LAYOUT;
  p.tokens = tokens;
  p.tokens_ld = tokens_ld;
  p.parents = parents;
  p.parents_ld = parents_ld;
  p.draft_lens = draft_lens;
  p.uniform = uniform;
  p.uniform_ld = uniform_ld;
  p.new_tokens = new_tokens;
  p.path = path;
  p.counts = counts;
  p.batch = batch;
  p.drafts = drafts;
  p.vocab = vocab;
  p.dtype = dtype;
  int rc = CT_OK;
  const DeviceInfo* dev = current_device(&rc);
  if (rc != CT_OK) return rc;
  return launch_verify_drafts(p, *dev, reinterpret_cast<cudaStream_t>(stream));
}

int ct_kv_compact(void* const* caches, const int64_t* cache_strides, int64_t caches_n,
                  const int32_t* block_table, int64_t table_stride, const int32_t* context_lens,
                  const int32_t* keep, int64_t keep_ld, const int32_t* counts, int64_t batch,
                  int64_t drafts, int64_t kv_heads, int64_t head_dim, int64_t pages,
                  int64_t page_size, int64_t max_pages, int cache_dtype, void* stream) {
  int rc = check_sizes(caches_n, kv_heads, head_dim, pages, page_size, cache_dtype);
  if (rc != CT_OK) return rc;
  if (!in_range(batch, 0) || !in_range(max_pages, 0) || max_pages * page_size > kMaxTokens ||
      !in_range(drafts, 0) || keep_ld < 0)
    return CT_ERR_INVALID_ARGUMENT;
  if (caches_n == 0 || batch == 0 || drafts == 0) return CT_OK;
  if (!caches || !cache_strides || !context_lens || !keep || !counts || (max_pages > 0 && !block_table))
    return CT_ERR_INVALID_ARGUMENT;
  KvCompact p{};
  p.table = block_table;
  p.table_s = table_stride;
  p.batch = batch;
  p.kv_heads = kv_heads;
  p.pages = pages;
  p.max_pages = max_pages;
  p.drafts = drafts;
  p.context_lens = context_lens;
  p.keep = keep;
  p.keep_ld = keep_ld;
  p.counts = counts;
  p.page_size = (int)page_size;
  p.head_dim = (int)head_dim;
  p.dtype = cache_dtype;
  // (what is there twice would be moved twice, by threads that do not wait for each other)
  return for_caches(p, caches, cache_strides, caches_n, kv_heads, head_dim, pages, page_size, true,
                    [&](const DeviceInfo& dev) {
                      return launch_kv_compact(p, dev, reinterpret_cast<cudaStream_t>(stream));
                    });
}

int ct_kv_copy_pages(void* const* caches, const int64_t* cache_strides, int64_t caches_n,
                     const int32_t* src, const int32_t* dst, int64_t count, int64_t kv_heads,
                     int64_t head_dim, int64_t pages, int64_t page_size, int cache_dtype,
                     void* stream) {
  int rc = check_sizes(caches_n, kv_heads, head_dim, pages, page_size, cache_dtype);
  if (rc != CT_OK) return rc;
  if (!in_range(count, 0)) return CT_ERR_INVALID_ARGUMENT;
  if (caches_n == 0 || count == 0) return CT_OK;
  if (!caches || !cache_strides || !src || !dst) return CT_ERR_INVALID_ARGUMENT;
  KvCopyPages p{};
  p.src = src;
  p.dst = dst;
  p.count = count;
  p.kv_heads = kv_heads;
  p.pages = pages;
  p.page_size = (int)page_size;
  p.head_dim = (int)head_dim;
  p.dtype = cache_dtype;
  return for_caches(p, caches, cache_strides, caches_n, kv_heads, head_dim, pages, page_size, false,
                    [&](const DeviceInfo& dev) {
                      return launch_kv_copy_pages(p, dev, reinterpret_cast<cudaStream_t>(stream));
                    });
}

}  // extern "C"
