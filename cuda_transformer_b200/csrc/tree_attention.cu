// tree_attention.cu -- attention of several new tokens per sequence (a draft: a
// tree or a chain of tokens) over a paged key/value cache that holds them too:
//   s_ij = scale q_i . k_j over the tokens j before the draft and the drafted
//   ones that i's mask names,  O_i = sum_j softmax(s_i)_j v_j,
//   L_i = ln sum_j exp(s_ij);  O = 0 and L = -inf for rows that see nothing.
// A warp works on one row, a lane on every 32nd dim.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kThreads = 128;

template <class A, class C, int D>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const __grid_constant__ TreeAttention p) {
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= p.batch * p.drafts * p.q_heads) return;
  const int h = (int)(row % p.q_heads);
  const int64_t i = row / p.q_heads % p.drafts, b = row / p.q_heads / p.drafts;
  const int64_t kh = h / (p.q_heads / p.kv_heads);
  constexpr int N = D / 32;
  float q[N], o[N] = {};
  for (int e = 0; e < N; ++e)
    q[e] = to_f32(((const A*)p.q)[b * p.qs[0] + i * p.qs[1] + h * p.qs[2] + (lane + 32 * e) * p.qs[3]]) * p.scale;
  int64_t n = p.draft_lens ? p.draft_lens[b] : p.drafts;
  n = n < 0 ? 0 : n > p.drafts ? p.drafts : n;
  const int64_t context = p.context_lens[b];
  bool bad = context + n > p.kv.max_pages * p.kv.page_size;
  float m = -INFINITY, l = 0.0f;
  if (context >= 0 && i < n && !bad) {
    for (int64_t j = 0; j < context + n; ++j) {
      const int page = p.kv.table[b * p.kv.table_s + j / p.kv.page_size];
      if (page < 0 || page >= p.kv.pages) {
        bad = true;
        break;
      }
      const int64_t d = j - context;
      if (d >= 0 && !(p.mask ? p.mask[b * p.ms[0] + i * p.ms[1] + d / 32] >> (d % 32) & 1u : d <= i)) continue;
      const int64_t slot = j % p.kv.page_size;
      const C* k = (const C*)p.kv.k + page * p.kv.ks[0] + kh * p.kv.ks[1] + slot * p.kv.ks[2];
      const C* v = (const C*)p.kv.v + page * p.kv.vs[0] + kh * p.kv.vs[1] + slot * p.kv.vs[2];
      float s = 0.0f;
      for (int e = 0; e < N; ++e) s += q[e] * to_f32(k[lane + 32 * e]);
      for (int w = 16; w; w /= 2) s += __shfl_xor_sync(0xffffffffu, s, w);
      if (s == -INFINITY) continue;
      const float top = fmaxf(m, s), f = m == -INFINITY ? 0.0f : expf(m - top), w = expf(s - top);
      l = l * f + w;
      for (int e = 0; e < N; ++e) o[e] = o[e] * f + w * to_f32(v[lane + 32 * e]);
      m = top;
    }
  }
  const bool there = context >= 0 && i < n;
  for (int e = 0; e < N; ++e)
    ((A*)p.out)[row * D + lane + 32 * e] = from_f32<A>(there && bad ? NAN : l == 0.0f ? 0.0f : o[e] / l);
  if (lane == 0 && p.lse) p.lse[row] = there && bad ? NAN : l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t tree_attention_workspace(int64_t, int64_t, int64_t, int64_t) { return 0; }

int launch_tree_attention(const TreeAttention& p, const DeviceInfo&, cudaStream_t st) {
  return with_dtype(p.act_dtype, [&](auto a) {
    return with_dtype(p.kv.dtype, [&](auto c) {
      using A = decltype(a);
      using C = decltype(c);
      if constexpr (std::is_same<A, C>::value || std::is_same<A, float>::value) {
        const int64_t rows = p.batch * p.drafts * p.q_heads;
        const unsigned grid = (unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32));
        if (p.head_dim == 32) tree_attention_kernel<A, C, 32><<<grid, kThreads, 0, st>>>(p);
        else if (p.head_dim == 64) tree_attention_kernel<A, C, 64><<<grid, kThreads, 0, st>>>(p);
        else tree_attention_kernel<A, C, 128><<<grid, kThreads, 0, st>>>(p);
        return check_launch();
      } else {
        return (int)CT_ERR_INVALID_ARGUMENT;
      }
    });
  });
}

}  // namespace ct
