// paged_attention.cu -- attention of one new token per sequence over a paged
// key/value cache:
//   s_j = scale q . k_j,  O = sum_j softmax(s)_j v_j,  L = ln sum_j exp(s_j)
// over the sequence's cached tokens j; O = 0 and L = -inf when there are none.
// Query heads share key/value heads in groups of q_heads / kv_heads.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kWarps = 8;

// One CTA per (sequence, query head): each warp takes every eighth key with a
// running maximum and sum, and the warps are joined at the end.
template <class A, class C, int D>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_kernel(const PagedAttention p) {
  constexpr int E = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t b = blockIdx.x / p.q_heads, h = blockIdx.x % p.q_heads;
  const int64_t kh = h / (p.q_heads / p.kv_heads);
  const int64_t capacity = p.kv.max_pages * p.kv.page_size;
  const int len = p.seq_lens[b];
  bool bad = len > capacity;
  const int n = bad ? 0 : len;
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = to_f32(((const A*)p.q)[b * p.qs[0] + h * p.qs[1] + (e * 32 + lane) * p.qs[2]]);
    o[e] = 0.0f;
  }
  for (int j = w; j < n; j += kWarps) {
    const int index = j / p.kv.page_size, slot = j - index * p.kv.page_size;
    const int page = p.kv.table[b * p.kv.table_s + index];
    if (page < 0 || page >= p.kv.pages) {
      bad = true;
      break;
    }
    const C* k = (const C*)p.kv.k + page * p.kv.ks[0] + kh * p.kv.ks[1] + slot * p.kv.ks[2];
    const C* v = (const C*)p.kv.v + page * p.kv.vs[0] + kh * p.kv.vs[1] + slot * p.kv.vs[2];
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f32(k[e * 32 + lane]), s);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= p.scale;
    const float mn = fmaxf(m, s), c = m == mn ? 1.0f : expf(m - mn), pr = expf(s - mn);
    m = mn;
    l = l * c + pr;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(pr, to_f32(v[e * 32 + lane]), o[e] * c);
  }
  if (bad) l = NAN;
  if (lane == 0) {
    sm[w] = m;
    sl[w] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[w][e * 32 + lane] = o[e];
  __syncthreads();
  float mt = -INFINITY, lt = 0.0f;
  for (int i = 0; i < kWarps; ++i) mt = fmaxf(mt, sm[i]);
  for (int i = 0; i < kWarps; ++i) lt += sl[i] * (sm[i] == -INFINITY ? 1.0f : expf(sm[i] - mt));
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float x = 0.0f;
    for (int i = 0; i < kWarps; ++i)
      x += sm[i] == -INFINITY ? 0.0f : so[i][d] * expf(sm[i] - mt);
    ((A*)p.out)[(b * p.q_heads + h) * D + d] = from_f32<A>(lt == 0.0f ? 0.0f : x / lt);
  }
  if (p.lse && threadIdx.x == 0) p.lse[b * p.q_heads + h] = lt != lt ? lt : mt + logf(lt);
}

}  // namespace

size_t paged_attention_workspace(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  (void)q_heads;
  (void)kv_heads;
  (void)head_dim;
  return 256;  // no scratch yet: the interface's smallest workspace
}

int launch_paged_attention(const PagedAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  (void)dev;
  const unsigned blocks = (unsigned)(p.batch * p.q_heads);
  return with_dtype(p.act_dtype, [&](auto a) {
    return with_dtype(p.kv.dtype, [&](auto c) {
      using A = decltype(a);
      using C = decltype(c);
      if constexpr (std::is_same<A, C>::value || std::is_same<A, float>::value) {
        if (p.head_dim == 32)
          paged_attention_kernel<A, C, 32><<<blocks, kWarps * 32, 0, st>>>(p);
        else if (p.head_dim == 64)
          paged_attention_kernel<A, C, 64><<<blocks, kWarps * 32, 0, st>>>(p);
        else
          paged_attention_kernel<A, C, 128><<<blocks, kWarps * 32, 0, st>>>(p);
        return check_launch();
      } else {
        return (int)CT_ERR_INVALID_ARGUMENT;
      }
    });
  });
}

}  // namespace ct
