// kv_append.cu -- new keys and values into a paged cache, with the rotary
// position embedding applied on the way.
//
// For token t of sequence s at position p, page = block_table[s, p / S] and
// slot = p % S (S slots a page):
//   k_cache[page, h, slot] = rot(k[t, h], p),  v_cache[page, h, slot] = v[t, h]
//   q_out[t, h] = rot(q[t, h], p),             k_out[t, h] = rot(k[t, h], p)
// rot turns the pairs (a, b) of the first rot_dim elements,
//   a' = a cos - b sin,  b' = b cos + a sin,
// with cos and sin of (p, pair) from a table; the pairs are (i, i + rot_dim/2)
// or, interleaved, (2i, 2i + 1).  Formed in FP32 and rounded once.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kThreads = 256;

template <class A, class C>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const KvAppend p) {
  const int heads = (int)(p.q_heads + 2 * p.kv_heads), half = p.head_dim / 2;
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int u = (int)(item % half);
  const int64_t th = item / half;
  const int h = (int)(th % heads);
  const int64_t t = th / heads;
  if (t >= p.tokens) return;

  const int pos = p.positions[t];
  const int64_t seq = p.seq_ids ? p.seq_ids[t] : t;
  // a negative position marks a padding token; one that has no place in the
  // cache (or no row in the table of angles) gives NaN
  bool bad = pos >= 0 && (seq < 0 || seq >= p.batch || pos >= p.max_positions);
  const int hr = p.rot_dim / 2;
  int page = -1, slot = 0;
  if (pos >= 0 && !bad) {
    const int index = pos / p.kv.page_size;
    slot = pos - index * p.kv.page_size;
    bad = index >= p.kv.max_pages;
    if (!bad) page = p.kv.table[seq * p.kv.table_s + index];
    bad = bad || page < 0 || page >= p.kv.pages;
  }

  const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
  const int kh = is_q ? h : is_k ? h - (int)p.q_heads : h - (int)(p.q_heads + p.kv_heads);
  int a, b;
  if (p.interleaved) {
    a = 2 * u;
    b = a + 1;
  } else if (u < hr) {
    a = u;
    b = u + hr;
  } else {
    a = p.rot_dim + (u - hr);
    b = a + (half - hr);
  }
  const A* src = (is_q ? (const A*)p.q + t * p.qs[0] + kh * p.qs[1]
                  : is_k ? (const A*)p.k + t * p.ks[0] + kh * p.ks[1]
                         : (const A*)p.v + t * p.vs[0] + kh * p.vs[1]);
  float x = to_f32(src[a]), y = to_f32(src[b]);
  if (!is_k && !is_q) {
    if (pos >= 0 && !bad) {
      C* dst = (C*)p.kv.v + page * p.kv.vs[0] + kh * p.kv.vs[1] + slot * p.kv.vs[2];
      dst[a] = from_f32<C>(x);
      dst[b] = from_f32<C>(y);
    }
    return;
  }
  if (pos >= 0 && !bad && u < hr) {
    const float c = p.cos[(int64_t)pos * hr + u], s = p.sin[(int64_t)pos * hr + u];
    const float xr = x * c - y * s, yr = y * c + x * s;
    x = xr;
    y = yr;
  }
  if (is_k && pos >= 0 && !bad) {
    C* dst = (C*)p.kv.k + page * p.kv.ks[0] + kh * p.kv.ks[1] + slot * p.kv.ks[2];
    dst[a] = from_f32<C>(x);
    dst[b] = from_f32<C>(y);
  }
  A* out = is_q ? (A*)p.q_out : (A*)p.k_out;
  if (out) {
    if (pos < 0 || bad) x = y = bad ? NAN : 0.0f;
    out += (t * (is_q ? p.q_heads : p.kv_heads) + kh) * p.head_dim;
    out[a] = from_f32<A>(x);
    out[b] = from_f32<A>(y);
  }
}

}  // namespace

int launch_kv_append(const KvAppend& p, cudaStream_t st) {
  const int64_t items = p.tokens * (p.q_heads + 2 * p.kv_heads) * (p.head_dim / 2);
  const int64_t blocks = (items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) return CT_ERR_INVALID_ARGUMENT;
  return with_dtype(p.act_dtype, [&](auto a) {
    return with_dtype(p.kv.dtype, [&](auto c) {
      using A = decltype(a);
      using C = decltype(c);
      if constexpr (std::is_same<A, C>::value || std::is_same<A, float>::value) {
        kv_append_kernel<A, C><<<(unsigned)blocks, kThreads, 0, st>>>(p);
        return check_launch();
      } else {
        return (int)CT_ERR_INVALID_ARGUMENT;
      }
    });
  });
}

}  // namespace ct
