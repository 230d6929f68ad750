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
//
// Bound by HBM for prompts and by latency for single tokens: every value is
// read and written once, and the loads of q, k and v do not wait for the chain
// position -> table -> page that the stores need.  A thread holds the two
// vectors whose elements pair up; its part of a head is the same for every
// head that it handles, so angles, page and slot are fetched once a thread.
//
// Device time on a B200 (floor: bytes at the 6.53 TB/s of a copy):
//   12 prompts of 300 to 4096 tokens, 32 on 32 heads of 64, FP32 into a bf16
//   cache                                      115.9 us  floor 114.6 (99 %)
//   32 on 8 of 128 in bf16, turned / not       80 / 71.5 us   69.0 / 68.7
//   7 prompts of 100 to 2000, 8 on 8 of 128, FP32, half of a head turned
//                                               23.0 us  18.6 (81 %)
//   one token each of 64 sequences, bf16         2.4 us  0.25 (the launch)
// In bf16 with angles a thread's chain (angles, page, then the stores) is what
// is left: its bytes are half and its latencies the same.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kThreads = 128;

// VEC elements as they lie in memory, in accesses of up to 16 bytes.
template <class T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
  T v[VEC];
};
template <int VEC, class T>
__device__ __forceinline__ const Pack<T, VEC>& pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
// The same as words, to hold them until they are needed.
template <class T, int VEC>
struct Raw {
  static constexpr int kWords = (int)sizeof(T) * VEC / 4 > 0 ? (int)sizeof(T) * VEC / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * VEC == 16) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x;
      w[1] = x.y;
      w[2] = x.z;
      w[3] = x.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    const uint32_t x = w[e / 2];
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float(e & 1 ? x & 0xffff0000u : x << 16);
    const __half2 h = *reinterpret_cast<const __half2*>(&x);
    return e & 1 ? __high2float(h) : __low2float(h);
  }
};
template <class T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float (&x)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC > 1) {  // two conversions an instruction
    uint32_t words[VEC / 2];
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[e], x[e + 1]);
        words[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[e], x[e + 1]);
        words[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(words[0], words[1], words[2], words[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(words[0], words[1]);
  } else {
    Pack<T, VEC> w;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w.v[e] = from_f32<T>(x[e]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = w;
  }
}

// One token a CTA (and, along y, ITEMS * kThreads parts of its heads): q heads,
// then k heads, then v heads; a head has 2^unit_shift parts of two vectors.
template <class A, class C, int VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads, 6)
    kv_append_kernel(const __grid_constant__ KvAppend p, const int unit_shift) {
  const int64_t t = blockIdx.x;
  const int item0 = blockIdx.y * (ITEMS * kThreads) + threadIdx.x;
  const int u = item0 & ((1 << unit_shift) - 1);
  const int heads = (int)(p.q_heads + 2 * p.kv_heads);

  // where the part's two vectors lie, and its first pair
  const int half = p.head_dim / 2, hr = p.rot_dim / 2, first = u * VEC;
  int a, b;
  bool turns;
  if (p.interleaved) {
    a = 2 * first;
    b = a + VEC;
    turns = a < p.rot_dim;
  } else if (first < hr) {
    a = first;
    b = a + hr;
    turns = true;
  } else {
    a = p.rot_dim + (first - hr);
    b = a + (half - hr);
    turns = false;
  }

  Raw<A, VEC> x_in[ITEMS], y_in[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int h = (item0 + i * kThreads) >> unit_shift;
    if (h >= heads) continue;
    const int kh = h - (int)p.q_heads, vh = kh - (int)p.kv_heads;
    const A* src = kh < 0   ? (const A*)p.q + t * p.qs[0] + h * p.qs[1]
                   : vh < 0 ? (const A*)p.k + t * p.ks[0] + kh * p.ks[1]
                            : (const A*)p.v + t * p.vs[0] + vh * p.vs[1];
    x_in[i].load(src + a);
    y_in[i].load(src + b);
  }

  const int pos = p.positions[t];
  const int64_t seq = p.seq_ids ? p.seq_ids[t] : t;
  // a negative position marks a padding token; one that has no place in the
  // cache (or no row in the table of angles) gives NaN
  const bool pad = pos < 0;
  // (a drafted token's angles are those of its depth in the tree, not of its slot)
  const int angle = p.rotary_positions ? p.rotary_positions[t] : pos;
  bool bad = !pad && (seq < 0 || seq >= p.batch || angle < 0 || angle >= p.max_positions);
  const bool angles = !pad && !bad && turns;
  Pack<float, VEC> cs{}, sn{};
  if (angles) {
    cs = pack<VEC>(p.cos + (int64_t)angle * hr + first);
    sn = pack<VEC>(p.sin + (int64_t)angle * hr + first);
  }
  int page = 0, slot = 0;
  if (!pad && !bad) {
    const int index = pos / p.kv.page_size;
    slot = pos - index * p.kv.page_size;
    bad = index >= p.kv.max_pages;
    if (!bad) page = p.kv.table[seq * p.kv.table_s + index];
    bad = bad || page < 0 || page >= p.kv.pages;
  }

#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int h = (item0 + i * kThreads) >> unit_shift;
    if (h >= heads) continue;
    const int kh = h - (int)p.q_heads, vh = kh - (int)p.kv_heads;
    float x[VEC], y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      x[e] = x_in[i].get(e);
      y[e] = y_in[i].get(e);
    }
    if (vh < 0) {
      if (angles) {
        if (p.interleaved && VEC > 1) {  // pairs are neighbours in x, then in y
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float(&z)[VEC] = e < VEC / 2 ? x : y;
            constexpr int kLast = VEC > 1 ? VEC - 2 : 0;
            const int j = 2 * e % VEC < kLast ? 2 * e % VEC : kLast;
            const float even = z[j], odd = z[j + (VEC > 1)];
            z[j] = even * cs.v[e] - odd * sn.v[e];
            z[j + (VEC > 1)] = odd * cs.v[e] + even * sn.v[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xe = x[e], ye = y[e];
            x[e] = xe * cs.v[e] - ye * sn.v[e];
            y[e] = ye * cs.v[e] + xe * sn.v[e];
          }
        }
      }
      A* out = kh < 0 ? (A*)p.q_out + (t * p.q_heads + h) * p.head_dim
                      : p.k_out ? (A*)p.k_out + (t * p.kv_heads + kh) * p.head_dim : nullptr;
      if (out) {
        if (pad || bad) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[e] = y[e] = bad ? NAN : 0.0f;
        }
        store_pack(out + a, x);
        store_pack(out + b, y);
      }
    }
    if (kh >= 0 && !pad && !bad) {
      C* dst = vh < 0 ? (C*)p.kv.k + page * p.kv.ks[0] + kh * p.kv.ks[1] + slot * p.kv.ks[2]
                      : (C*)p.kv.v + page * p.kv.vs[0] + vh * p.kv.vs[1] + slot * p.kv.vs[2];
      store_pack(dst + a, x);
      store_pack(dst + b, y);
    }
  }
}

// 16-byte vectors of the activations (FP32 into bf16: 115.9 us, in single
// elements 247; bf16: 80 and 312): halves of the rotated part and of the
// rest in whole vectors, all rows aligned to their vectors.  Otherwise single
// elements.
bool vectors_fit(const KvAppend& p) {
  const int act = dtype_bytes(p.act_dtype), cache = dtype_bytes(p.kv.dtype), vec = 16 / act;
  if ((p.interleaved ? p.rot_dim : p.rot_dim / 2) % (p.interleaved ? 2 * vec : vec) != 0)
    return false;
  auto fits = [&](const void* base, const int64_t* s, int n, int bytes) {
    const int align = vec * bytes < 16 ? vec * bytes : 16;
    bool ok = reinterpret_cast<uintptr_t>(base) % align == 0;
    for (int i = 0; i < n; ++i) ok = ok && s[i] * bytes % align == 0;
    return ok;
  };
  return (p.q_heads == 0 || (fits(p.q, p.qs, 2, act) && aligned16(p.q_out))) &&
         fits(p.k, p.ks, 2, act) && fits(p.v, p.vs, 2, act) && aligned16(p.k_out) &&
         fits(p.kv.k, p.kv.ks, 3, cache) && fits(p.kv.v, p.kv.vs, 3, cache) &&
         aligned16(p.cos) && aligned16(p.sin);
}

template <class A, class C, int VEC>
int launch(const KvAppend& p, const DeviceInfo& dev, cudaStream_t st) {
  int unit_shift = 0;
  while ((VEC << (unit_shift + 1)) < p.head_dim) ++unit_shift;
  const int64_t parts = (p.q_heads + 2 * p.kv_heads) << unit_shift;
  // Several parts a thread (fewer fetches of angles and pages) once every SM has
  // work for many rounds (12 prompts of 300 to 4096 tokens, FP32 into bf16: 115.9
  // us, one part a thread 135.9; in bf16, 54000 CTAs of one part, 80 and 92); one
  // part below that (7 FP32 prompts, 15000 CTAs: 23.0 us, three parts 24.4).
  const int64_t rows = (parts + kThreads - 1) / kThreads;
  int items = 1;
  if (p.tokens * rows >= (int64_t)dev.sm_count * 128)
    items = rows % 3 == 0 ? 3 : rows % 4 == 0 ? 4 : rows % 2 == 0 ? 2 : rows == 1 ? 1 : 3;
  const dim3 grid((unsigned)p.tokens, (unsigned)((rows + items - 1) / items));
  switch (items) {
    case 1: kv_append_kernel<A, C, VEC, 1><<<grid, kThreads, 0, st>>>(p, unit_shift); break;
    case 2: kv_append_kernel<A, C, VEC, 2><<<grid, kThreads, 0, st>>>(p, unit_shift); break;
    case 3: kv_append_kernel<A, C, VEC, 3><<<grid, kThreads, 0, st>>>(p, unit_shift); break;
    default: kv_append_kernel<A, C, VEC, 4><<<grid, kThreads, 0, st>>>(p, unit_shift); break;
  }
  return check_launch();
}

}  // namespace

int launch_kv_append(const KvAppend& p, const DeviceInfo& dev, cudaStream_t st) {
  const bool vectors = vectors_fit(p);
  return with_dtype(p.act_dtype, [&](auto a) {
    return with_dtype(p.kv.dtype, [&](auto c) {
      using A = decltype(a);
      using C = decltype(c);
      if constexpr (std::is_same<A, C>::value || std::is_same<A, float>::value) {
        return vectors ? launch<A, C, 16 / sizeof(A)>(p, dev, st) : launch<A, C, 1>(p, dev, st);
      } else {
        return (int)CT_ERR_INVALID_ARGUMENT;
      }
    });
  });
}

}  // namespace ct
