// tree_attention_tc.cu -- tree_attention on tcgen05: 16-bit caches with activations
// of the same type, head dims 64 and 128, more than 16 rows an item, pages of a
// multiple of 8 slots.
//
// Bounds: K and V are read once, 4 D bytes a token and head, for 4 D operations a row
// of it: up to 256 rows the bytes at 6.56 TB/s take longer than the products at 1.68
// PFLOP/s.  Beside both, a row's thread forms an exponential a key, which with many
// rows is what bounds a tile.
//
// A CTA has up to 128 rows, which are the lanes of Tensor Memory, and goes through
// its share in tiles of 64 keys: S = Q K^T (128 x 64) into one of two buffers, a
// thread a row forms the weights and writes them over S as the 16-bit operands (two
// terms) of O += P V (128 x D).  Two CTAs an SM overlap each other's latencies, and S of the
// next tile is formed while the weights of this one are.  Warps 0-3 have the rows,
// warp 4 fetches pages by TMA, warp 5 issues the products.
//
// Roundings: the weights are two terms of the cache's type for the products (16 bits
// and more) and are summed unrounded; the base of a row's exponents may lie below its
// maximum by a factor of 2^kMaxSlack, which changes no relative rounding.  One term
// would leave O with the rounding of every weight (bf16 0.0021 to 0.0024 of O where the
// output's own rounding is 0.0017), a step over one token with paged_attention would not.
//
// Measured (device): one tree of 64 on 32 and 8 heads of 128 over 131,072 tokens,
// BF16, 256 rows an item: 195 us, 2.8 TB/s, in bursts; 234 in a stream of such calls, where
// the power limit takes the clock to 1.48 GHz.  A tile of a CTA takes about 2600 cycles,
// the tensor pipe is busy 58 % of them.  With one term of the weights, 155 us, it took
// about 1850, of which the softmax needed 1400 and the issuing of products 1540; loads
// alone took 114 us, everything but the softmax 152, everything but the products 128.
// Tried then and slower, the same state 165: eight warps with the rows 189, tiles of 128
// keys with one S 201, one CTA an SM with two groups of warps that alternate 170, with
// 256 rows that share the keys 214.  64 trees of 16 over 16 to 4096 tokens: 58 us.
#include "tree_attention.cuh"

namespace ct {

using namespace tree;

namespace {

constexpr int kThreads = 192;
constexpr int kBad = 16;  // tiles on the way at most

template <class C_, int D_>
struct TcCfg {
  using C = C_;
  using A = C_;
  static constexpr int D = D_;
  static constexpr bool kBf16 = std::is_same<C, __nv_bfloat16>::value;
  static constexpr int kRows = 128;
  static constexpr int kKeys = 64;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kParts = kRowBytes / 128;  // 128-byte parts of a row
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kQBytes = kRows * kRowBytes;
  static constexpr int kUnit = kKeys * kRowBytes;  // K or V of a tile
  static constexpr int kUnits = (112 * 1024 - kQBytes) / kUnit < 12 ? (112 * 1024 - kQBytes) / kUnit : 12;
  // Two CTAs' 512 columns of Tensor Memory: O, then two buffers of S.
  static constexpr int kColumns = 256, kS = 128;
  // What an item costs beside its tiles, in tiles; units of a share at least.  2, 4,
  // 6, 9: 64 trees of 16 over 16 to 4096 tokens 61, 58, 61, 67 us, 32 of up to 33 on
  // one head 44, 43, 43, 46.
  static constexpr int kItemCost = 4;
  static constexpr int kMinShare = kItemCost + 2;
  // Tiles whose products (8 each) may pile up in Tensor Memory: the tensor core cuts
  // its sums off, by 2^-24 at most each time, so after 512 products O moves to FP32
  // sums in the workspace.
  static constexpr int kFlush = 64;
  // f16 weights reach up to 2^14 instead of 1, clear of the subnormals.
  static constexpr float kBelow = kBf16 ? 0.0f : 8.0f;
  // Tables of at most so many tokens are not split (as in tree_attention.cu).  Not
  // split / split, us: 8 sequences on 32 and 8 heads of 128, 16 drafts, 480 tokens 16.3
  // / 21.5, 750 21.3 / 22.6, 980 26.3 / 23.9.
  static constexpr int64_t kWholeTokens = 768;
  static_assert(kWholeTokens / kKeys < kFlush, "no sums in the workspace");
};

struct Bars {
  uint64_t full[12], empty[12];  // units
  uint64_t s_full[2], p_ready[2];  // of a buffer: S is there, the weights (and V) are
  uint64_t q_ready, q_free, last;  // q is there; its last product is done
  CtaCtl ctl;
  int bad[kBad];   // of a tile: a page out of range
  int skip[2];     // of a buffer: O has been formed by the rows' threads
  int raised;
  Finder finder;
};
template <class K>
constexpr int smem_bytes() {
  return K::kQBytes + K::kUnits * K::kUnit + (int)sizeof(Bars);
}

// Instruction descriptor for kind::f16, FP32 sums (bits as for kind::tf32; formats
// 0 f16, 1 bf16).
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, int m, int n, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
      "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
      "r"(idesc), "r"(accumulate)
      : "memory");
}

template <class C>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (std::is_same<C, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Two FP32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 parts(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The two terms of weights x and y (x in the low half).  Both are positive, so that an
// infinite cached value times them is that infinity, not NaN: high2 cuts off, f16 what is
// 2^-10 less (low terms of weights below 2^-14, 2^-22 of the largest, may be 0 even so),
// and low2 of bf16 takes 2^-23 of the weight on top.
template <class C>
__device__ __forceinline__ uint32_t high2(float x, float y) {
  if constexpr (std::is_same<C, __nv_bfloat16>::value) {
    return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632u);
  } else {
    constexpr float kBelowOne = 1.0f - 0x1p-10f;
    const float2 f = parts(fma2(pair(x, y), pair(kBelowOne, kBelowOne), pair(0.0f, 0.0f)));
    uint32_t w;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(f.y), "f"(f.x));
    return w;
  }
}
template <class C>
__device__ __forceinline__ uint32_t low2(float x, float y, uint32_t high) {
  float2 rest;
  if constexpr (std::is_same<C, __nv_bfloat16>::value) {
    constexpr float kAboveOne = 1.0f + 0x1p-23f;
    rest = parts(fma2(pair(x, y), pair(kAboveOne, kAboveOne),
                      pair(-__uint_as_float(high << 16), -__uint_as_float(high & 0xffff0000u))));
  } else {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&high));
    rest = parts(fma2(pair(h.x, h.y), pair(-1.0f, -1.0f), pair(x, y)));
  }
  return pack2<C>(rest.x, rest.y);
}
// Whether one of the two 16-bit values of w is not finite.
template <class C>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t kExp = std::is_same<C, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || (w >> 16 & kExp) == kExp;
}

// Byte position of 16-byte chunk c of row r in a tile of ROWS rows (128-byte parts one
// behind the other, swizzled as TMA does).
template <int ROWS>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// O += weights V of one tile without the tensor core, for the tokens that a row sees
// (fresh: O = ...).  All threads of a warp.
template <class K>
__device__ __noinline__ void add_tile(uint32_t lanes, const float* each, uint32_t sees0,
                                      uint32_t sees1, const char* v, int rows, bool fresh) {
  using C = typename K::C;
#pragma unroll 1
  for (int d = 0; d < K::D; d += 16) {
    float o[16];
    if (fresh) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0.0f;
    } else {
      tmem_ld16(lanes + d, o);
    }
#pragma unroll 1
    for (int k = 0; k < rows; ++k) {
      if (!((k < 32 ? sees0 : sees1) >> (k & 31) & 1u)) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        o[e] += each[k] * to_f32(((const C*)(v + chunk_at<K::kKeys>(k, (d + e) / 8)))[e % 8]);
    }
    __syncwarp();
    tmem_st16(lanes + d, o);
  }
}

// The rows' q into shared memory by threads 0 .. 127, where TMA does not do it (odd
// groups, strides that are no vectors, a negative scale).
template <class K>
__device__ __forceinline__ void load_rows(const Launch& a, const Cursor& c, int row0, char* shared) {
  using C = typename K::C;
  const TreeAttention& p = a.p;
  const int rows = min(K::kRows, c.drafts * a.group - row0);
  const uint32_t sign = a.negative ? 0x80008000u : 0u;
#pragma unroll 1
  for (int e = threadIdx.x; e < rows * K::kChunks; e += 128) {
    const int r = e / K::kChunks, d = e % K::kChunks * 8;
    const int i = token_of(a, row0 + r), h = c.head * a.group + (row0 + r) - i * a.group;
    const C* src = (const C*)p.q + c.b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
    const uint4 w = a.q_vectors ? *reinterpret_cast<const uint4*>(src + d)
                                : gather8(src + d * p.qs[3], p.qs[3]);
    *reinterpret_cast<uint4*>(shared + chunk_at<K::kRows>(r, d / 8)) =
        make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
  }
}

template <class K>
__global__ void __launch_bounds__(kThreads, 2)
    tree_attention_tc_kernel(const __grid_constant__ Launch a,
                             const __grid_constant__ CUtensorMap k_map,
                             const __grid_constant__ CUtensorMap v_map,
                             const __grid_constant__ CUtensorMap q_map, const int slot_rows,
                             const int q_rows) {
  using C = typename K::C;
  constexpr int D = K::D;
  extern __shared__ __align__(1024) char shared[];
  Bars& bars = *reinterpret_cast<Bars*>(shared + K::kQBytes + K::kUnits * K::kUnit);
  CtaCtl* const ctl = &bars.ctl;
  const TreeAttention& p = a.p;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int share = blockIdx.x / a.blocks, block = a.block0 + blockIdx.x % a.blocks;
  const int row0 = block * K::kRows;  // row r: token (row0 + r) / group, head (row0 + r) % group
  const uint32_t q_smem = smem_u32(shared), ring = q_smem + K::kQBytes;
  auto B = [](const uint64_t& x) { return smem_u32(&x); };
  asm volatile("griddepcontrol.launch_dependents;");
  if (tid == 0) {
    bars.raised = *reinterpret_cast<const volatile uint32_t*>(a.status) != 0u;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
    if (q_rows > 0) tma_prefetch_desc(&q_map);
    for (int u = 0; u < K::kUnits; ++u) {
      mbar_init(B(bars.full[u]), 1);
      mbar_init(B(bars.empty[u]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(B(bars.s_full[i]), 1);
      mbar_init(B(bars.p_ready[i]), 4);
    }
    mbar_init(B(bars.q_ready), q_rows > 0 ? 1 : 4);
    mbar_init(B(bars.q_free), 1);
    mbar_init(B(bars.last), 1);
    ctl->abort = 0u;
    fence_barrier_init();
    if (!a.whole) a.records[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(&ctl->tmem_base), K::kColumns);
    tmem_relinquish();
  }
  int64_t share_units, within;
  Cursor cur = first_place<K>(a, share, bars.finder, share_units, within);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  bool more = !bars.raised && enter<K>(a, cur, within, row0);
  auto next_part = [&]() {
    ++cur.head;
    more = enter<K>(a, cur, 0, row0);
  };
  auto warp_wait = [&](const uint64_t& bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar), parity, ctl, a.status));
  };
  // The units of a part of T tiles, from number u0 on, in the order of their use:
  // K_0, K_1, V_0, K_2, V_1, ...
  auto k_unit = [](uint32_t u0, int t) { return t == 0 ? u0 : u0 + 2 * t - 1; };
  auto v_unit = [](uint32_t u0, int t, int T) { return t < T - 1 ? u0 + 2 * t + 2 : u0 + 2 * T - 1; };

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    uint32_t unit = 0, tile_count = 0, part = 0;
    // boxes of a tile, tiles whose boxes' pages are looked up together; lane's box
    const int boxes = K::kKeys / a.box, batch = 32 / boxes, row = lane * a.box;
    bool ok = true;
    auto page_of = [&](int position, int& slot) {
      const int index = a.page_shift >= 0 ? position >> a.page_shift : position / p.kv.page_size;
      slot = position - index * p.kv.page_size;
      return index;
    };
    while (more && ok) {
      const int len = cur.context + cur.drafts, T = cur.stop - cur.tile;
      // The pages of 32 boxes at a time (`batch` tiles from base on, and those before).
      int base = 0, page_now = -1, slot_now = 0, page_old = -1, slot_old = 0;
      auto look_up = [&](int t0) {
        const int t = t0 + lane / boxes, position = (cur.tile + t) * K::kKeys + lane % boxes * a.box;
        const bool in = t < T && position < len;
        const int index = page_of(position, slot_now);
        page_now = in ? p.kv.table[cur.b * p.kv.table_s + index] : -1;
      };
      auto fetch = [&](int t, bool is_k) {
        const int u = unit % K::kUnits;
        const bool old = t < base;
        const int from = (t - (old ? base - batch : base)) * boxes + lane % boxes;
        const int page = __shfl_sync(0xffffffffu, old ? page_old : page_now, from);
        const int slot = __shfl_sync(0xffffffffu, old ? slot_old : slot_now, from);
        if (unit >= K::kUnits)
          ok = ok && warp_wait(bars.empty[u], (unit / K::kUnits - 1) & 1);
        if (!ok) return;
        const bool in = lane < boxes && (cur.tile + t) * K::kKeys + row < len;
        const bool fine = in && page >= 0 && page < p.kv.pages;
        const uint32_t vote = __ballot_sync(0xffffffffu, fine);
        const bool bad = __any_sync(0xffffffffu, in && !fine);
        if (lane == 0) {
          if (is_k) bars.bad[(tile_count + t) % kBad] = bad;
          mbar_arrive_expect_tx(B(bars.full[u]), __popc(vote) * a.box * K::kRowBytes);
        }
        __syncwarp();
        if (fine) {
          const CUtensorMap* map = is_k ? &k_map : &v_map;
#pragma unroll
          for (int h = 0; h < K::kParts; ++h)
            tma_load_4d(ring + u * K::kUnit + h * (K::kKeys * 128) + row * 128, map, B(bars.full[u]),
                        64 * h, slot, cur.head, page);
        }
        ++unit;
      };
      look_up(0);
      fetch(0, true);
      if (q_rows > 0) {  // q_rows rows of whole tokens, as rows (token, head) of the box
        if (part > 0) ok = ok && warp_wait(bars.q_free, (part - 1) & 1);
        if (ok && lane == 0) {
          mbar_arrive_expect_tx(B(bars.q_ready), q_rows * K::kRowBytes);
          for (int h = 0; h < K::kParts; ++h)
            tma_load_4d(q_smem + h * (K::kRows * 128), &q_map, B(bars.q_ready), 64 * h,
                        cur.head * a.group, token_of(a, row0), (int)cur.b);
        }
        ++part;
      }
      for (int t = 0; t < T && ok; ++t) {
        if (t + 1 < T) {
          if (t + 1 == base + batch) {
            page_old = page_now;
            slot_old = slot_now;
            base += batch;
            look_up(base);
          }
          fetch(t + 1, true);
        }
        fetch(t, false);
      }
      tile_count += T;
      if (ok) next_part();
    }
    if (ctl->abort)  // copies still on the way end before the memory is given back
      for (uint32_t u = unit > K::kUnits ? unit - K::kUnits : 0; u < unit; ++u)
        for (int i = 0; i < 1 << 20; ++i)
          if (mbar_test_wait(B(bars.full[u % K::kUnits]), u / K::kUnits & 1)) break;
  } else if (warp == 5) {
    // ------------------------------------------------------------ products
    // (all lanes wait: a warp of which only one does wakes later; lane 0 issues)
    {
      constexpr uint32_t kIdescS = idesc_f16(K::kBf16, 128, K::kKeys, false);
      constexpr uint32_t kIdescO = idesc_f16(K::kBf16, 128, D, true);
      uint32_t unit = 0, j = 0, part = 0;
      bool ok = true;
      while (more && ok) {
        const int T = cur.stop - cur.tile;
        auto issue_s = [&](int t) {
          const uint32_t n = k_unit(unit, t), u = n % K::kUnits, buf = (j + t) & 1;
          ok = ok && warp_wait(bars.full[u], n / K::kUnits & 1);
          if (!ok) return;
          tc_fence_after();
          if (lane != 0) return;
          const uint32_t k = ring + u * K::kUnit;
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            umma_f16_ss(tmem + K::kS + K::kKeys * buf,
                        sdesc_kmajor(q_smem + s / 4 * (K::kRows * 128) + s % 4 * 32),
                        sdesc_kmajor(k + s / 4 * (K::kKeys * 128) + s % 4 * 32), kIdescS, s > 0);
          umma_commit(B(bars.s_full[buf]));
          if (t == T - 1) umma_commit(B(bars.q_free));
        };
        ok = ok && warp_wait(bars.q_ready, part & 1);
        issue_s(0);
        for (int t = 0; t < T && ok; ++t) {
          if (t + 1 < T) issue_s(t + 1);
          const uint32_t n = v_unit(unit, t, T), u = n % K::kUnits, buf = (j + t) & 1;
          ok = ok && warp_wait(bars.p_ready[buf], (j + t) >> 1 & 1);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0 && !*(volatile int*)&bars.skip[buf]) {
            const uint32_t v = ring + u * K::kUnit;
#pragma unroll
            for (int s = 0; s < K::kKeys / 16; ++s)
#pragma unroll
              for (int term = 0; term < 2; ++term)
                umma_f16_ts(tmem, tmem + K::kS + K::kKeys * buf + K::kKeys / 2 * term + 8 * s,
                            sdesc(v + s * 2048, K::kKeys * 128, 1024, 2), kIdescO,
                            s + term > 0 || t % K::kFlush != 0);
          }
          if (lane == 0) umma_commit(B(bars.empty[u]));
          __syncwarp();
        }
        unit += 2 * T;
        j += T;
        ++part;
        if (ok) next_part();
      }
      if (lane == 0) umma_commit(B(bars.last));
      __syncwarp();
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(B(bars.last), 0))
        if (globaltimer_ns() - t0 > CT_WAIT_TIMEOUT_NS) break;
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ rows
    const float c2 = a.c2;
    const uint32_t lanes = tmem_addr(tmem, 32 * warp, 0);
    uint32_t unit = 0, j = 0;
    bool ok = true;
    auto arrive = [&](const uint64_t& bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar));
    };
    // weights V of the part's tile t is in O (its V is free then; the rows' threads may
    // be two products behind: the parity of a barrier a buffer would not tell)
    auto product_done = [&](int t, int T) {
      const uint32_t n = v_unit(unit, t, T);
      return warp_wait(bars.empty[n % K::kUnits], n / K::kUnits & 1);
    };
    uint2 kept = make_uint2(0u, 0u);  // the row's mask
    auto load_q = [&]() {
      const int i = token_of(a, row0 + tid);
      kept = make_uint2(mask_word(p, cur.b, i, 0), mask_word(p, cur.b, i, 1));
      if (q_rows > 0) return;  // TMA does it
      load_rows<K>(a, cur, row0, shared);
      fence_proxy_async_smem();
      arrive(bars.q_ready);
    };
    if (more) load_q();
    while (more && ok) {
      const int64_t b = cur.b;
      const int head = cur.head, context = cur.context, drafts = cur.drafts;
      const int part0 = cur.tile, tiles = cur.tiles, T = cur.stop - cur.tile;
      const int r = row0 + tid, i = token_of(a, r);
      const bool active = row0 + 32 * warp < drafts * a.group, there = i < drafts;
      float* const slot = a.partials + ((int64_t)blockIdx.x * 2 + (part0 == 0 ? 1 : 0)) *
                                           partial_floats(slot_rows, D);
      float base = -INFINITY, sum = 0.0f, flushed = 0.0f;
      bool has_flushed = false;
      for (int t = 0; t < T && ok; ++t, ++j) {
        const uint32_t buf = j & 1;
        const bool fresh = t % K::kFlush == 0;  // O holds nothing yet
        if (!(ok = warp_wait(bars.s_full[buf], j >> 1 & 1))) break;
        if (tid == 0) mbar_arrive(B(bars.empty[k_unit(unit, t) % K::kUnits]));  // K has been read
        if (!active) {
          arrive(bars.p_ready[buf]);
          continue;
        }
        tc_fence_after();
        if (bars.bad[j % kBad]) sum = NAN;
        float s[2][32];
        tmem_ld32(lanes + K::kS + K::kKeys * buf, s[0]);
        tmem_ld32(lanes + K::kS + K::kKeys * buf + 32, s[1]);
        const int position = (part0 + t) * K::kKeys;
        const bool masked = position + K::kKeys > context;
        uint32_t sees[2] = {~0u, ~0u};
        if (masked) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sees[h] = seen_from(p, kept, b, i, position + 32 * h - context, drafts);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(sees[h] >> e & 1u)) s[h][e] = -INFINITY;
          }
        }
        float tops[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
        for (int e = 0; e < 32; ++e) tops[e % 4] = max3(tops[e % 4], s[0][e], s[1][e]);
        float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
        top = top * c2 - K::kBelow;
        if (__any_sync(0xffffffffu, top > base + kMaxSlack)) {
          const float old = base;
          // (a row's own scores decide: lanes without a row hold anything)
          base = top > old + kMaxSlack ? top : old;
          const float f = old == -INFINITY ? 0.0f : ex2(old - base);
          sum = old == -INFINITY ? sum : sum * f;
          if (!fresh) {
            if (!(ok = product_done(t - 1, T))) break;
            tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              float o[32];
              tmem_ld32(lanes + d, o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] *= f;
              tmem_st32(lanes + d, o);
            }
          }
        }
        const float from = base == -INFINITY ? 0.0f : base;
        float w[32];
        const uint64_t factor = pair(c2, c2), shift = pair(-from, -from);
        uint64_t part_sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 z = parts(fma2(pair(s[e / 16][e % 16 * 2], s[e / 16][e % 16 * 2 + 1]), factor, shift));
          const float x = ex2(z.x), y = ex2(z.y);
          part_sum[e % 4] = add2(part_sum[e % 4], pair(x, y));
          s[e / 16][e % 16 * 2] = x;
          s[e / 16][e % 16 * 2 + 1] = y;
          w[e] = __uint_as_float(high2<C>(x, y));
        }
        const float2 both = parts(add2(add2(part_sum[0], part_sum[1]), add2(part_sum[2], part_sum[3])));
        sum += both.x + both.y;
        tmem_st32(lanes + K::kS + K::kKeys * buf, w);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          w[e] = __uint_as_float(low2<C>(s[e / 16][e % 16 * 2], s[e / 16][e % 16 * 2 + 1],
                                         __float_as_uint(w[e])));
        tmem_st32(lanes + K::kS + K::kKeys * buf + 32, w);
        bool dirty = false;
        if (masked) {
          // V behind the last token counts as zero (a weight of 0 would leave its
          // NaN); values that are not finite reach the rows that see their token only
          const uint32_t n = v_unit(unit, t, T), u = n % K::kUnits;
          if (!(ok = warp_wait(bars.full[u], n / K::kUnits & 1))) break;
          char* const v = shared + K::kQBytes + u * K::kUnit;
          const int rows = min(K::kKeys, context + drafts - position);
          const int zeroers = min(4, (drafts * a.group - row0 + 31) / 32);  // active warps
          for (int e = rows * K::kChunks + tid; e < K::kKeys * K::kChunks; e += 32 * zeroers)
            *reinterpret_cast<uint4*>(v + chunk_at<K::kKeys>(e / K::kChunks, e % K::kChunks)) =
                make_uint4(0u, 0u, 0u, 0u);
          for (int e = max(0, context - position) * K::kChunks + lane; e < rows * K::kChunks; e += 32) {
            const uint4 x = *reinterpret_cast<const uint4*>(
                v + chunk_at<K::kKeys>(e / K::kChunks, e % K::kChunks));
            dirty = dirty || not_finite<C>(x.x) || not_finite<C>(x.y) || not_finite<C>(x.z) ||
                    not_finite<C>(x.w);
          }
          fence_proxy_async_smem();
          dirty = __any_sync(0xffffffffu, dirty);
          if (dirty) {  // (rare) the tile's O without the tensor core
            if (!fresh && !(ok = product_done(t - 1, T))) break;
            tc_fence_after();
            float each[K::kKeys];
#pragma unroll
            for (int e = 0; e < K::kKeys; ++e) each[e] = s[e / 32][e % 32];
            add_tile<K>(lanes, each, sees[0], sees[1], v, rows, fresh);
          }
        }
        if (warp == 0 && !masked) {  // (the issuing thread waits for the weights only)
          const uint32_t n = v_unit(unit, t, T);
          if (!(ok = warp_wait(bars.full[n % K::kUnits], n / K::kUnits & 1))) break;
        }
        if (lane == 0) *(volatile int*)&bars.skip[buf] = dirty;
        tmem_wait_st();
        tc_fence_before();
        arrive(bars.p_ready[buf]);
        if ((t + 1) % K::kFlush == 0 && t + 1 < T) {
          // O moves to FP32 sums in this part's slot
          if (!(ok = product_done(t, T))) break;
          tc_fence_after();
          const float f = has_flushed && flushed > -INFINITY ? ex2(flushed - base) : 0.0f;
#pragma unroll 1
          for (int d = 0; d < D; d += 32) {
            float o[32];
            tmem_ld32(lanes + d, o);
            if (there) {
              float4* const at = reinterpret_cast<float4*>(slot + tid * D + d);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float4 x = has_flushed ? at[e] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                x.x = x.x * f + o[4 * e];
                x.y = x.y * f + o[4 * e + 1];
                x.z = x.z * f + o[4 * e + 2];
                x.w = x.w * f + o[4 * e + 3];
                at[e] = x;
              }
            }
            __syncwarp();
          }
          flushed = base;
          has_flushed = true;
        }
      }
      if (!ok) break;
      // the next part's q (S of the last tile is there: q has been read)
      next_part();
      if (more) load_q();
      if (!(ok = product_done(T - 1, T))) break;
      unit += 2 * T;
      tc_fence_after();
      const bool whole = part0 == 0 && T == tiles;
      if (active) {
        const float f = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
        const float g = has_flushed && flushed > -INFINITY ? ex2(flushed - base) : 0.0f;
        const int64_t row = (b * p.drafts + i) * p.q_heads + head * a.group + r - i * a.group;
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          float o[32];
          tmem_ld32(lanes + d, o);
          if (there) {
            float4* const at = reinterpret_cast<float4*>(slot + tid * D + d);
            if (has_flushed) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 x = at[e];
                o[4 * e] += x.x * g;
                o[4 * e + 1] += x.y * g;
                o[4 * e + 2] += x.z * g;
                o[4 * e + 3] += x.w * g;
              }
            }
            if (whole) {
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                *reinterpret_cast<uint4*>((C*)p.out + row * D + d + e) =
                    make_uint4(pack2<C>(o[e] * f, o[e + 1] * f), pack2<C>(o[e + 2] * f, o[e + 3] * f),
                               pack2<C>(o[e + 4] * f, o[e + 5] * f), pack2<C>(o[e + 6] * f, o[e + 7] * f));
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                at[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
          __syncwarp();
        }
        if (there && whole && p.lse)
          p.lse[row] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * kLn2;
        if (there && !whole)
          *reinterpret_cast<float2*>(slot + slot_rows * D + 2 * tid) = make_float2(base, sum);
      }
      tc_fence_before();
      if (!whole && part0 == 0 && tid == 0) {
        // the item ends in the share that has its last unit
        const int64_t end = (int64_t)(share + 1) * share_units + (tiles - T);
        a.records[blockIdx.x] = make_int4((int)((end - 1) / share_units) - share + 1, (int)b, head, drafts);
      }
    }
  }
  __syncwarp();
  if (!bars.raised && a.block0 == 0) write_rows_not_there<K>(p);
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, K::kColumns);
  }
}

template <class K>
int launch(Launch a, const DeviceInfo& dev, cudaStream_t st) {
  const TreeAttention& p = a.p;
  static_assert(smem_bytes<K>() <= 113 * 1024, "two CTAs an SM");
  int rc = allow_shared<tree_attention_tc_kernel<K>>(smem_bytes<K>(), dev);
  if (rc != CT_OK) return rc;
  const int64_t rows = p.drafts * a.group, items = p.batch * p.kv_heads;
  const int blocks = (int)((rows + K::kRows - 1) / K::kRows);
  int ctas = 2 * dev.sm_count;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  a.whole = p.kv.max_pages * p.kv.page_size <= K::kWholeTokens;
  CUtensorMap k_map{}, v_map{};
  make_maps(a, &k_map, &v_map, K::kKeys);
  if (a.box == 0) return kNoTc;
  // q by TMA where a block's rows are whole tokens
  CUtensorMap q_map{};
  int q_rows = blocks == 1 ? (int)rows : K::kRows % a.group == 0 ? K::kRows : 0;
  if (!a.q_vectors || a.negative || q_rows == 0 ||
      make_tmap_pages(&q_map, p.q, p.act_dtype, p.batch, p.drafts, p.q_heads, K::D, p.qs, a.group,
                      q_rows / a.group) != CT_OK)
    q_rows = 0;
  const int slot_rows = rows >= K::kRows ? K::kRows : (int)(rows + 15) / 16 * 16;
  // a part of the blocks a launch where they are more than half the CTAs of a wave (a
  // piece of a prompt, 4096 tokens over 4096, 32 and 8 heads of 128: 1.70 ms; all by the
  // warps of tree_attention.cu 5.02)
  const int launches = a.whole ? 1 : (blocks + ctas / 2 - 1) / (ctas / 2);
  a.blocks = (blocks + launches - 1) / launches;
  const int64_t shares = a.whole ? items : ctas / a.blocks;
  if (shares * a.blocks >= 1ll << 31) return CT_ERR_INVALID_ARGUMENT;
  a.shares = (int)shares;
  for (a.block0 = 0; a.block0 < blocks; a.block0 += a.blocks) {
    const unsigned grid = (unsigned)(shares * a.blocks);
    tree_attention_tc_kernel<K><<<grid, kThreads, smem_bytes<K>(), st>>>(a, k_map, v_map, q_map,
                                                                        slot_rows, q_rows);
    rc = check_launch();
    if (rc == CT_OK && !a.whole) rc = launch_join<typename K::A, K::D>(a, grid, slot_rows, dev, st);
    if (rc != CT_OK) return rc;
  }
  return CT_OK;
}

}  // namespace

namespace tree {

// From 17 rows on: below, the products on half-empty tiles lose to those of the warps
// (tree_attention.cu), or gain little.  Warps / here, us, 32 sequences of 2048 tokens, 32 and 8 heads:
// of 128, 16 rows 61 / 58, 24 96 / 60, 64 140 / 65; of 64, 16 rows 38 / 47, 24 51 / 47.
int launch_tc(const TreeAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  const int64_t rows = p.drafts * (p.q_heads / p.kv_heads);
  if (p.act_dtype != p.kv.dtype || p.kv.dtype == CT_DTYPE_F32 || p.head_dim == 32 || rows <= 16 ||
      p.kv.page_size % 8 != 0)
    return kNoTc;
  const Launch a = begin_launch(p, dev);
  if (p.kv.dtype == CT_DTYPE_BF16)
    return p.head_dim == 64 ? launch<TcCfg<__nv_bfloat16, 64>>(a, dev, st)
                            : launch<TcCfg<__nv_bfloat16, 128>>(a, dev, st);
  return p.head_dim == 64 ? launch<TcCfg<__half, 64>>(a, dev, st)
                          : launch<TcCfg<__half, 128>>(a, dev, st);
}

}  // namespace tree
}  // namespace ct
