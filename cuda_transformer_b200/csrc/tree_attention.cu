// tree_attention.cu -- attention of several new tokens per sequence (a draft: a
// tree or a chain of tokens) over a paged key/value cache that holds them too:
//   s_ij = scale q_i . k_j over the tokens j before the draft and the drafted
//   ones that i's mask names,  O_i = sum_j softmax(s_i)_j v_j,
//   L_i = ln sum_j exp(s_ij);  O = 0 and L = -inf for rows that see nothing.
// The rows of a (sequence, key/value head) are its drafted tokens times the
// query heads that share the head.
//
// Here all that tree_attention_tc.cu does not take: FP32 activations or caches, head
// dim 32, up to 16 rows, odd pages.  Bound by HBM for few rows (K and V are read once,
// the products cost next to nothing) and by mma.sync for many with FP32 activations,
// which need several products for one.
//
// Four warps.  A warp has 16 rows (8, or 32) and the groups of warps that cover an
// item's rows take turns at the tiles, each with a ring of its own that its lanes fill
// by TMA (by copies of 16 bytes where pages have no box) and that needs no barrier of
// the CTA; their sums meet at the item's end.  Scores stay in registers: the result
// layout of Q K^T is the operand's of P V.
//
// Roundings: FP32 activations over 16-bit caches are split into 16-bit terms, three
// for BF16 and two for f16 (22 bits and more; a row of q is brought into f16's range by
// a power of two first, as in paged_attention), and so are the weights; FP32 caches run
// as two TF32 terms each way (22 bits).  16-bit activations: the weights in two terms of
// that type (16 bits and more), as in paged_attention; they are summed unrounded.
//
// Measured (device): 16 chains of up to 5 on 32 heads of 64 with FP32 activations over a
// BF16 cache of 3500 to 4096 tokens: 90 us, 5.5 TB/s of K and V; with a product a term
// instead of two terms a product, two CTAs an SM, 114.  FP32 on FP32, 8 sequences of 2000
// tokens on 32 and 8 heads of 128, 8, 32 and 128 rows: 39, 73 and 240 us for 20 us of
// bytes (three products for one; the tensor pipe is busy 41 % of the last).  8 trees of 8 on 6 heads of 64 over
// up to 248 tokens, FP32: 12.5 us, of which the launch and one pass through the
// latencies are most.
#include <cfloat>

#include "tree_attention.cuh"

namespace ct {

using namespace tree;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// C: the cache's type; F32ACT: q and out are FP32, else of type C; MT: 16-row tiles
// of a warp, 0 for 8 rows; WR: warps along the rows, a group.  The groups take turns
// at the tiles.  With 8 rows two terms of q and of the weights share a product, in
// rows 0-7 and 8-15, whose sums then sit in the same lane.
template <class C_, bool F32ACT_, int D_, int MT_, int WR_>
struct Cfg {
  static constexpr bool kPack = MT_ == 0;
  using C = C_;
  static constexpr bool F32ACT = F32ACT_;
  static constexpr int D = D_, MT = kPack ? 1 : MT_, WR = WR_;
  static constexpr int kH = kPack ? 1 : 2;  // rows of a lane in a 16-row tile
  using A = std::conditional_t<F32ACT, float, C>;
  static constexpr bool kF32 = sizeof(C) == 4;
  static constexpr bool kBf16 = std::is_same<C, __nv_bfloat16>::value;
  static constexpr int kRows = kPack ? 8 : 16 * MT * WR;
  static constexpr int kCtas = kPack ? 3 : 2;  // of an SM
  static constexpr int WK = kWarps / WR;  // groups
  static constexpr int kRowBytes = D * (int)sizeof(C);
  static constexpr int kChunks = kRowBytes / 16;
  // Keys of a tile: 8 KB of K and as many of V (4 KB where four groups have a ring
  // each), 128 at most.
  static constexpr int kHalf = WK == 4 ? 4096 : 8192;
  static constexpr int kKeys = kHalf / kRowBytes < 128 ? kHalf / kRowBytes : 128;
  // Keys that a warp's scores are formed of at a time.
  static constexpr int kMost = (F32ACT || MT > 1) && D == 128 ? 16 : 32;
  static constexpr int kBlock = kKeys < kMost ? kKeys : kMost;
  static constexpr int NT = kBlock / 8;
  static constexpr int kTileBytes = kKeys * kRowBytes;  // K or V
  // 16-bit terms of q and of the weights (FP32 activations: 22 bits and more).
  static constexpr int kTerms = kF32 || !F32ACT ? 1 : kBf16 ? 3 : 2;
  static constexpr int kWTerms = kF32 ? 1 : F32ACT ? kTerms : 2;
  // Rows of q have factors of their own (load_rows).
  static constexpr bool kRowScale = F32ACT && !kF32 && !kBf16;
  // All terms of the weights are positive (take_weights).
  static constexpr bool kPositive = !kRowScale;
  // (packed: pairs of terms, 16 rows each)
  static constexpr int kQTiles = kPack ? (kTerms + 1) / 2 : kTerms;
  static constexpr int kWTiles = kPack ? (kWTerms + 1) / 2 : kWTerms;
  static constexpr int kQRows = kPack && !kF32 ? 16 : kRows;
  static constexpr int kQBytes = kQTiles * kQRows * kRowBytes;
  static constexpr int kJoinDims = 32;
  static constexpr int kJoinBytes = WK > 1 ? (WK - 1) * kRows * kJoinDims * 4 : 0;
  static constexpr int kStatBytes = WK > 1 ? 2 * WK * kRows * 4 : 0;
  static constexpr int kHeadBytes =
      ((kQBytes > kJoinBytes + kStatBytes ? kQBytes : kJoinBytes + kStatBytes) + 1023) / 1024 * 1024;
  // Stages of a group's ring: kCtas CTAs an SM (228 KB, of which each takes 1 KB and
  // the static 1 KB; 1 KB more to begin at a whole one).
  static constexpr int kFit = ((kPack ? 72 : 110) * 1024 - kHeadBytes) / (2 * kTileBytes) / WK;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static_assert(kStages >= 1 && kStages * WK >= 3, "tiles on the way");
  static constexpr int kSmem = 1024 + kHeadBytes + WK * kStages * 2 * kTileBytes;
  // What an item (a sequence and a key/value head) costs beside its tiles (q, the
  // end), in tiles; units of a share at least.  (Tiles of 8 KB; costs of 4, 8, 12 and
  // 20 of them: the chains above 114, 114, 116, 120 us, 64 trees of 16 on 32 and 8
  // heads of 128, then here, 150, 123, 107, 120.)
  static constexpr int kItemCost = 16384 / kHalf * 6;
  static constexpr int kMinShare = kItemCost + 2 * WK;
  // Tables of at most so many tokens are not split (an item a CTA, and no join): the
  // longer, the cheaper a token.  Not split / split, us: 8 sequences of 750 tokens on
  // 32 and 8 heads of 128, BF16, 4 drafts 21.0 / 23.1, of 980 25.6 / 23.5; FP32, 8
  // drafts on 6 heads of 64, 480 tokens 15.8 / 21.8, 980 26.1 / 24.0; 64 drafts, 300
  // tokens 38 / 44, 600 64 / 58.
  static constexpr int64_t kWholeTokens = !F32ACT ? 768 : kF32 && !kPack ? 256 : 512;
  // f16 weights reach up to 2^14 instead of 1, clear of the subnormals.
  static constexpr float kBelow = !kF32 && !kBf16 ? 8.0f : 0.0f;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// Arrives on `bar` when this thread's copies so far are done.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// c += A B for one tile: 16 x 8 x 8 in TF32, 16 x 8 x 16 in the 16-bit types.
template <class C>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(C) == 4)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if constexpr (std::is_same<C, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c = A B.
template <class C>
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (sizeof(C) == 4)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else if constexpr (std::is_same<C, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <class C>
__device__ __forceinline__ void mma_next(bool first, float (&c)[4], const uint32_t (&a)[4],
                                         uint32_t b0, uint32_t b1) {
  if (first) mma_first<C>(c, a, b0, b1); else mma<C>(c, a, b0, b1);
}
// What is left of x beside the TF32 value that the tensor core makes of it (it
// drops the 13 low bits), rounded to nearest once it drops its own (without the half
// step errors all point one way: 1.2e-6 of O, with it 7e-7).  An infinity leaves -0:
// inf - inf is 0x7fffffff, which the half step turns over.
__device__ __forceinline__ uint32_t low_tf32(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u)) + 0x1000u;
}
// Infinite cached values.  Terms of a weight that share a sum are positive, all of them
// (those of a weight of 0 are 0), so that an infinite value times them is that infinity,
// not NaN.  Where low terms may be 0 or negative (f16 with FP32 activations) they have a
// sum of their own, which counts where the first terms' is finite.
__device__ __forceinline__ float positive_rest(float x, float high) {
  return fmaxf(x - high, fminf(x, FLT_MIN));
}
__device__ __forceinline__ uint32_t low_weight(uint32_t x) {
  return __float_as_uint(positive_rest(__uint_as_float(x), __uint_as_float(x & 0xffffe000u))) + 0x1000u;
}
__device__ __forceinline__ float with_rest(float first, float rest) {
  return fabsf(first) < INFINITY ? first + rest : first;
}
// The next 16-bit term of x and y (x in the low half); x and y keep the rest.
template <class C>
__device__ __forceinline__ uint32_t take_term(float& x, float& y) {
  uint32_t w;
  if constexpr (std::is_same<C, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    w = *reinterpret_cast<const uint32_t*>(&h);
    x -= __uint_as_float(w << 16);
    y -= __uint_as_float(w & 0xffff0000u);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    w = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    x -= f.x;
    y -= f.y;
  }
  return w;
}
// The next term of weights x and y, of which `left` follow: positive where K::kPositive
// says so.  It is cut off then, f16's from 2^-10 less (what follows is 0 all the same
// for weights below 2^-14, 2^-22 of the largest; 21 bits).
template <class K>
__device__ __forceinline__ uint32_t take_weights(float& x, float& y, int left) {
  using C = typename K::C;
  if (!K::kPositive || left == 0) return take_term<C>(x, y);
  uint32_t w;
  if constexpr (K::kBf16) {
    w = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632u);
    x = positive_rest(x, __uint_as_float(w << 16));
    y = positive_rest(y, __uint_as_float(w & 0xffff0000u));
  } else {
    constexpr float kBelowOne = 1.0f - 0x1p-10f;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y * kBelowOne), "f"(x * kBelowOne));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x -= f.x;
    y -= f.y;
  }
  return w;
}
template <class C>
__device__ __forceinline__ float half_value(uint32_t w, int e) {
  if constexpr (std::is_same<C, __nv_bfloat16>::value)
    return __uint_as_float(e ? w & 0xffff0000u : w << 16);
  else
    return e ? __high2float(*reinterpret_cast<const __half2*>(&w))
             : __low2float(*reinterpret_cast<const __half2*>(&w));
}
// A word of V (one FP32 or two 16-bit values) with what is not finite as 0.
template <class C>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
  if constexpr (sizeof(C) == 4) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  constexpr uint32_t kExp = std::is_same<C, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  if ((w & kExp) == kExp) w &= 0xffff0000u;
  if ((w >> 16 & kExp) == kExp) w &= 0xffffu;
  return w;
}

// Byte position of 16-byte chunk c of row r in a tile of `ROWS` rows: parts of 128
// bytes of all rows one behind the other, chunks permuted so that eight rows' meet
// different banks (as TMA writes them with a swizzle of 128 bytes, of 64 for
// shorter rows).
template <int ROW_BYTES, int ROWS>
__device__ __forceinline__ uint32_t chunk_pos(int r, int c) {
  if constexpr (ROW_BYTES >= 128)
    return (uint32_t)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
  return (uint32_t)(r * ROW_BYTES + ((c ^ (r >> 1 & 3)) << 4));  // 64-byte rows
}

// A part's q into shared memory: rows of 16-byte chunks as the cache's type, or its
// terms one behind the other; and the rows' first mask words.  f16 terms hold the row
// times a power of two that brings its largest element to 2^14 .. 2^15, so that large
// ones do not overflow and what falls below f16's range is below 2^-38 of the largest;
// row_scale is what undoes it.
template <class K>
__device__ __forceinline__ void load_rows(const Launch& a, const Cursor& c, int row0, char* shared,
                                       uint2* mask_words, float* row_scale) {
  using C = typename K::C;
  using A = typename K::A;
  constexpr int D = K::D, kEight = D / 8;
  const TreeAttention& p = a.p;
  const int tid = threadIdx.x, head = c.head, drafts = c.drafts;
  const int64_t b = c.b;
  for (int r = tid; r < K::kRows; r += kThreads) {
    const int i = token_of(a, row0 + r);
    mask_words[r] = make_uint2(mask_word(p, b, i, 0), mask_word(p, b, i, 1));
  }
  constexpr int kPieces = K::kRows * kEight;
  constexpr int kBatch = kPieces / kThreads < 1 ? 1 : kPieces / kThreads < 4 ? kPieces / kThreads : 4;
  constexpr int kWords = sizeof(A) == 2 ? 1 : 2;
  for (int e0 = tid; e0 < kPieces; e0 += kBatch * kThreads) {
    uint4 in[kBatch][kWords];  // 8 elements
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = (e0 + k * kThreads) / kEight, d = (e0 + k * kThreads) % kEight * 8;
      const int i = token_of(a, row0 + r), h = head * a.group + (row0 + r) - i * a.group;
      const A* src = (const A*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2];
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        in[k][w] = make_uint4(0u, 0u, 0u, 0u);
        if (i < drafts) {
          if (a.q_vectors) {
            in[k][w] = reinterpret_cast<const uint4*>(src + d)[w];
          } else {
            in[k][w] = gather8(src + (d + w * 4) * p.qs[3], p.qs[3]);
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = (e0 + k * kThreads) / kEight, d = (e0 + k * kThreads) % kEight * 8;
      if constexpr (sizeof(A) == 2) {
        const uint32_t sign = a.negative ? 0x80008000u : 0u;
        const uint4 w = in[k][0];
        *reinterpret_cast<uint4*>(shared + chunk_pos<K::kRowBytes, K::kQRows>(r, d / 8)) =
            make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
      } else {
        float x[8];
        *reinterpret_cast<uint4*>(x) = in[k][0];
        *reinterpret_cast<uint4*>(x + 4) = in[k][kWords - 1];
#pragma unroll
        for (int y = 0; y < 8; ++y) x[y] = a.negative ? -x[y] : x[y];
        if constexpr (K::kRowScale) {  // (kEight lanes side by side have a row)
          float top = 0.0f;
#pragma unroll
          for (int y = 0; y < 8; ++y)
            if (fabsf(x[y]) < INFINITY) top = fmaxf(top, fabsf(x[y]));
#pragma unroll
          for (int w = 1; w < kEight; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          int power = 15;
          frexpf(top, &power);
          power = top == 0.0f ? 0 : 15 - power < 120 ? 15 - power : 120;  // 2^+-power are normal
#pragma unroll
          for (int y = 0; y < 8; ++y) x[y] *= __int_as_float((127 + power) << 23);
          if (d == 0) row_scale[r] = __int_as_float((127 - power) << 23);
        }
        if constexpr (K::kF32) {
          *reinterpret_cast<float4*>(shared + chunk_pos<K::kRowBytes, K::kRows>(r, d / 4)) =
              *reinterpret_cast<float4*>(x);
          *reinterpret_cast<float4*>(shared + chunk_pos<K::kRowBytes, K::kRows>(r, d / 4 + 1)) =
              *reinterpret_cast<float4*>(x + 4);
        } else {
#pragma unroll
          for (int t = 0; t < K::kTerms; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = take_term<C>(x[2 * j], x[2 * j + 1]);
            *reinterpret_cast<uint4*>(
                shared + (K::kPack ? t / 2 : t) * K::kQRows * K::kRowBytes +
                chunk_pos<K::kRowBytes, K::kQRows>(K::kPack ? r + t % 2 * 8 : r, d / 8)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
}

// A tile, chunk by chunk (pages that TMA boxes do not fit); whether a page of this
// lane's is out of range.
template <class K>
__device__ __forceinline__ bool copy_chunks(const Launch& a, const Cursor& next, uint32_t k_tile) {
  using C = typename K::C;
  const TreeAttention& p = a.p;
  const int lane = threadIdx.x % 32, len = next.context + next.drafts, from = next.tile * K::kKeys;
  const uint32_t v_tile = k_tile + K::kTileBytes;
  auto page_of = [&](int position, int& slot) {
    const int index = a.page_shift >= 0 ? position >> a.page_shift : position / p.kv.page_size;
    slot = position - index * p.kv.page_size;
    return index;
  };
  const int chunk = lane % K::kChunks;
  const C* kh = (const C*)p.kv.k + next.head * p.kv.ks[1] + chunk * (16 / (int)sizeof(C));
  const C* vh = (const C*)p.kv.v + next.head * p.kv.vs[1] + chunk * (16 / (int)sizeof(C));
  bool bad = false;
#pragma unroll 4
  for (int i = 0; i < K::kKeys * K::kChunks / 32; ++i) {
    const int row = i * (32 / K::kChunks) + lane / K::kChunks;
    int slot;
    const int index = page_of(from + row, slot);
    const bool in = from + row < len;
    const int64_t page = in ? p.kv.table[next.b * p.kv.table_s + index] : -1;
    const bool fine = in && page >= 0 && page < p.kv.pages;
    bad = bad || (in && !fine);
    const uint32_t at = chunk_pos<K::kRowBytes, K::kKeys>(row, chunk);
    // (nothing is read where there is no page)
    const void* k = fine ? (const void*)(kh + page * p.kv.ks[0] + slot * p.kv.ks[2]) : p.out;
    const void* v = fine ? (const void*)(vh + page * p.kv.vs[0] + slot * p.kv.vs[2]) : p.out;
    cp_async16(k_tile + at, k, fine ? 16 : 0);
    cp_async16(v_tile + at, v, fine ? 16 : 0);
  }
  return bad;
}

template <class K>
__global__ void __launch_bounds__(kThreads, K::kCtas)
    tree_attention_kernel(const __grid_constant__ Launch a, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map) {
  using C = typename K::C;
  using A = typename K::A;
  constexpr int D = K::D, MT = K::MT, NT = K::NT;
  extern __shared__ char shared_base[];
  char* const shared = shared_base + (-smem_u32(shared_base) & 1023u);
  // (the join's buffers lie where q was)
  float(*const stat)[K::WK][K::kRows] =
      reinterpret_cast<float(*)[K::WK][K::kRows]>(shared + K::kJoinBytes);
  __shared__ Finder finder;
  __shared__ uint2 mask_words[K::kRows];
  __shared__ float row_scale[K::kRowScale ? K::kRows : 1];
  __shared__ alignas(8) uint64_t full[K::WK][K::kStages], empty[K::WK][K::kStages];
  __shared__ int stage_bad[K::WK][K::kStages];
  __shared__ CtaCtl ctl;
  __shared__ bool raised;
  const TreeAttention& p = a.p;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int wr = warp % K::WR, wk = warp / K::WR;  // row part, group
  const int share = blockIdx.x / a.blocks, block = blockIdx.x % a.blocks;
  const uint32_t q_smem = smem_u32(shared);
  const uint32_t ring = q_smem + K::kHeadBytes + wk * (K::kStages * 2 * K::kTileBytes);
  asm volatile("griddepcontrol.launch_dependents;");
  if (a.box && warp == 0) {
    if (lane == 0) tma_prefetch_desc(&k_map);
    if (lane == 1) tma_prefetch_desc(&v_map);
  }
  if (tid == 0) {
    raised = *reinterpret_cast<const volatile uint32_t*>(a.status) != 0u;
    ctl.abort = 0u;
    for (int g = 0; g < K::WK; ++g)
      for (int s = 0; s < K::kStages; ++s) {
        mbar_init(smem_u32(&full[g][s]), a.box ? 1 : 33);
        mbar_init(smem_u32(&empty[g][s]), K::WR);
      }
    fence_barrier_init();
    if (!a.whole) a.records[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  __syncthreads();
  if (raised) return;

  // ---- this CTA's share of the units
  int64_t share_units, within;
  Cursor next = first_place<K>(a, share, finder, share_units, within);
  const int row0 = block * K::kRows;  // row r: token (row0 + r) / group, head (row0 + r) % group
  bool more = enter<K>(a, next, within, row0);
  Cursor cur = next;

  // ---- copies: the group's first warp fetches the tiles that are its group's, as
  // many ahead as there are stages
  const bool leader = wr == 0;
  int page_next = -1;  // of lane's box of `next`'s tile
  uint32_t in_count = 0, out_count = 0;
  auto page_of = [&](int position, int& slot) {
    const int index = a.page_shift >= 0 ? position >> a.page_shift : position / p.kv.page_size;
    slot = position - index * p.kv.page_size;
    return index;
  };
  auto look_up = [&]() {
    const int len = next.context + next.drafts, from = next.tile * K::kKeys, row = lane * a.box;
    int slot;
    page_next = row < K::kKeys && from + row < len
                    ? p.kv.table[next.b * p.kv.table_s + page_of(from + row, slot)] : -1;
  };
  // `next` goes to the group's tile at or behind it
  bool more_in = more;
  auto to_own_tile = [&]() {
    while (more_in && next.tile >= next.stop) {
      ++next.head;
      more_in = enter<K>(a, next, 0, row0);
      next.tile += wk;
    }
    if (more_in && a.box) look_up();
  };
  auto copy_in = [&]() {
    const int stage = in_count % K::kStages;
    if (K::WR > 1 && in_count >= K::kStages)
      mbar_wait(smem_u32(&empty[wk][stage]), (in_count / K::kStages - 1) & 1, &ctl, a.status);
    __syncwarp();
    const int len = next.context + next.drafts, from = next.tile * K::kKeys;
    const uint32_t k_tile = ring + stage * 2 * K::kTileBytes, v_tile = k_tile + K::kTileBytes;
    const uint32_t bar = smem_u32(&full[wk][stage]);
    if (a.box) {
      const int row = lane * a.box;
      const bool in = row < K::kKeys && from + row < len;
      const bool fine = in && page_next >= 0 && page_next < p.kv.pages;
      const uint32_t vote = __ballot_sync(0xffffffffu, fine);
      const bool bad = __any_sync(0xffffffffu, in && !fine);
      if (lane == 0) {
        stage_bad[wk][stage] = bad;
        mbar_arrive_expect_tx(bar, __popc(vote) * a.box * 2 * K::kRowBytes);
      }
      __syncwarp();
      if (fine) {
        int slot;
        page_of(from + row, slot);
        constexpr int kPart = K::kRowBytes < 128 ? K::kRowBytes : 128;
#pragma unroll
        for (int h = 0; h < K::kRowBytes / kPart; ++h) {
          const uint32_t at = h * (K::kKeys * kPart) + row * kPart;
          const int dim = h * (kPart / (int)sizeof(C));
          tma_load_4d(k_tile + at, &k_map, bar, dim, slot, next.head, page_next);
          tma_load_4d(v_tile + at, &v_map, bar, dim, slot, next.head, page_next);
        }
      }
    } else {
      const bool bad = __any_sync(0xffffffffu, copy_chunks<K>(a, next, k_tile));
      if (lane == 0) {
        stage_bad[wk][stage] = bad;
        mbar_arrive(bar);
      }
      cp_async_arrive(bar);
    }
    ++in_count;
    next.tile += K::WK;
    to_own_tile();
  };
  if (leader) {
    next.tile += wk;
    to_own_tile();
  }
  if (more) load_rows<K>(a, cur, row0, shared, mask_words, row_scale);
  if (leader) {
#pragma unroll 1
    for (int s = 0; s < K::kStages && more_in; ++s) copy_in();
  }

  // ---- the parts of items
  while (more) {
    const int context = cur.context, drafts = cur.drafts;
    const int64_t b = cur.b;
    const int head = cur.head, part0 = cur.tile, part1 = cur.stop, tiles = cur.tiles;
    __syncthreads();  // q has been written

    constexpr int H = K::kH;
    float o[MT][D / 8][2 * H], base[MT][H], sum[MT][H];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        base[m][h] = -INFINITY;
        sum[m][h] = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[m][n][2 * h] = o[m][n][2 * h + 1] = 0.0f;
      }
    }
    // a thread's rows: warp_row + 16 m + lane / 4, and 8 below
    const int warp_row = wr * 16 * MT;
    float row_c2[K::kRowScale ? MT : 1][K::kRowScale ? H : 1];
    if constexpr (K::kRowScale) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float x = fabsf(p.scale) * kLog2e * row_scale[warp_row + 16 * m + lane / 4 + 8 * h];
          row_c2[m][h] = x < FLT_MIN ? FLT_MIN : x;  // (as a.c2)
        }
    }
    auto c2_of = [&](int m, int h) {
      if constexpr (K::kRowScale) return row_c2[m][h];
      else return a.c2;
    };
    auto seen = [&](int r, int position) {
      return seen_from(p, mask_words[r], b, token_of(a, row0 + r), position - context, drafts);
    };

#pragma unroll 1
    for (int tile = part0 + wk; tile < part1; tile += K::WK) {
      const int stage = out_count % K::kStages;
      mbar_wait(smem_u32(&full[wk][stage]), out_count / K::kStages & 1, &ctl, a.status);
      const char* const k_at = shared + K::kHeadBytes + (wk * K::kStages + stage) * 2 * K::kTileBytes;
      const char* const v_at = k_at + K::kTileBytes;
      const uint32_t k_tile = ring + stage * 2 * K::kTileBytes, v_tile = k_tile + K::kTileBytes;
      const bool masked = (tile + 1) * K::kKeys > context;
      if (stage_bad[wk][stage]) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < H; ++h) sum[m][h] = NAN;
      }

#pragma unroll 1
      for (int k0 = 0; k0 < K::kKeys; k0 += K::kBlock) {
        const int position0 = tile * K::kKeys + k0;
        if (masked && position0 >= context + drafts) break;
        // ---- scores; of several terms the first one's product apart, which alone
        // has the right infinity or NaN
        float s[MT][NT][4], rest[K::F32ACT ? MT : 1][NT][4];
        if constexpr (K::kF32) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t k[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
              ldsm4(k[n], k_tile + chunk_pos<K::kRowBytes, K::kKeys>(k0 + 8 * n + lane % 8,
                                                                    4 * kk + lane / 8));
            if constexpr (K::kPack) {  // q in rows 0-7, what TF32 leaves of it in 8-15
              uint32_t q4[4];
              ldsm4(q4, q_smem + chunk_pos<K::kRowBytes, K::kRows>(lane % 8, 4 * kk + lane / 8));
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint32_t qa[4] = {q4[2 * j], low_tf32(q4[2 * j]), q4[2 * j + 1],
                                        low_tf32(q4[2 * j + 1])};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint32_t b0 = k[n][2 * j], b1 = k[n][2 * j + 1];
                  mma_next<C>(kk + j == 0, s[0][n], qa, b0, b1);
                  mma_next<C>(kk + j == 0, rest[0][n], qa, low_tf32(b0), low_tf32(b1));
                }
              }
              continue;
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t qa[4], ql[4];
                ldsm4(qa, q_smem + chunk_pos<K::kRowBytes, K::kRows>(warp_row + 16 * m + lane % 16,
                                                                    4 * kk + 2 * j + lane / 16));
#pragma unroll
                for (int e = 0; e < 4; ++e) ql[e] = low_tf32(qa[e]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint32_t b0 = k[n][2 * j], b1 = k[n][2 * j + 1];
                  mma_next<C>(kk + j == 0, s[m][n], qa, b0, b1);
                  mma_next<C>(kk + j == 0, rest[m][n], ql, b0, b1);
                  mma<C>(rest[m][n], qa, low_tf32(b0), low_tf32(b1));
                }
              }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t k[NT / 2][4];
#pragma unroll
            for (int n = 0; n < NT / 2; ++n)
              ldsm4(k[n], k_tile + chunk_pos<K::kRowBytes, K::kKeys>(
                                       k0 + 16 * n + lane / 16 * 8 + lane % 8, 2 * ks + lane / 8 % 2));
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int t = 0; t < K::kQTiles; ++t) {
                uint32_t qa[4];
                ldsm4(qa, q_smem + t * K::kQRows * K::kRowBytes +
                              chunk_pos<K::kRowBytes, K::kQRows>(warp_row + 16 * m + lane % 16,
                                                                2 * ks + lane / 16));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint32_t b0 = k[n / 2][n % 2 * 2], b1 = k[n / 2][n % 2 * 2 + 1];
                  if constexpr (K::F32ACT) {
                    if (t > 0) {
                      mma_next<C>(ks == 0 && t == 1, rest[m][n], qa, b0, b1);
                      continue;
                    }
                  }
                  mma_next<C>(ks == 0, s[m][n], qa, b0, b1);
                }
              }
          }
        }
        if constexpr (K::F32ACT) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2 * H; ++e) {
                float others;
                if constexpr (!K::kPack) others = rest[m][n][e];
                else if constexpr (K::kF32) others = s[m][n][2 + e] + (rest[m][n][e] + rest[m][n][2 + e]);
                else others = K::kTerms > 2 ? s[m][n][2 + e] + rest[m][n][e] : s[m][n][2 + e];
                const float x = s[m][n][e] + others;
                s[m][n][e] = x == x ? x : s[m][n][e];
              }
        }
        bool dirty = false;
        uint32_t sees[MT][H];
        if (masked) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              sees[m][h] = seen(warp_row + 16 * m + lane / 4 + 8 * h, position0);
              const uint32_t bits = sees[m][h] >> (lane % 4 * 2);
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (!(bits >> (8 * n + e) & 1u)) s[m][n][2 * h + e] = -INFINITY;
            }
          // what lies behind the last token counts as zero (a weight of 0 would leave
          // its NaN)
          const int rows = context + drafts - position0;
          if (rows < K::kBlock) {
            for (int e = rows * K::kChunks + lane; e < K::kBlock * K::kChunks; e += 32)
              *reinterpret_cast<uint4*>(
                  shared + (v_tile - q_smem) +
                  chunk_pos<K::kRowBytes, K::kKeys>(k0 + e / K::kChunks, e % K::kChunks)) =
                  make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();  // (before a TMA copy writes there)
            __syncwarp();
          }
          // values that are not finite, where not all rows see them
          const int scanned = rows < K::kBlock ? rows : K::kBlock;
          for (int e = max(0, context - position0) * K::kChunks + lane; e < scanned * K::kChunks; e += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(
                v_at + chunk_pos<K::kRowBytes, K::kKeys>(k0 + e / K::kChunks, e % K::kChunks));
            dirty = dirty || only_finite<C>(w.x) != w.x || only_finite<C>(w.y) != w.y ||
                    only_finite<C>(w.z) != w.z || only_finite<C>(w.w) != w.w;
          }
          dirty = __any_sync(0xffffffffu, dirty);
        }

        // ---- the exponents' base, weights
        bool raise = false;
        float top[MT][H];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < H; ++h) {
            float t = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) t = fmaxf(t, fmaxf(s[m][n][2 * h], s[m][n][2 * h + 1]));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            top[m][h] = t * c2_of(m, h) - K::kBelow;
            raise = raise || top[m][h] > base[m][h] + kMaxSlack;
          }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const float old = base[m][h];
              base[m][h] = top[m][h] > old + kMaxSlack ? top[m][h] : old;
              const float f = old == -INFINITY ? 0.0f : ex2(old - base[m][h]);
              sum[m][h] = old == -INFINITY ? sum[m][h] : sum[m][h] * f;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                o[m][n][2 * h] *= f;
                o[m][n][2 * h + 1] *= f;
              }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const float from = base[m][h] == -INFINITY ? 0.0f : base[m][h];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 2 * h; e < 2 * h + 2; ++e) {
                s[m][n][e] = ex2(__fmaf_rn(s[m][n][e], c2_of(m, h), -from));
                sum[m][h] += s[m][n][e];
              }
          }

        // ---- O += weights V, a block's products apart (the tensor core cuts its
        // sums off: a whole sequence's would be too small)
        if constexpr (K::kF32) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            float acc[MT][4];
#pragma unroll
            for (int ks = 0; ks < NT; ++ks) {
              // the product's keys k and k + 4 are 2 k and 2 k + 1 of the eight
              const int key = k0 + 8 * ks + lane % 4 * 2, dim = 8 * n + lane / 4;
              uint32_t v[2], vl[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                v[j] = *reinterpret_cast<const uint32_t*>(
                    v_at + chunk_pos<K::kRowBytes, K::kKeys>(key + j, dim / 4) + dim % 4 * 4);
                if (dirty) v[j] = only_finite<C>(v[j]);
                vl[j] = low_tf32(v[j]);
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                if constexpr (K::kPack) {
                  const uint32_t w0 = __float_as_uint(s[m][ks][0]), w1 = __float_as_uint(s[m][ks][1]);
                  const uint32_t w[4] = {w0, low_weight(w0), w1, low_weight(w1)};
                  mma_next<C>(ks == 0, acc[m], w, v[0], v[1]);
                  mma<C>(acc[m], w, vl[0], vl[1]);
                  continue;
                }
                const uint32_t w[4] = {__float_as_uint(s[m][ks][0]), __float_as_uint(s[m][ks][2]),
                                       __float_as_uint(s[m][ks][1]), __float_as_uint(s[m][ks][3])};
                const uint32_t wl[4] = {low_weight(w[0]), low_weight(w[1]), low_weight(w[2]),
                                        low_weight(w[3])};
                mma_next<C>(ks == 0, acc[m], w, v[0], v[1]);
                mma<C>(acc[m], wl, v[0], v[1]);
                mma<C>(acc[m], w, vl[0], vl[1]);
              }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int e = 0; e < 2 * H; ++e)
                o[m][n][e] += K::kPack ? acc[m][e] + acc[m][2 + e] : acc[m][e];
          }
        } else {
          uint32_t w[MT][NT / 2][K::kWTiles][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int ks = 0; ks < NT / 2; ++ks)
#pragma unroll
              for (int t = 0; t < K::kWTiles; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  if constexpr (K::kPack) {  // rows 0-7 and 8-15: two terms
                    const int term = 2 * t + j % 2;  // (of three: the fourth is next to nothing)
                    w[m][ks][t][j] = term >= K::kWTerms
                                         ? __vminu2(w[m][ks][0][j], 0x00800080u)
                                         : take_weights<K>(s[m][2 * ks + j / 2][0],
                                                           s[m][2 * ks + j / 2][1], K::kWTerms - 1 - term);
                  } else {
                    w[m][ks][t][j] = take_weights<K>(s[m][2 * ks + j / 2][j % 2 * 2],
                                                     s[m][2 * ks + j / 2][j % 2 * 2 + 1],
                                                     K::kWTerms - 1 - t);
                  }
                }
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            constexpr bool kApart = !K::kPositive && !K::kPack;
            float acc[MT][2][4], others[kApart ? MT : 1][2][4];
#pragma unroll
            for (int ks = 0; ks < NT / 2; ++ks) {
              uint32_t v[4];
              ldsm4_trans(v, v_tile + chunk_pos<K::kRowBytes, K::kKeys>(k0 + 16 * ks + lane % 16,
                                                                       2 * n + lane / 16));
              if (dirty) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = only_finite<C>(v[j]);
              }
#pragma unroll
              for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < K::kWTiles; ++t)
#pragma unroll
                  for (int j = 0; j < 2; ++j) {
                    if constexpr (kApart) {
                      if (t > 0) {
                        mma_next<C>(ks == 0, others[m][j], w[m][ks][t], v[2 * j], v[2 * j + 1]);
                        continue;
                      }
                    }
                    mma_next<C>(ks + t == 0, acc[m][j], w[m][ks][t], v[2 * j], v[2 * j + 1]);
                  }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2 * H; ++e) {
                  const float first = acc[m][j][e];
                  if constexpr (kApart) o[m][2 * n + j][e] += with_rest(first, others[m][j][e]);
                  else if constexpr (!K::kPack) o[m][2 * n + j][e] += first;
                  else if constexpr (K::kPositive) o[m][2 * n + j][e] += first + acc[m][j][2 + e];
                  else o[m][2 * n + j][e] += with_rest(first, acc[m][j][2 + e]);
                }
          }
        }
        if (dirty) {  // infinities and NaN, for the rows that see their token
#pragma unroll 1
          for (int k = 0; k < K::kBlock; ++k) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int dim = 8 * n + lane % 4 * 2 + j;
                const C* v = (const C*)(v_at + chunk_pos<K::kRowBytes, K::kKeys>(
                                                   k0 + k, dim * (int)sizeof(C) / 16));
                const float x = to_f32(v[dim % (16 / (int)sizeof(C))]);
                if (!(fabsf(x) < INFINITY)) {
#pragma unroll
                  for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int h = 0; h < H; ++h)
                      if (sees[m][h] >> k & 1u) o[m][n][2 * h + j] += x;
                  }
                }
              }
          }
        }
      }
      __syncwarp();
      if (K::WR > 1 && lane == 0) mbar_arrive(smem_u32(&empty[wk][stage]));
      ++out_count;
      if (leader && more_in) copy_in();
    }

    // ---- the part's end: the four lanes of a row, then the warps that divided
    // the keys, meet
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 1);
        sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 2);
      }
    __syncthreads();  // (q has been read)
    if constexpr (K::WK > 1) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < H; ++h)
          if (lane % 4 == 0) {
            stat[0][wk][warp_row + 16 * m + lane / 4 + 8 * h] = base[m][h];
            stat[1][wk][warp_row + 16 * m + lane / 4 + 8 * h] = sum[m][h];
          }
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int r = warp_row + 16 * m + lane / 4 + 8 * h;
          float top = -INFINITY, all = 0.0f;
#pragma unroll
          for (int w = 0; w < K::WK; ++w) top = fmaxf(top, stat[0][w][r]);
#pragma unroll
          for (int w = 0; w < K::WK; ++w) {
            const float t = stat[0][w][r];
            // (a base of -inf has a sum of 0, or NaN from a page out of range)
            all += t == -INFINITY ? stat[1][w][r] : stat[1][w][r] * ex2(t - top);
          }
          const float f = base[m][h] == -INFINITY ? 1.0f : ex2(base[m][h] - top);
          base[m][h] = top;
          sum[m][h] = all;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[m][n][2 * h] *= f;
            o[m][n][2 * h + 1] *= f;
          }
        }
      float* const join = reinterpret_cast<float*>(shared);
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += K::kJoinDims) {
        if (d0 > 0) __syncthreads();
        if (wk > 0) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < K::kJoinDims / 8; ++n)
#pragma unroll
              for (int h = 0; h < H; ++h)
                *reinterpret_cast<float2*>(
                    join + (((wk - 1) * K::kRows + warp_row + 16 * m + lane / 4 + 8 * h) *
                                K::kJoinDims + (8 * n ^ (lane / 4 % 4 * 8)) + lane % 4 * 2)) =
                    make_float2(o[m][d0 / 8 + n][2 * h], o[m][d0 / 8 + n][2 * h + 1]);
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
          for (int w = 1; w < K::WK; ++w)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int n = 0; n < K::kJoinDims / 8; ++n)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                  const float2 x = *reinterpret_cast<const float2*>(
                      join + (((w - 1) * K::kRows + warp_row + 16 * m + lane / 4 + 8 * h) *
                                  K::kJoinDims + (8 * n ^ (lane / 4 % 4 * 8)) + lane % 4 * 2));
                  o[m][d0 / 8 + n][2 * h] += x.x;
                  o[m][d0 / 8 + n][2 * h + 1] += x.y;
                }
        }
      }
    }
    const bool whole = part0 == 0 && part1 == tiles;
    if (wk == 0) {
      float* const slot = a.partials + ((int64_t)blockIdx.x * 2 + (part0 == 0 ? 1 : 0)) *
                                           partial_floats(K::kRows, D);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int r = warp_row + 16 * m + lane / 4 + 8 * h, i = token_of(a, row0 + r);
          if (i >= drafts) continue;
          if (whole) {
            const float f = sum[m][h] == 0.0f ? 0.0f : 1.0f / sum[m][h];
            const int64_t row = (b * p.drafts + i) * p.q_heads + head * a.group + (row0 + r) - i * a.group;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              store2<A>(p.out, row * D + 8 * n + lane % 4 * 2, o[m][n][2 * h] * f,
                        o[m][n][2 * h + 1] * f);
            if (lane % 4 == 0 && p.lse)
              p.lse[row] = sum[m][h] == 0.0f ? -INFINITY : (base[m][h] + log2f(sum[m][h])) * kLn2;
          } else {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<float2*>(slot + r * D + 8 * n + lane % 4 * 2) =
                  make_float2(o[m][n][2 * h], o[m][n][2 * h + 1]);
            if (lane % 4 == 0)
              *reinterpret_cast<float2*>(slot + K::kRows * D + 2 * r) =
                  make_float2(base[m][h], sum[m][h]);
          }
        }
    }
    if (!whole && part0 == 0 && tid == 0) {
      // the item ends in the share that has its last unit
      const int64_t end = (int64_t)(share + 1) * share_units + (tiles - part1);
      a.records[blockIdx.x] = make_int4((int)((end - 1) / share_units) - share + 1, (int)b, head, drafts);
    }
    __syncthreads();  // (the join has been read, q may be written)
    ++cur.head;
    more = enter<K>(a, cur, 0, row0);
    if (more) load_rows<K>(a, cur, row0, shared, mask_words, row_scale);
  }
  write_rows_not_there<K>(p);
  // after a wait that ran out: copies still on the way end before the memory is
  // given back
  if (ctl.abort && leader)
    for (uint32_t n = in_count > K::kStages ? in_count - K::kStages : 0; n < in_count; ++n)
      for (int i = 0; i < 1 << 20; ++i)
        if (mbar_test_wait(smem_u32(&full[wk][n % K::kStages]), n / K::kStages & 1)) break;
}

template <class K>
int launch(Launch a, const DeviceInfo& dev, cudaStream_t st) {
  const TreeAttention& p = a.p;
  int rc = allow_shared<tree_attention_kernel<K>>(K::kSmem, dev);
  if (rc != CT_OK) return rc;
  a.blocks = (int)((p.drafts * a.group + K::kRows - 1) / K::kRows);
  const int64_t items = p.batch * p.kv_heads;
  int ctas = K::kCtas * dev.sm_count;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  a.whole = p.kv.max_pages * p.kv.page_size <= K::kWholeTokens || a.blocks > ctas / 2;
  int64_t shares = a.whole ? items : ctas / a.blocks;
  if (shares * a.blocks >= 1ll << 31) return CT_ERR_INVALID_ARGUMENT;
  a.shares = (int)shares;
  CUtensorMap k_map{}, v_map{};
  make_maps(a, &k_map, &v_map, K::kKeys);
  const unsigned grid = (unsigned)(shares * a.blocks);
  tree_attention_kernel<K><<<grid, kThreads, K::kSmem, st>>>(a, k_map, v_map);
  rc = check_launch();
  if (rc != CT_OK || a.whole) return rc;
  return launch_join<typename K::A, K::D>(a, grid, K::kRows, dev, st);
}

template <class C, bool F32ACT, int D>
int launch_rows(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  const int64_t rows = a.p.drafts * a.group;
  constexpr int MT = F32ACT ? 1 : 2;
  if (rows <= 8) return launch<Cfg<C, F32ACT, D, 0, 1>>(a, dev, st);
  if (rows <= 16) return launch<Cfg<C, F32ACT, D, 1, 1>>(a, dev, st);
  if (rows <= 32) return launch<Cfg<C, F32ACT, D, MT, 2 / MT>>(a, dev, st);
  return launch<Cfg<C, F32ACT, D, MT, 4 / MT>>(a, dev, st);
}

}  // namespace

size_t tree_attention_workspace(int64_t drafts, int64_t q_heads, int64_t kv_heads,
                                int64_t head_dim) {
  const int64_t rows = drafts * (q_heads / kv_heads);
  // (rows of a slot: a block's of this kernel, or up to 128 on tcgen05)
  const int tile = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows >= 128 ? 128 : (int)(rows + 15) / 16 * 16;
  return kMaxCtas * (sizeof(int4) + 2 * (size_t)partial_floats(tile, (int)head_dim) * sizeof(float));
}

int launch_tree_attention(const TreeAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  const int rc = launch_tc(p, dev, st);
  if (rc != kNoTc) return rc;
  const Launch a = begin_launch(p, dev);
  return with_dtype(p.act_dtype, [&](auto act) {
    return with_dtype(p.kv.dtype, [&](auto cache) {
      using A = decltype(act);
      using C = decltype(cache);
      if constexpr (std::is_same<A, C>::value || std::is_same<A, float>::value) {
        constexpr bool kF32Act = std::is_same<A, float>::value;
        if (p.head_dim == 32) return launch_rows<C, kF32Act, 32>(a, dev, st);
        if (p.head_dim == 64) return launch_rows<C, kF32Act, 64>(a, dev, st);
        return launch_rows<C, kF32Act, 128>(a, dev, st);
      } else {
        return (int)CT_ERR_INVALID_ARGUMENT;
      }
    });
  });
}

}  // namespace ct
