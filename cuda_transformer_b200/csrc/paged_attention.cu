// paged_attention.cu -- attention of one new token per sequence over a paged
// key/value cache:
//   s_j = scale q . k_j,  O = sum_j softmax(s)_j v_j,  L = ln sum_j exp(s_j)
// over the sequence's cached tokens j; O = 0 and L = -inf when there are none.
// Query heads share key/value heads in groups of q_heads / kv_heads.
//
// Every cached value is read once and used for 2 * group FLOPs, so the bound
// is HBM.  The design follows from that:
//  * Work is cut into tiles of 8 to 32 keys of one item (a sequence and a
//    key/value head), and every CTA takes an equal share of the tiles, counted
//    on the device from seq_lens (the host knows no lengths).  Ragged batches
//    and one long sequence load the GPU alike.  Short items stay whole; the
//    shortest belong to one warp, which needs nobody else, at the others the
//    four warps of a CTA take turns and join at the end.  A share that starts
//    or ends inside a long item leaves a partial (maximum, sum, O) in the
//    workspace; the CTA that arrives last joins the partials in their order,
//    so results do not depend on timing and no CTA waits for another.
//  * Each warp streams q and its keys and values through a private cp.async
//    ring (16-byte copies gather pages of any size and layout) that runs ahead
//    across items; a block barrier comes only where a long item ends.
//  * Products run on mma.sync: 16-bit cache values go in as they are, FP32 q and
//    the probabilities as two or three 16-bit terms (16 bits and more for 16-bit
//    outputs, 22 and more for FP32 ones); of FP32 caches both sides are two TF32
//    terms (21 bits and more), all four products of which are formed by two
//    instructions.  8 heads put two terms into the 16 rows of one product (high and
//    low sums of a head then sit in the same lane).  The order of keys and dims
//    inside a product is chosen so that every operand is a 16-byte shared-memory
//    vector: no shuffles, no transposes.  On tcgen05 keys or dims would be the 128
//    rows and the heads the 8 or 16 columns; up to 8 heads the tensor pipe is not
//    what bounds this kernel (15 % active with 4), beyond them that form has not
//    been built.  One or two heads are cheaper as plain FMAs of FP32 (a lane has a
//    part of a key's dims, so only scores are added up across four lanes).
//    Relative error of O against 64 bits, 8 x 100..3000 tokens, FP32 q: one head
//    1.6e-7 to 1.8e-7, 16-bit caches with 4 or 8 heads 1.8e-7 to 2.6e-7, FP32 caches
//    4.0e-7 to 5.6e-7 (FP32 throughout in PyTorch: 1.9e-7 to 4.5e-7).
//
// Device time of a launch on a B200 (floor: the cached values at the 6.53 TB/s
// of a copy); 32 heads on 8 of 128, bf16, unless it says otherwise:
//   64 sequences of 4096 tokens            174 us         floor 164
//   one of 131072                          91.5           82.2
//   32 on 32 of 64, FP32 q, 16 x 3500..4096 82.8          76.0
//   64 of 16 .. 4096                       44.4           30.4
//   FP32, 8 on 8 of 128, 5 x 777..4097     24.7           13.2
//   FP32, 32 on 8 of 64 / 128, 16 / 8 x 4096 60.6 / 60.8  41.1
//   f16, 16 on 1 of 64, 128 x 1..16384     28.6           8.7
//   one of 8192 / 1024 / 64         17.9 / 13.0 / 6.5     5.1 / 0.6 / 0.04
// Long batches run at the copy's rate.  The rest is a fixed chain of latencies:
// 2 us to start, 2 us for the lengths and the table, 2 to 3 us until the first
// tile is worked on, 1 us at the end of an item and about 3 us (write, fence,
// counter, read) for each level of joining, two of them from 9 parts on.  Where
// a choice below names a figure, both sides were measured on the code of its day.
#include <cfloat>

#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kMaxCtas = 448;  // counters (of each level) and partial slots in the workspace
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
// Partials that are joined at a time.  (32: 8192 tokens 32 us instead of 24,
// 131072 105 instead of 96; 16, where a thread holds them: FP32, 8 on 8 of 128,
// 5 x 777..4097 27.1 instead of 26.1.)
constexpr int kFan = 8;
constexpr int kLevels = 3;     // kFan^kLevels >= kMaxCtas
// Items of at most so many tiles are never split between CTAs: joining the
// parts costs more than the tiles, in short shares above all.  Those of no more
// tiles than a warp's part of its CTA's share are one warp's.  (Whole up to 12
// tiles against 16: 64 sequences of 16 to 4096 tokens, in six random orders, 48
// us against 49 on average and 48 against 56 at most; FP32, 6 on 6 of 64,
// 128 x 1..256, which have shares of 19 tiles, 13.5 against 11.5.)
constexpr int kShortShare = 32;
__device__ __forceinline__ int longest_whole(int64_t share) { return share < kShortShare ? 16 : 12; }
// What an item costs beside its tiles (q, the end), in tiles.  (The same six,
// 3 / 7 / 12: 52 / 49 / 51 us; FP32, 8 on 8 of 128, 5 x 777..4097 26.7 / 25.1 /
// 24.9.)
constexpr int kItemCost = 7;
// Tiles of a CTA, unless there are fewer in all: one for each warp.  (With 16,
// one sequence of 1024 tokens takes 16.4 us instead of 13.3 and one of 64 9.6
// instead of 6.4; 8192 tokens 21.7 instead of 23.2, 16 heads on one of 64 over
// 128 x 490 tokens 11.4 instead of 13.4.)
constexpr int kMinShare = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is raised only when a score passes it by this much (in
// powers of two): probabilities stay below 2^6, which FP32 sums hold as well
// as values below 1, and most tiles skip the rescaling of O.
constexpr float kMaxSlack = 6.0f;

#pragma nv_diag_suppress 177  // not every configuration refers to every member
template <class C, bool F32ACT>
constexpr int q_terms() {
  return sizeof(C) == 4 ? 2 : !F32ACT ? 1 : std::is_same<C, __nv_bfloat16>::value ? 3 : 2;
}

// C: the cache's type; F32ACT: q and out are FP32, else of type C; M: query
// heads a CTA works on.  8: on the tensor cores, high and low parts share a
// product's rows; 1 and 2: plain FMAs.
template <class C, bool F32ACT, int D, int M>
struct Cfg {
  static constexpr bool kLanes = M <= 2;                    // no tensor cores
  using A = std::conditional_t<F32ACT, float, C>;           // type of q and out
  static constexpr bool kF32 = sizeof(C) == 4;
  static constexpr bool kBf16 = std::is_same<C, __nv_bfloat16>::value;
  static constexpr int kVec = 16 / (int)sizeof(C);          // elements of a 16-byte chunk
  static constexpr int kRowBytes = D * (int)sizeof(C);
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kKIter = D / (4 * kVec);              // K chunks a lane reads per key
  static constexpr int kVVec = kVec < D / 8 ? kVec : D / 8;  // V elements a lane reads at once
  static constexpr int kVIter = D / (8 * kVVec);
  static constexpr int kOTiles = D / 8;
  // Terms q and the probabilities are split into (pairs share a product, a term
  // in rows 0-7 and a term in rows 8-15).  With 16-bit activations q
  // is exact as it is, and two terms of p leave an error (2^-16 in bf16) far
  // below the output's own rounding; FP32 activations take as many as hold 22
  // bits or more.
  static constexpr int kQTerms = q_terms<C, F32ACT>();
  static constexpr int kPTerms = F32ACT && kBf16 ? 3 : 2;
  // The exponent's base lies this far below the running maximum (in powers of
  // two): f16 probabilities reach up to 2^14 instead of 1, so that the many
  // small ones of a long sequence stay clear of the subnormals.
  static constexpr float kBelow = !kF32 && !kBf16 ? 8.0f : 0.0f;
  // A operands of one step (8 dims in TF32, 16 in the 16-bit types): rows 0-7
  // and 8-15 hold two terms.
  static constexpr int kQOps = (kQTerms + 1) / 2, kPOps = (kPTerms + 1) / 2;
  static constexpr int kSteps = kF32 ? D / 8 : D / 16;
  static constexpr int kQRegs = kLanes ? M * D / 4 : kSteps * kQOps * 4;
  // Keys of a warp's tile: 8 KB of K and V, 32 at most; a smaller one (8 keys in
  // TF32, 16 in the 16-bit types) where q and O leave no registers for the
  // larger one's scores (they would spill).
  static constexpr int kLeast = kF32 ? 8 : 16;
  static constexpr int kMost = 4096 / kRowBytes < 32 ? 4096 / kRowBytes : 32;
  static constexpr int kKeys = kLanes || kQRegs + D / 2 <= 48 ? kMost : kLeast;
  static constexpr int kRun = kKeys < 16 ? kKeys : 16;       // keys that are copied from one page
  static constexpr int kNt = kKeys / 8;
  static constexpr int kCopies = kKeys * kRowChunks / 32;    // of a lane, for K or V
  static constexpr int kCopyRows = 32 / kRowChunks;          // rows of one copy instruction
  static constexpr int kStageBytes = 2 * kKeys * kRowBytes;  // K tile, V tile
  // Three CTAs an SM of 168 registers a thread, with two stages of 8 KB or as
  // many smaller ones; two CTAs with three stages where q and O of several heads
  // of 128 dims leave too few registers.  (32 heads on 8 of 128: FP32 q on f16,
  // 16 x 4096 tokens, 55 us instead of 72; bf16, 64 x 16..4096 43.9 instead of 45.5,
  // 64 x 64 9.7 instead of 11.9, 64 x 4096 174.9 instead of 173.  Two CTAs at 64
  // dims: FP32, 32 on 8, 16 x 4096 61.4 instead of 59.4.)  FP32 q of several heads
  // still spills a little: 44 (f16), 146 (bf16) and 172 (FP32) bytes a thread at 128
  // dims with 255 registers, 4 to 74 below, 8 with 16-bit q at 64.
  static constexpr int kCtas = D == 128 && M > 1 ? 2 : 3;
  static constexpr int kRing = kCtas == 3 ? 16384 : 24576;
  static constexpr int kStages = kRing / kStageBytes > 6 ? 6 : kRing / kStageBytes;
  static_assert(M * D * 4 <= kStageBytes, "the warps' O meet in stages of their rings");
  static constexpr int kQRowChunks = D * (int)sizeof(A) / 16;
  static constexpr int kQChunks = M * kQRowChunks;
  static_assert(kQChunks * 16 <= kStageBytes, "q passes through a stage of the ring");
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// D = A B + C for one tile: 16 x 8 x 8 in TF32, 16 x 8 x 16 in the 16-bit types.
template <class C>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
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
// x = high + low, both TF32 (11 significant bits): the high part is cut off,
// the rest (13 bits) rounded, so the error is below 2^-22 of x.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}
// The same of a cached value: the tensor core drops the 13 low bits of what it
// is given, so x itself is the high part and the low part is not rounded (the
// error is below 2^-21 of x).
__device__ __forceinline__ uint32_t low_tf32(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u));
}
// The next 16-bit term of x and y (x in the low half); x and y keep the rest.
template <class C, bool CUT = false>
__device__ __forceinline__ uint32_t take_term(float& x, float& y) {
  uint32_t w;
  if constexpr (CUT) {  // cut off instead of rounded: the rest has x's sign
    static_assert(std::is_same<C, __nv_bfloat16>::value, "");
    w = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= __uint_as_float(w << 16);
    y -= __uint_as_float(w & 0xffff0000u);
  } else if constexpr (std::is_same<C, __nv_bfloat16>::value) {
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

// Infinite cached values.  The product of the first terms alone has the right
// infinity, or NaN; the others' are 0 * inf or of either sign.  So a result is
// the first terms' sum where that is not finite, and their rows or accumulators
// hold nothing of the others that could be NaN.
__device__ __forceinline__ float with_rest(float first, float rest) {
  return fabsf(first) < INFINITY ? first + rest : first;
}
// The low part of a cached V, whose products join the first terms': some finite
// number (and no sum over KEYS keys overflows) where inf - inf made it NaN.
// (It is below 2^116, and so kept, of values below 2^126.  A NaN is one by its
// high mantissa bits here, which every NaN that arithmetic makes has set.)
template <int KEYS>
__device__ __forceinline__ uint32_t finite_low_tf32(uint32_t x) {
  return __float_as_uint(fminf(__uint_as_float(low_tf32(x)), 0x1p121f / KEYS));
}

// Element e of a 16-byte chunk.
template <class C>
__device__ __forceinline__ float chunk_value(const uint32_t (&w)[4], int e) {
  if constexpr (sizeof(C) == 4)
    return __uint_as_float(w[e]);
  else if constexpr (std::is_same<C, __nv_bfloat16>::value)
    return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  else
    return e & 1 ? __high2float(*reinterpret_cast<const __half2*>(&w[e / 2]))
                 : __low2float(*reinterpret_cast<const __half2*>(&w[e / 2]));
}

// Position of 16-byte chunk `c` of tile row `r`.  Chunks are permuted within
// 128-byte lines so that the eight lanes of an access phase (two keys times
// four K chunks; four key pairs times two V chunks) meet different banks.
template <int ROW_BYTES>
__device__ __forceinline__ int chunk_pos(int r, int c) {
  if constexpr (ROW_BYTES >= 128)
    return r * ROW_BYTES + ((c ^ (r & 6) ^ ((r & 1) << 2)) << 4);
  else  // 64-byte rows, two to a line
    return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (r & 6)) << 4);
}

// Position of 16-byte chunk c of q's row h in its stage.
template <int ROW_CHUNKS>
__device__ __forceinline__ int q_pos(int h, int c) {
  return (h * ROW_CHUNKS + (c ^ (h & (ROW_CHUNKS < 8 ? ROW_CHUNKS - 1 : 7)))) * 16;
}

__device__ __forceinline__ void store_act4(void* p, int64_t i, int dtype, float4 x) {
  if (dtype == CT_DTYPE_F32) {
    *reinterpret_cast<float4*>((float*)p + i) = x;
  } else if (dtype == CT_DTYPE_BF16) {
    alignas(8) __nv_bfloat162 v[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>((__nv_bfloat16*)p + i) = *reinterpret_cast<uint2*>(v);
  } else {
    alignas(8) __half2 v[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>((__half*)p + i) = *reinterpret_cast<uint2*>(v);
  }
}

// Floats of a partial: O [heads][D], then maximum and sum [heads] each; a
// multiple of 4 (16 bytes).
constexpr int64_t partial_floats(int heads, int D) { return ((int64_t)heads * (D + 2) + 3) / 4 * 4; }

struct Launch {
  PagedAttention p;
  int group, blocks;  // query heads of a key/value head; its blocks of M heads
  int items;          // (key/value head, block) pairs of a sequence
  int page_shift;     // log2 of page_size, -1 when it is no power of two
  bool whole_tiles;   // a tile's keys (runs of 16) lie in one page
  bool q_vectors;     // q's rows are 16-byte vectors
  uint32_t* counters;
  float* partials;
};

// A place in the list of tiles: sequence, item, tile in the item.
struct Cursor {
  int64_t b;
  int item, tile, tiles, len;
  bool bad;
};

// A long item that other CTAs work on too: the first of them, how many, the
// item's row of the output.
struct Split {
  int64_t row;
  int first, n, heads;
};

template <int KEYS>
__device__ __forceinline__ void read_length(const Launch& a, Cursor& c) {
  const int n = a.p.seq_lens[c.b];
  c.bad = n > a.p.kv.max_pages * a.p.kv.page_size;
  c.len = n < 0 || c.bad ? 0 : n;
  c.tiles = c.len > KEYS ? (c.len + KEYS - 1) / KEYS : 1;  // one, empty, at length 0
}

// A head's result from its unnormalised O and its maximum and sum.
__device__ __forceinline__ void write_out(const PagedAttention& p, int64_t row, int d, int D,
                                          float4 x, float m, float l) {
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  store_act4(p.out, row * D + d, p.act_dtype, make_float4(x.x * r, x.y * r, x.z * r, x.w * r));
  if (d == 0 && p.lse) p.lse[row] = (m + log2f(l)) * kLn2;
}

// a / b of non-negative numbers, quickly where 32 bits hold them.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((uint64_t)a | (uint64_t)b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// 2^x to 2 ulp (0 for -inf and for results below the normal range).
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Reference point of a maximum: sums that have seen no key are 0 to any.
__device__ __forceinline__ float finite(float top) { return top == -INFINITY ? 0.0f : top; }

// Joins the partials k0, k0 + step, .. (n of them, kFan at most) of the item
// that CTA c0 starts, in that order: into partial k0 or the output.
template <int HEADS, int D>
__device__ __forceinline__ void join_partials(const Launch& a, int c0, int k0, int step, int n,
                                              bool to_partial, int64_t row, int heads) {
  constexpr int64_t kSize = partial_floats(HEADS, D);
  constexpr int kItems = HEADS * D / 4;  // float4s, one or two to a thread
  constexpr int kPart = kItems > kThreads ? 2 : 1;
  static_assert(kItems <= kPart * kThreads, "");
  auto at = [&](int k) { return a.partials + (k == 0 ? 2 * c0 + 1 : 2 * (c0 + k)) * kSize; };
  float km[kPart][kFan], kl[kPart][kFan];
  float4 y[kPart][kFan];
#pragma unroll
  for (int j = 0; j < kFan; ++j) {
    if (j >= n) continue;
    const float* s = at(k0 + j * step);
#pragma unroll
    for (int i = 0; i < kPart; ++i) {
      const int id = threadIdx.x + i * kThreads;
      if (id >= kItems) continue;
      km[i][j] = __ldcg(s + HEADS * D + id / (D / 4));
      kl[i][j] = __ldcg(s + HEADS * D + HEADS + id / (D / 4));
      y[i][j] = __ldcg(reinterpret_cast<const float4*>(s + id * 4));
    }
  }
  // a head's maxima and sums are read by the lanes of one warp; partial k0 is
  // overwritten after they have them
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPart; ++i) {
    const int id = threadIdx.x + i * kThreads, h = id / (D / 4), d = id % (D / 4) * 4;
    if (id >= kItems) continue;
    float m = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kFan; ++j)
      if (j < n) m = fmaxf(m, km[i][j]);
    const float ref = finite(m);
#pragma unroll
    for (int j = 0; j < kFan; ++j) {
      if (j >= n) continue;
      const float f = exp2_fast(km[i][j] - ref);
      x.x = fmaf(y[i][j].x, f, x.x);
      x.y = fmaf(y[i][j].y, f, x.y);
      x.z = fmaf(y[i][j].z, f, x.z);
      x.w = fmaf(y[i][j].w, f, x.w);
      l = fmaf(kl[i][j], f, l);
    }
    if (to_partial) {
      float* s = at(k0);
      *reinterpret_cast<float4*>(s + id * 4) = x;
      if (d == 0) {
        s[HEADS * D + h] = m;
        s[HEADS * D + HEADS + h] = l;
      }
    } else if (h < heads) {
      write_out(a.p, row + h, d, D, x, m, l);
    }
  }
}

template <class C, bool F32ACT, int D, int M>
__global__ void __launch_bounds__(kThreads, Cfg<C, F32ACT, D, M>::kCtas)
    paged_attention_kernel(const __grid_constant__ Launch a) {
  using F = Cfg<C, F32ACT, D, M>;
  using A = typename F::A;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_scan[kWarps];
  __shared__ int64_t s_rest[kWarps];
  __shared__ Cursor s_edge[2];
  __shared__ int64_t s_first[2];
  __shared__ float s_m[kWarps][M], s_l[kWarps][M];
  __shared__ int s_area[kWarps];
  __shared__ bool s_last[2];
  __shared__ Split s_split[2];
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const PagedAttention& p = a.p;

  // ---- this CTA's share of the tiles: a scan of the sequences' tiles (and
  // items' costs), a block's worth at a time (nearly always one)
  if (tid == 0) s_edge[1].b = p.batch;  // where the last share ends
  if (tid < 2) s_split[tid] = Split{};
  Cursor c{};
  c.b = tid;
  if (c.b < p.batch) read_length<F::kKeys>(a, c);
  int64_t rest = 0;  // tiles of the sequences past the first block's worth
  if (p.batch > kThreads) {
    for (int64_t b = tid + kThreads; b < p.batch; b += kThreads) {
      Cursor x;
      x.b = b;
      read_length<F::kKeys>(a, x);
      rest += x.tiles + kItemCost;
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(0xffffffffu, rest, o);
    if (lane == 0) s_rest[w] = rest;
  }
  auto warp_scan = [&]() {  // 32 sequences have fewer than 2^32 tiles
    uint32_t x = c.b < p.batch ? c.tiles + kItemCost : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[w] = x;
    return (int64_t)x;
  };
  int64_t upto = warp_scan(), block = 0, before = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) upto += s_scan[i];
    block += s_scan[i];
  }
  rest = 0;
  if (p.batch > kThreads)
    for (int i = 0; i < kWarps; ++i) rest += s_rest[i];
  const int64_t total = (block + rest) * a.items;
  int64_t ctas = divide(total + kMinShare - 1, kMinShare);
  if (ctas > gridDim.x) ctas = gridDim.x;
  if (blockIdx.x >= ctas) return;
  // CTA c's share begins at tile c * total / ctas, rounded down
  const int64_t share = divide(total, ctas);
  const int whole = longest_whole(share);
  auto cta_of = [&](int64_t tile) { return divide((tile + 1) * ctas - 1, total); };
  int64_t edge[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) edge[e] = divide((blockIdx.x + e) * total, ctas);
  while (true) {
    const int cost = c.tiles + kItemCost;
    const int64_t start = (before + upto - cost) * a.items;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      const int64_t from = edge[e] - start;
      if (c.b < p.batch && from >= 0 && from < (int64_t)cost * a.items) {
        Cursor x = c;
        x.item = (int)divide(from, cost);
        x.tile = (int)(from - (int64_t)x.item * cost) - kItemCost;
        s_first[e] = edge[e] - x.tile;  // the item's first tile, in the count
        // an edge in the item's cost, or inside a short item, moves to its start
        if (x.tile < 0 || x.tiles <= whole) x.tile = 0;
        s_edge[e] = x;
      }
    }
    before += block;
    __syncthreads();
    if (before * a.items > edge[1] || before * a.items == total) break;
    c = Cursor{c.b + kThreads, 0, 0, 0, 0, false};
    if (c.b < p.batch) read_length<F::kKeys>(a, c);
    upto = warp_scan();
    __syncthreads();
    block = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < w) upto += s_scan[i];
      block += s_scan[i];
    }
  }
  Cursor cur = s_edge[0];
  const int64_t end_b = s_edge[1].b;
  const int end_item = end_b < p.batch ? s_edge[1].item : 0;
  const int end_tile = end_b < p.batch ? s_edge[1].tile : 0;
  if (cur.b == end_b && cur.item == end_item && cur.tile >= end_tile) return;
  const int brief = (int)(share / kWarps < whole ? share / kWarps : whole);

  // Walks the share item by item: true with `seg`, the tiles of the item that
  // lie in the share, and whether it is this warp's alone; false at the end.
  // Short items of other warps are passed over.
  auto next_item = [&](Cursor& x, int& seg, bool& own, bool fresh) {
    while (true) {
      if (!fresh) {
        if (x.b == end_b && x.item == end_item) return false;
        x.tile = 0;
        if (++x.item == a.items) {
          x.item = 0;
          if (++x.b < p.batch) read_length<F::kKeys>(a, x);
        }
      }
      fresh = false;
      seg = (x.b == end_b && x.item == end_item ? end_tile : x.tiles) - x.tile;
      if (seg <= 0 || x.b >= p.batch) return false;
      own = x.tiles <= brief;
      if (!own || (uint32_t)(x.b * a.items + x.item) % kWarps == w) return true;
    }
  };

  // ---- the copy side: q, then the tiles of this warp, kStages - 1 ahead of
  // the products
  const uint32_t ring = smem_addr(smem) + w * (F::kStages * F::kStageBytes);
  const uint8_t* ring_ptr = smem + w * (F::kStages * F::kStageBytes);
  const int my_row = lane % F::kKeys;
  const int copy_row = lane / F::kRowChunks, copy_chunk = lane % F::kRowChunks;
  const int64_t k_step = p.kv.ks[2] * (int64_t)sizeof(C), v_step = p.kv.vs[2] * (int64_t)sizeof(C);
  const int64_t k_page = p.kv.ks[0] * (int64_t)sizeof(C), v_page = p.kv.vs[0] * (int64_t)sizeof(C);
  const uint8_t* k_lane = (const uint8_t*)p.kv.k + copy_row * k_step + copy_chunk * 16;
  const uint8_t* v_lane = (const uint8_t*)p.kv.v + copy_row * v_step + copy_chunk * 16;
  Cursor ahead = cur;
  int ahead_seg = 0;
  bool ahead_own = false;
  // of the item that is being copied: this warp's tiles still to go, the key of
  // the lane's row in the next, the end of the keys, where its head and its row
  // of the table begin
  int tiles_left = 0, key = 0, key_end = 0;
  const uint8_t *k_item = k_lane, *v_item = v_lane;
  const int32_t* pages = p.kv.table;
  // What the next issue copies: nothing, q, or a tile whose rows' pages and
  // slots have been looked up
  enum { kNothing, kQuery, kTile };
  int next = kNothing, next_page = -1, next_slot = 0;
  bool next_there = false;
  auto look_up = [&]() {
    next_there = key < key_end;
    if (next_there) {
      const int index = a.page_shift >= 0 ? key >> a.page_shift : key / p.kv.page_size;
      next_slot = key - index * p.kv.page_size;
      next_page = pages[index];
    }
  };
  auto begin_item = [&]() {
    next = kQuery;
    tiles_left = ahead_own ? ahead_seg : (ahead_seg + kWarps - 1) / kWarps;
    key = (ahead.tile + (ahead_own ? 0 : w)) * F::kKeys + my_row;
    key_end = (ahead.tile + ahead_seg) * F::kKeys;
    if (key_end > ahead.len) key_end = ahead.len;
    const int64_t head = ahead.item / a.blocks;
    k_item = k_lane + head * p.kv.ks[1] * (int64_t)sizeof(C);
    v_item = v_lane + head * p.kv.vs[1] * (int64_t)sizeof(C);
    pages = p.kv.table + ahead.b * p.kv.table_s;
  };
  auto step_ahead = [&]() {  // past what has been issued
    if (next == kTile && --tiles_left > 0) {
      key += (ahead_own ? 1 : kWarps) * F::kKeys;
      look_up();
    } else if (next == kQuery) {
      next = kTile;
      look_up();
    } else if (next == kTile) {
      next = kNothing;
      if (next_item(ahead, ahead_seg, ahead_own, false)) begin_item();
    }
  };
  if (next_item(ahead, ahead_seg, ahead_own, true)) begin_item();
  auto issue = [&](int stage) {
    const uint32_t base = ring + stage * F::kStageBytes;
    if (next == kTile) {
      const bool fine = next_there && (unsigned)next_page < (unsigned)p.kv.pages;
      if (a.whole_tiles && __all_sync(0xffffffffu, fine)) {
        // all rows are there and follow one another in one page (or two)
#pragma unroll
        for (int run = 0; run < F::kKeys / F::kRun; ++run) {
          const int64_t page = F::kKeys == F::kRun ? next_page
                                                   : __shfl_sync(0xffffffffu, next_page, run * F::kRun);
          const int slot = F::kKeys == F::kRun ? next_slot - my_row
                                               : __shfl_sync(0xffffffffu, next_slot, run * F::kRun);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int64_t row_step = kv ? v_step : k_step, step = F::kCopyRows * row_step;
            const uint8_t* src = (kv ? v_item : k_item) + page * (kv ? v_page : k_page) + slot * row_step;
#pragma unroll
            for (int i = 0; i < F::kRun / F::kCopyRows; ++i)
              cp_async16(base + kv * (F::kKeys * F::kRowBytes) +
                             chunk_pos<F::kRowBytes>(run * F::kRun + i * F::kCopyRows + copy_row,
                                                     copy_chunk),
                         src + i * step, 16);
          }
        }
      } else if (__any_sync(0xffffffffu, next_there)) {
        // bytes from the item's first row: -1 past the length (zeros), -2 where
        // there is no such page (NaN)
        int64_t off[2] = {next_there ? -2 : -1, next_there ? -2 : -1};
        if (fine) {
          off[0] = next_page * k_page + next_slot * k_step;
          off[1] = next_page * v_page + next_slot * v_step;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint8_t* from = kv ? v_item - copy_row * v_step : k_item - copy_row * k_step;
#pragma unroll
          for (int i = 0; i < F::kCopies; ++i) {
            const int r = i * F::kCopyRows + copy_row;
            const int64_t o = __shfl_sync(0xffffffffu, off[kv], r);
            const uint32_t dst =
                base + kv * (F::kKeys * F::kRowBytes) + chunk_pos<F::kRowBytes>(r, copy_chunk);
            if (o < 0)  // (0x7fc07fc0 is NaN in each of the three types)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst),
                           "r"(o == -2 ? 0x7fc07fc0u : 0u)
                           : "memory");
            else
              cp_async16(dst, from + o, 16);
          }
        }
      }
    } else if (next == kQuery) {
      const int head = ahead.item / a.blocks, head0 = (ahead.item % a.blocks) * M;
      const A* q = (const A*)p.q + ahead.b * p.qs[0] + ((int64_t)head * a.group + head0) * p.qs[1];
#pragma unroll 1
      for (int i = lane; i < F::kQChunks; i += 32) {
        const int h = i / F::kQRowChunks, ch = i % F::kQRowChunks;
        const bool there = head0 + h < a.group;
        const A* row = there ? q + h * p.qs[1] + ch * (16 / (int)sizeof(A)) * p.qs[2] : q;
        const uint32_t dst = base + q_pos<F::kQRowChunks>(h, ch);
        if (a.q_vectors) {
          cp_async16(dst, row, there ? 16 : 0);
        } else {
          alignas(16) A x[16 / sizeof(A)];
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(A); ++e) x[e] = there ? row[e * p.qs[2]] : A(0.0f);
          const uint4 v = *reinterpret_cast<const uint4*>(x);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y),
                       "r"(v.z), "r"(v.w)
                       : "memory");
        }
      }
    }
    cp_async_commit();
    step_ahead();
  };

  // While the first copies are on their way: the items that the share has a
  // part of, the one it starts in (if that began before it or goes on after
  // it) and the one it ends in.
  auto find_splits = [&]() {
    if (tid >= 2) return;
    const Cursor& x = s_edge[tid];
    bool part = tid == 0 || end_b < p.batch;
    if (part) part = x.tiles > whole;  // (short ones lie in one share)
    if (part) {
      const bool same = x.b == end_b && x.item == end_item;
      part = tid == 0 ? x.tile > 0 || same
                      : x.tile > 0 && !(x.b == s_edge[0].b && x.item == s_edge[0].item);
    }
    if (!part) return;
    Split s;
    s.first = (int)cta_of(s_first[tid]);
    s.n = (int)cta_of(s_first[tid] + x.tiles - 1) - s.first + 1;
    const int head0 = (x.item % a.blocks) * M;
    s.row = x.b * p.q_heads + (int64_t)(x.item / a.blocks) * a.group + head0;
    s.heads = a.group - head0 < M ? a.group - head0 : M;
    s_split[tid] = s;
  };

  // q, O, maxima and sums: of a lane's rows of the products, or (plain FMAs) of
  // keys g, g + 8, .. and the dims of chunks t + 4 i, in parts of four
  uint32_t q_regs[F::kLanes ? 1 : F::kSteps][F::kQOps][4];
  float o_acc[F::kLanes ? 1 : F::kOTiles][4];
  constexpr int kChunks = F::kLanes ? D / 16 : 1, kHeads = F::kLanes ? M : 1;
  alignas(16) float q_lane[kHeads][kChunks][4], o_lane[kHeads][kChunks][4];
  auto lane_dim = [&](int part) {  // the first of part's four dims
    constexpr int kParts = F::kVec / 4;
    return (t + 4 * (part / kParts)) * F::kVec + part % kParts * 4;
  };
  constexpr int kMine = F::kLanes ? M : 1;  // heads of a lane
  float m_run[kMine], l_run[kMine], s_mul[kMine];
  int stage = 0;  // the next to fill
  int filled = 0;

  int seg = 0;  // tiles of the item in this share
  bool own = false;
  for (bool more = next_item(cur, seg, own, true); more;
       more = next_item(cur, seg, own, false)) {
    const int kv_head = cur.item / a.blocks, head0 = (cur.item % a.blocks) * M;
    const int heads = a.group - head0 < M ? a.group - head0 : M;
    const int64_t row = cur.b * p.q_heads + (int64_t)kv_head * a.group + head0;
    const int steps = own ? seg : (seg + kWarps - 1) / kWarps;
    int key0 = (cur.tile + (own ? 0 : w)) * F::kKeys;
    int end_key = (cur.tile + seg) * F::kKeys;
    if (end_key > cur.len) end_key = cur.len;

    for (int u = -1; u < steps;) {
      // fill a stage; the one to work on is the kStages - 1 filled before it
      if (filled == F::kStages - 1) cp_async_wait<F::kStages - 2>();
      __syncwarp();
      issue(stage);
      stage = stage + 1 == F::kStages ? 0 : stage + 1;
      if (filled < F::kStages - 1) {
        if (++filled == F::kStages - 1) find_splits();
        continue;
      }
      const uint8_t* tile = ring_ptr + stage * F::kStageBytes;
      if (u < 0) {
        // ---- the item's start: q in the order of the products' A operands,
        // the dims that lane t of step s multiplies; rows g and g + 8 are two
        // terms
        u = 0;
        auto q_at = [&](int d) {
          return to_f32(*reinterpret_cast<const A*>(
              tile + q_pos<F::kQRowChunks>(g, d * (int)sizeof(A) / 16) +
              d * (int)sizeof(A) % 16));
        };
        // FP32 q in f16 terms is scaled by a power of two that brings the
        // head's largest element to 2^14 .. 2^15: what falls below the f16
        // range is then below 2^-38 of it.  s_mul undoes it, with the softmax
        // scale.
        float q_mul[kMine];
#pragma unroll
        for (int r = 0; r < kMine; ++r) {
          m_run[r] = -INFINITY;
          l_run[r] = 0.0f;
          q_mul[r] = 1.0f;
          s_mul[r] = p.scale * kLog2e;
          if constexpr (!F::kLanes && !F::kF32 && !F::kBf16 && F32ACT) {
            float top = 0.0f;
#pragma unroll 4
            for (int d = t; d < D; d += 4) top = fmaxf(top, fabsf(q_at(d)));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (top > 0.0f && top < INFINITY) {
              int e;
              frexpf(top, &e);
              e = 15 - e < 120 ? 15 - e : 120;  // 2^e and 2^-e are normal
              q_mul[r] = __int_as_float((127 + e) << 23);
              s_mul[r] *= __int_as_float((127 - e) << 23);
            }
          }
        }
        if constexpr (F::kLanes) {
#pragma unroll
          for (int h = 0; h < M; ++h)
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = lane_dim(i) + e;
                q_lane[h][i][e] = to_f32(*reinterpret_cast<const A*>(
                    tile + q_pos<F::kQRowChunks>(h, d * (int)sizeof(A) / 16) +
                    d * (int)sizeof(A) % 16));
                o_lane[h][i][e] = 0.0f;
              }
            }
        } else {
#pragma unroll
          for (int s = 0; s < F::kSteps; ++s) {
            constexpr int kPart = F::kF32 ? 2 : 4;  // dims of a lane in a step
            const int d = (t + 4 * (s / (F::kVec / kPart))) * F::kVec + s % (F::kVec / kPart) * kPart;
            if constexpr (F::kF32) {
              split_tf32(q_at(d), q_regs[s][0][0], q_regs[s][0][1]);
              split_tf32(q_at(d + 1), q_regs[s][0][2], q_regs[s][0][3]);
            } else {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if constexpr (!F32ACT) {  // exact as it is
                  q_regs[s][0][2 * h] = *reinterpret_cast<const uint32_t*>(
                      tile + q_pos<F::kQRowChunks>(g, (d + 2 * h) * 2 / 16) + (d + 2 * h) * 2 % 16);
                  q_regs[s][0][1 + 2 * h] = 0u;
                } else {
                  float x = q_at(d + 2 * h) * q_mul[0], y = q_at(d + 2 * h + 1) * q_mul[0];
#pragma unroll
                  for (int k = 0; k < F::kQTerms; ++k)
                    q_regs[s][k / 2][k % 2 + 2 * h] = take_term<C>(x, y);
                  if (F::kQTerms % 2) q_regs[s][F::kQTerms / 2][1 + 2 * h] = 0u;
                }
              }
            }
          }
#pragma unroll
          for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[j][e] = 0.0f;
        }
        continue;
      }
      const int first_key = key0;
      key0 += (own ? 1 : kWarps) * F::kKeys;
      ++u;
      if (first_key >= end_key) continue;

      if constexpr (F::kLanes) {
        // ---- keys n * 8 + g of the tile, the dims of chunks t + 4 i
        constexpr int kSums = F::kNt == 1 ? 4 : 2;  // chains of a score
        float s[F::kNt][M][kSums];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int h = 0; h < M; ++h)
#pragma unroll
            for (int e = 0; e < kSums; ++e) s[n][h][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < F::kKIter; ++i)
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            alignas(16) uint32_t kw[4];
            *reinterpret_cast<uint4*>(kw) =
                *reinterpret_cast<const uint4*>(tile + chunk_pos<F::kRowBytes>(n * 8 + g, t + 4 * i));
#pragma unroll
            for (int e = 0; e < F::kVec; ++e) {
              const float x = chunk_value<C>(kw, e);
#pragma unroll
              for (int h = 0; h < M; ++h)
                s[n][h][e % kSums] =
                    fmaf(q_lane[h][i * (F::kVec / 4) + e / 4][e % 4], x, s[n][h][e % kSums]);
            }
          }
        float pr[F::kNt][M];
#pragma unroll
        for (int h = 0; h < M; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            float& x = pr[n][h];
            x = s[n][h][0] + s[n][h][1];
            if constexpr (kSums == 4) x += s[n][h][2] + s[n][h][3];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            x *= s_mul[h];
            if (first_key + n * 8 + g >= end_key) x = -INFINITY;
            top = fmaxf(top, x);
          }
          // each lane has a maximum of its own keys
          if (__any_sync(0xffffffffu, top > m_run[h] + kMaxSlack)) {
            top = fmaxf(top, m_run[h]);
            const float f = exp2_fast(m_run[h] - finite(top));
            m_run[h] = top;
            l_run[h] *= f;
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o_lane[h][i][e] *= f;
          }
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            pr[n][h] = exp2_fast(pr[n][h] - finite(m_run[h]));
            l_run[h] += pr[n][h];
          }
        }
#pragma unroll
        for (int i = 0; i < F::kKIter; ++i)
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            alignas(16) uint32_t vw[4];
            *reinterpret_cast<uint4*>(vw) = *reinterpret_cast<const uint4*>(
                tile + F::kKeys * F::kRowBytes + chunk_pos<F::kRowBytes>(n * 8 + g, t + 4 * i));
#pragma unroll
            for (int e = 0; e < F::kVec; ++e) {
              const float x = chunk_value<C>(vw, e);
#pragma unroll
              for (int h = 0; h < M; ++h) {
                float& o = o_lane[h][i * (F::kVec / 4) + e / 4][e % 4];
                o = fmaf(pr[n][h], x, o);
              }
            }
          }
        continue;
      } else {
      // ---- S = q k^T, in two chains for each 8 keys
      float s_acc[F::kNt][2][4];
#pragma unroll
      for (int n = 0; n < F::kNt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_acc[n][0][e] = s_acc[n][1][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < F::kKIter; ++i) {
        alignas(16) uint32_t kw[F::kNt][4];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
          *reinterpret_cast<uint4*>(kw[n]) = *reinterpret_cast<const uint4*>(
              tile + chunk_pos<F::kRowBytes>(n * 8 + g, t + 4 * i));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int s = 2 * i + e;
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            if constexpr (F::kF32) {
              const uint32_t x = kw[n][2 * e], y = kw[n][2 * e + 1];
              mma<C>(s_acc[n][0], q_regs[s][0], x, y);
              mma<C>(s_acc[n][1], q_regs[s][0], low_tf32(x), low_tf32(y));
            } else {
#pragma unroll
              for (int k = 0; k < F::kQOps; ++k)
                mma<C>(s_acc[n][F::kQOps == 2 ? k : e], q_regs[s][k], kw[n][2 * e], kw[n][2 * e + 1]);
            }
          }
        }
      }

      // ---- probabilities of keys n * 8 + 2 t and + 1; head g
      constexpr int kKSteps = F::kF32 ? F::kNt : F::kNt / 2;  // products over the tile's keys
      uint32_t pa[kKSteps][F::kPOps][4];
      {
        float v[F::kNt][2], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float(&x)[2][4] = s_acc[n];
            if constexpr (F::kQTerms == 1)
              v[n][e] = (x[0][e] + x[1][e]) * s_mul[0];
            else if constexpr (F::kF32)
              v[n][e] = with_rest(x[0][e], x[1][e] + (x[0][e + 2] + x[1][e + 2])) * s_mul[0];
            else if constexpr (F::kQTerms == 2)
              v[n][e] = with_rest(x[0][e] + x[1][e], x[0][e + 2] + x[1][e + 2]) * s_mul[0];
            else
              v[n][e] = with_rest(x[0][e], x[1][e] + x[0][e + 2]) * s_mul[0];
            if (first_key + n * 8 + 2 * t + e >= end_key) v[n][e] = -INFINITY;
            top = fmaxf(top, v[n][e]);
          }
        if (__any_sync(0xffffffffu, top > m_run[0] + (F::kBelow + kMaxSlack))) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top - F::kBelow, m_run[0]);
          const float f = exp2_fast(m_run[0] - finite(top));
          m_run[0] = top;
          l_run[0] *= f;
#pragma unroll
          for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[j][e] *= f;
        }
        const float m = finite(m_run[0]);
#pragma unroll
        for (int n = 0; n < F::kNt; ++n) {
          float x = exp2_fast(v[n][0] - m), y = exp2_fast(v[n][1] - m);
          l_run[0] += x + y;
          if constexpr (F::kF32) {
            split_tf32(x, pa[n][0][0], pa[n][0][1]);
            split_tf32(y, pa[n][0][2], pa[n][0][3]);
          } else {
            constexpr bool kCut = F::kPTerms == 3;
#pragma unroll
            for (int k = 0; k < 2; ++k)
              pa[n / 2][0][k + 2 * (n % 2)] = take_term<C, kCut>(x, y);
            if constexpr (kCut) {
              // it shares rows with the first term: positive, so that infinite
              // values times it have their own sign
              x = fmaxf(x, FLT_MIN);
              y = fmaxf(y, FLT_MIN);
              pa[n / 2][1][2 * (n % 2)] = take_term<C>(x, y);
              pa[n / 2][1][1 + 2 * (n % 2)] = 0u;
            }
          }
        }
      }

      // ---- O += P V.  The tensor cores cut sums off instead of rounding
      // them, which adds up over a long sequence (f16, 450 sequences of 524288
      // tokens, values about 1: 9.6e-4 of O, against 2.4e-4 at most of the output's
      // rounding), so each tile's product is formed by itself and added in FP32.
      const uint8_t* vt = tile + F::kKeys * F::kRowBytes;
#pragma unroll
      for (int i = 0; i < F::kVIter; ++i) {
        float c[F::kVVec][4];
#pragma unroll
        for (int e = 0; e < F::kVVec; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x)  // (the low part's sum may be cut off)
            c[e][x] = x >= 2 ? o_acc[i * F::kVVec + e][x] : 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
          constexpr int kV = F::kF32 ? 2 : 4;  // of the lane's keys in a product
          alignas(16) uint32_t vw[kV][4];
#pragma unroll
          for (int n = 0; n < kV; ++n) {
            const int r = ks * 4 * kV + (n / 2) * 8 + 2 * t + n % 2;
            if constexpr (F::kVVec == F::kVec)
              *reinterpret_cast<uint4*>(vw[n]) = *reinterpret_cast<const uint4*>(
                  vt + chunk_pos<F::kRowBytes>(r, g + 8 * i));
            else  // 64-byte rows: half a chunk to a lane
              *reinterpret_cast<uint2*>(vw[n]) = *reinterpret_cast<const uint2*>(
                  vt + chunk_pos<F::kRowBytes>(r, g >> 1) + (g & 1) * 8);
          }
#pragma unroll
          for (int e = 0; e < F::kVVec; ++e) {
            if constexpr (F::kF32) {
              const uint32_t x = vw[0][e], y = vw[1][e];
              mma<C>(c[e], pa[ks][0], finite_low_tf32<F::kKeys>(x), finite_low_tf32<F::kKeys>(y));
              mma<C>(c[e], pa[ks][0], x, y);
            } else {
              // element e of keys 2 t and 2 t + 1 (and 8 further) in one word
              const uint32_t pick = e % 2 ? 0x7632u : 0x5410u;
              const uint32_t b0 = __byte_perm(vw[0][e / 2], vw[1][e / 2], pick);
              const uint32_t b1 = __byte_perm(vw[2][e / 2], vw[3][e / 2], pick);
#pragma unroll
              for (int k = 0; k < F::kPOps; ++k) mma<C>(c[e], pa[ks][k], b0, b1);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < F::kVVec; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float& o = o_acc[i * F::kVVec + e][x];
            o = x < 2 ? o + c[e][x] : c[e][x];
          }
      }
      }
    }

    // ---- the item's end.  `each` passes the lane's part of O to its caller:
    // head, dim, four values times the head's factor
    if constexpr (F::kLanes) {
      // join the eight key groups: halve the chunks with the partner while
      // there are two or more, then add whole chunks
#pragma unroll
      for (int h = 0; h < M; ++h) {
        float top = m_run[h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float f = exp2_fast(m_run[h] - finite(top));
        m_run[h] = top;
        l_run[h] *= f;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], o);
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o_lane[h][i][e] *= f;
#pragma unroll
        for (int o = 16, n = kChunks; o >= 4; o >>= 1, n = n > 1 ? n / 2 : 1) {
          const bool upper = lane & o;
#pragma unroll
          for (int i = 0; i < (n > 1 ? n / 2 : 1); ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float keep = n > 1 && upper ? o_lane[h][n > 1 ? i + n / 2 : 0][e] : o_lane[h][i][e];
              const float give = n > 1 && !upper ? o_lane[h][n > 1 ? i + n / 2 : 0][e] : o_lane[h][i][e];
              o_lane[h][i][e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < kMine; ++r) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      }
    }
    if (cur.bad)
#pragma unroll
      for (int r = 0; r < kMine; ++r) l_run[r] = NAN;
    // this lane's head r, and whether the lane speaks for it
    auto head_of = [&](int r) { return F::kLanes ? r : g; };
    const bool speaks = F::kLanes ? lane == 0 : t == 0;
    auto each = [&](int r, float f, auto&& put) {
      if constexpr (F::kLanes) {
        // the chunk that the halvings left: the group's high bits; groups that
        // hold the same one leave it to the first
        constexpr int kSame = 8 / kChunks;
        const int d = lane_dim(g / kSame);
        if (g % kSame == 0) {
          const float(&o)[4] = o_lane[r][0];
          put(d, make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f));
        }
      } else {
        // lane (g, t) holds dims of chunks 2 t and 2 t + 1 (+ 8 i) of head g
#pragma unroll
        for (int i = 0; i < F::kVIter; ++i) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int e = 0; e < F::kVVec; e += 4) {
              float4 x;
              float* xs = reinterpret_cast<float*>(&x);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float(&o)[4] = o_acc[i * F::kVVec + e + k];
                xs[k] = with_rest(o[cc], o[cc + 2]) * f;
              }
              put((2 * t + cc + 8 * i) * F::kVVec + e, x);
            }
        }
      }
    };
    if (own) {
#pragma unroll
      for (int r = 0; r < kMine; ++r) {
        const int h = head_of(r);
        if (h >= heads) continue;
        const float f = l_run[r] == 0.0f ? 0.0f : 1.0f / l_run[r];
        each(r, f, [&](int d, float4 x) { store_act4(p.out, (row + h) * D + d, p.act_dtype, x); });
        if (speaks && p.lse) p.lse[row + h] = (m_run[r] + log2f(l_run[r])) * kLn2;
      }
    } else {
      const bool whole = cur.tile == 0 && seg == cur.tiles;
      const bool tail = cur.tile != 0;
      float* slot = a.partials + (2 * (int64_t)blockIdx.x + (tail ? 0 : 1)) * partial_floats(M, D);
      // the warps' O meet in the stages that they worked on last (the next
      // copies into those come after the joining)
      float* area = reinterpret_cast<float*>(smem + (w * F::kStages + stage) * F::kStageBytes);
      __syncwarp();
      if (lane == 0) s_area[w] = (w * F::kStages + stage) * F::kStageBytes;
#pragma unroll
      for (int r = 0; r < kMine; ++r) {
        const int h = head_of(r);
        if (speaks) {
          s_m[w][h] = m_run[r];
          s_l[w][h] = l_run[r];
        }
        each(r, 1.0f, [&](int d, float4 x) { *reinterpret_cast<float4*>(area + h * D + d) = x; });
      }
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < M * D / 4; i += kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float top = -INFINITY, sum = 0.0f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_m[k][h]);
        const float ref = finite(top);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(smem + s_area[k] + i * 16);
          const float f = exp2_fast(s_m[k][h] - ref);
          x.x = fmaf(y.x, f, x.x);
          x.y = fmaf(y.y, f, x.y);
          x.z = fmaf(y.z, f, x.z);
          x.w = fmaf(y.w, f, x.w);
          sum = fmaf(s_l[k][h], f, sum);
        }
        if (!whole) {
          *reinterpret_cast<float4*>(slot + h * D + d) = x;
          if (d == 0) {
            slot[M * D + h] = top;
            slot[M * D + M + h] = sum;
          }
        } else if (h < heads) {
          write_out(p, row + h, d, D, x, top, sum);
        }
      }
      __syncthreads();
    }
  }
  cp_async_wait<0>();

  // ---- the items this share has a part of: its first and its last at most.
  // Contributors of an item are CTAs `first` (its first tiles, odd slot) and on.
  // They join in a tree: the last of kFan neighbours to arrive joins their
  // partials into the first's and goes on to the next level with it.
  // Both items of a CTA climb together: a CTA that joins one would be late for
  // the other.
  __syncthreads();
  int c0[2], n[2], at[2];  // partials on this level (0: no part in it), this CTA's
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    n[e] = s_split[e].n;
    c0[e] = n[e] > 0 ? s_split[e].first : 0;
    at[e] = n[e] > 0 ? (int)blockIdx.x - c0[e] : 0;
  }
  for (int level = 0, span = 1; n[0] + n[1] > 0; ++level, span *= kFan) {
    int members[2];
    __syncthreads();
    if (tid == 0) {
      // Counts this CTA in; the one that completes a group leaves its counter
      // at zero for the next launch.  Writes made before by any CTA that was
      // counted are visible after.
      __threadfence();
      uint32_t old[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int first = at[e] / kFan * kFan;
        members[e] = n[e] - first < kFan ? n[e] - first : kFan;
        // a group of one needs no counter, so the first CTA names a group alone
        old[e] = members[e] > 1
                     ? atomicAdd(a.counters + level * kMaxCtas + c0[e] + first * span, 1u)
                     : 0u;
      }
      bool any = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool last = old[e] + 1 == (uint32_t)members[e];
        if (last && members[e] > 1)
          a.counters[level * kMaxCtas + c0[e] + at[e] / kFan * kFan * span] = 0u;
        s_last[e] = last;
        any = any || last;
      }
      if (any) __threadfence();
    }
    __syncthreads();
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      if (n[e] == 0) continue;
      const int first = at[e] / kFan * kFan, of = n[e] - first < kFan ? n[e] - first : kFan;
      const bool top = n[e] <= kFan;
      if (s_last[e] && of > 1)
        join_partials<M, D>(a, c0[e], first * span, span, of, !top, s_split[e].row,
                            s_split[e].heads);
      at[e] /= kFan;
      n[e] = top || !s_last[e] ? 0 : (n[e] + kFan - 1) / kFan;
    }
  }
}

template <class C, bool F32ACT, int D, int M>
int launch(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  using F = Cfg<C, F32ACT, D, M>;
  constexpr auto kernel = paged_attention_kernel<C, F32ACT, D, M>;
  const int rc = allow_shared<kernel>(F::kSmem, dev);
  if (rc != CT_OK) return rc;
  Launch b = a;
  b.blocks = (a.group + M - 1) / M;
  b.items = (int)(a.p.kv_heads * b.blocks);
  b.whole_tiles = a.p.kv.page_size % F::kRun == 0;
  // no more CTAs than the table can hold work for
  const int64_t keys = a.p.kv.max_pages * a.p.kv.page_size;
  const int64_t tiles =
      a.p.batch * b.items * (kItemCost + (keys > F::kKeys ? (keys + F::kKeys - 1) / F::kKeys : 1));
  int64_t ctas = (int64_t)dev.sm_count * F::kCtas;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (ctas > (tiles + kMinShare - 1) / kMinShare) ctas = (tiles + kMinShare - 1) / kMinShare;
  // One sequence: as many whole CTAs to each item, so that none works on two
  // (the one that does ends some 3 us after the others): 8192 tokens 19.5 us
  // against 23.3, 131072 92.5 against 95.7.
  if (a.p.batch == 1 && b.items <= ctas / 8) ctas -= ctas % b.items;
  kernel<<<(unsigned)ctas, kThreads, F::kSmem, st>>>(b);
  return check_launch();
}

constexpr size_t kCounterBytes = CT_PAGED_ATTENTION_COUNTER_BYTES;
static_assert(kLevels * kMaxCtas * sizeof(uint32_t) <= kCounterBytes, "");

// Groups of more than 8 heads are blocks of 8, for each of which the cache is
// read again, mostly from L2.  (16 heads at a time, a product's rows filled by
// one term, spilled registers and was slower but for the most ragged batch:
// 16 heads on one, 32 x 4096 tokens, in bf16 of 128 46.2 us against 28.6, in
// FP32 of 64 45.2 against 36.9; f16 of 64, 128 x 1 .. 16384 27.5 against 28.7.)
template <class C, bool F32ACT, int D>
int launch_heads(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  // One head: plain FMAs.  (FP32, 8 on 8, 8 x 4096 tokens: 53 us against 72 of
  // the tensor cores at 128 dims, 34 against 42 at 64; 32 on 32 of 64, FP32 q on
  // bf16: 82 against 98.)
  if (a.group == 1) return launch<C, F32ACT, D, 1>(a, dev, st);
  // Two: where q would take three terms or the cache is FP32.  (16 on 8 of 64,
  // 32 x 4096, FP32 q on bf16: 54 us against 62; 16-bit q, and FP32 q on f16,
  // take 54 to 55 either way, at 32 dims 63.)
  if constexpr (sizeof(C) == 4 || (q_terms<C, F32ACT>() == 3 && D <= 64))
    if (a.group == 2) return launch<C, F32ACT, D, 2>(a, dev, st);
  return launch<C, F32ACT, D, 8>(a, dev, st);
}

template <class C, bool F32ACT>
int launch_dims(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  if (a.p.head_dim == 32) return launch_heads<C, F32ACT, 32>(a, dev, st);
  if (a.p.head_dim == 64) return launch_heads<C, F32ACT, 64>(a, dev, st);
  return launch_heads<C, F32ACT, 128>(a, dev, st);
}

}  // namespace

size_t paged_attention_workspace(int64_t head_dim) {
  return kCounterBytes + 2 * kMaxCtas * sizeof(float) * partial_floats(8, (int)head_dim);
}

int launch_paged_attention(const PagedAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  Launch a{};
  a.p = p;
  if (p.q_heads >= (1ll << 30)) return CT_ERR_INVALID_ARGUMENT;
  a.group = (int)(p.q_heads / p.kv_heads);
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (p.kv.page_size == 1 << s) a.page_shift = s;
  const int q_vec = 16 / dtype_bytes(p.act_dtype);
  a.q_vectors = aligned16(p.q) && p.qs[0] % q_vec == 0 && p.qs[1] % q_vec == 0 && p.qs[2] == 1;
  a.counters = static_cast<uint32_t*>(p.ws);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(p.ws) + kCounterBytes);
  return with_dtype(p.kv.dtype, [&](auto c) {
    using C = decltype(c);
    if (p.act_dtype == CT_DTYPE_F32) return launch_dims<C, true>(a, dev, st);
    if constexpr (sizeof(C) == 2) return launch_dims<C, false>(a, dev, st);
    return (int)CT_ERR_INVALID_ARGUMENT;
  });
}

}  // namespace ct
