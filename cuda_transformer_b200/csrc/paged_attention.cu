// paged_attention.cu -- attention of one new token per sequence over a paged
// key/value cache:
//   s_j = scale q . k_j,  O = sum_j softmax(s)_j v_j,  L = ln sum_j exp(s_j)
// over the sequence's cached tokens j; O = 0 and L = -inf when there are none.
// Query heads share key/value heads in groups of q_heads / kv_heads.
//
// Every cached value is read once and used for 2 * group FLOPs, so the bound
// is HBM.  The design follows from that:
//  * Work is cut into units of a few dozen keys of one (sequence, key/value
//    head), and every CTA takes an equal share of the units, counted on the
//    device from seq_lens (the host knows no lengths).  Ragged batches and one
//    long sequence load the GPU alike.  A share that starts or ends inside a
//    sequence leaves a partial (max, sum, O) in the workspace; the CTA that
//    arrives last joins the partials in their order, so results do not depend
//    on timing and no CTA waits for another.
//  * Each warp streams its own keys through a private cp.async ring (16-byte
//    copies gather pages of any size and layout), across sequence borders, with
//    no block barrier until a sequence's end.
//  * Products run on mma.sync m16n8k8 TF32 with FP32 accuracy: 8 heads fill
//    rows 0-7 with the high part of q (or of the probabilities) and rows 8-15
//    with the low part.  16-bit cache values are exact in TF32; FP32 ones are
//    split too.  High and low sums of a head sit in the same lane, and the
//    order of keys and dims inside a product is chosen so that every operand
//    is a 16-byte shared-memory vector: no shuffles, no transposes.  tcgen05
//    would take 8 heads as 128 rows (or as a column operand that has to be
//    written to shared memory); at 4 * group FLOPs a value the tensor pipe is
//    not what bounds this kernel.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCtas = 448;  // counters (two levels) and partial slots in the workspace
constexpr int kGroup = 16;     // partials that are joined at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is raised only when a score passes it by this much (in
// powers of two): probabilities stay below 2^6, which FP32 sums hold as well
// as values below 1, and most tiles skip the rescaling of O.
constexpr float kMaxSlack = 6.0f;

// C: the cache's type; F32ACT: q and out are FP32, else of type C; R: blocks
// of 8 query heads a CTA works on (1: high and low parts share a product's
// rows; 2: 16 heads fill them and the parts are products of their own).
template <class C, bool F32ACT, int D, int R>
struct Cfg {
  static constexpr bool kF32 = sizeof(C) == 4;
  static constexpr bool kBf16 = std::is_same<C, __nv_bfloat16>::value;
  static constexpr int kVec = 16 / (int)sizeof(C);          // elements of a 16-byte chunk
  static constexpr int kKeys = kF32 ? 8 : 16;                // keys of a warp's tile
  static constexpr int kNt = kKeys / 8;
  static constexpr int kUnit = kWarps * kKeys;               // keys of a work unit
  static constexpr int kRowBytes = D * (int)sizeof(C);
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kCopies = kKeys * kRowChunks / 32;    // of a lane, for K or V
  static constexpr int kCopyRows = 32 / kRowChunks;          // rows of one copy instruction
  static constexpr int kStageBytes = 2 * kKeys * kRowBytes;  // K tile, V tile
  static constexpr int kKIter = D / (4 * kVec);              // K chunks a lane reads per key
  static constexpr int kVVec = kVec < D / 8 ? kVec : D / 8;  // V elements a lane reads at once
  static constexpr int kVIter = D / (8 * kVVec);
  static constexpr int kOTiles = D / 8;
  // Terms q and the probabilities are split into.  With 16-bit activations q
  // is exact as it is, and two terms of p leave an error (2^-16 in bf16) far
  // below the output's own rounding; FP32 activations take as many as hold 22
  // bits or more.
  static constexpr int kQTerms = kF32 ? 2 : !F32ACT ? 1 : kBf16 ? 3 : 2;
  static constexpr int kPTerms = F32ACT && kBf16 ? 3 : 2;
  // The exponent's base lies this far below the running maximum (in powers of
  // two): f16 probabilities reach up to 2^14 instead of 1, so that the many
  // small ones of a long sequence stay clear of the subnormals.
  static constexpr float kBelow = !kF32 && !kBf16 ? 8.0f : 0.0f;
  // A operands of one step (8 dims in TF32, 16 in the 16-bit types).  R = 1:
  // rows 0-7 and 8-15 hold two terms; R = 2: one term of 16 heads.
  static constexpr int kQOps = R == 1 ? (kQTerms + 1) / 2 : kQTerms;
  static constexpr int kPOps = R == 1 ? (kPTerms + 1) / 2 : kPTerms;
  static constexpr int kSteps = kF32 ? D / 8 : D / 16;
  static constexpr int kQRegs = kSteps * kQOps * 4;
  static constexpr bool kQInRegs = kQRegs <= 64;             // else in shared memory
  // Registers: q, O (D / 2) and about 72 more.  Three CTAs an SM where that
  // fits 168 a thread, with two stages of 8 KB or as many smaller ones.
  static constexpr int kCtas = (kQInRegs ? kQRegs : 0) + D / 2 + 72 <= 168 ? 3 : 2;
  static constexpr int kRing = kCtas == 3 ? 16384 : 24576;
  static constexpr int kStages = kRing / kStageBytes > 6 ? 6 : kRing / kStageBytes;
  static constexpr int kJoinDims = D < 64 ? D : 64;          // dims of one joining pass
  static constexpr int kJoinBytes = kWarps * 8 * kJoinDims * 4;
  static constexpr int kQBytes = kQInRegs ? 0 : kQRegs * 32 * 4;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kSmem = kRingBytes + (kJoinBytes > kQBytes ? kJoinBytes : kQBytes);
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

__device__ __forceinline__ void store_act4(void* p, int64_t i, int dtype, float4 x) {
  if (dtype == CT_DTYPE_F32) {
    *reinterpret_cast<float4*>((float*)p + i) = x;
  } else if (dtype == CT_DTYPE_BF16) {
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(x.x, x.y), __floats2bfloat162_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>((__nv_bfloat16*)p + i) = *reinterpret_cast<uint2*>(v);
  } else {
    __half2 v[2] = {__floats2half2_rn(x.x, x.y), __floats2half2_rn(x.z, x.w)};
    *reinterpret_cast<uint2*>((__half*)p + i) = *reinterpret_cast<uint2*>(v);
  }
}

// Floats of a partial: O [heads][D], then maximum and sum [heads] each.
constexpr int64_t partial_floats(int heads, int D) { return (int64_t)heads * (D + 2); }

struct Launch {
  PagedAttention p;
  int group, blocks;  // query heads of a key/value head; its blocks of 8 R heads
  int items;          // (key/value head, block) pairs of a sequence
  int page_shift;     // log2 of page_size, -1 when it is no power of two
  bool whole_tiles;   // a tile's keys lie in one page
  uint32_t* counters;
  float* partials;
};

// Where a CTA stands in the list of units: sequence, item, unit in the item.
struct Cursor {
  int64_t b;
  int item, unit, units, len;
  bool bad;
};

template <int UNIT>
__device__ __forceinline__ void read_length(const Launch& a, Cursor& c) {
  const int n = a.p.seq_lens[c.b];
  c.bad = n > a.p.kv.max_pages * a.p.kv.page_size;
  c.len = n < 0 || c.bad ? 0 : n;
  c.units = c.len > UNIT ? (c.len + UNIT - 1) / UNIT : 1;  // one, empty, at length 0
}
template <int UNIT>
__device__ __forceinline__ void advance(const Launch& a, Cursor& c) {
  if (++c.unit < c.units) return;
  c.unit = 0;
  if (++c.item < a.items) return;
  c.item = 0;
  if (++c.b < a.p.batch) read_length<UNIT>(a, c);
}

// A head's result from its unnormalised O and its maximum and sum.
__device__ __forceinline__ void write_out(const PagedAttention& p, int64_t row, int d, int D,
                                          float4 x, float m, float l) {
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  store_act4(p.out, row * D + d, p.act_dtype, make_float4(x.x * r, x.y * r, x.z * r, x.w * r));
  if (d == 0 && p.lse) p.lse[row] = (m + log2f(l)) * kLn2;
}

__device__ __forceinline__ float exp2_diff(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2f(m - top);
}

// Counts a CTA in; true in all threads of the one that completes `n`, which
// leaves the counter at zero for the next launch.  Writes made before it by
// any CTA that was counted are visible after it.
__device__ __forceinline__ bool arrive_last(uint32_t* counter, int n, int* flag) {
  if (threadIdx.x == 0) {
    __threadfence();
    const bool last = atomicAdd(counter, 1u) == (uint32_t)(n - 1);
    if (last) *counter = 0u;
    *flag = last;
    __threadfence();
  }
  __syncthreads();
  return *flag != 0;
}

// Joins the partials k0, k0 + step, .. (n of them) of the item that CTA c0
// starts, in that order, eight loads in flight: into partial k0 or the output.
template <int HEADS, int D>
__device__ void join_partials(const Launch& a, int64_t c0, int k0, int step, int n, bool to_partial,
                              int64_t row, int heads) {
  constexpr int64_t kSize = partial_floats(HEADS, D);
  constexpr int kBatch = 8;
  auto at = [&](int k) { return a.partials + (k == 0 ? 2 * c0 + 1 : 2 * (c0 + k)) * kSize; };
  for (int i = threadIdx.x; i < HEADS * D / 4; i += kThreads) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = 0; b < n; b += kBatch) {
      float km[kBatch], kl[kBatch];
      float4 y[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        km[j] = -INFINITY;
        kl[j] = 0.0f;
        y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (b + j < n) {
          const float* s = at(k0 + (b + j) * step);
          km[j] = __ldcg(s + HEADS * D + h);
          kl[j] = __ldcg(s + HEADS * D + HEADS + h);
          y[j] = __ldcg(reinterpret_cast<const float4*>(s + h * D + d));
        }
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) top = fmaxf(top, km[j]);
      const float f0 = exp2_diff(m, top);
      m = top;
      l *= f0;
      x.x *= f0;
      x.y *= f0;
      x.z *= f0;
      x.w *= f0;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float f = exp2_diff(km[j], top);
        x.x = fmaf(y[j].x, f, x.x);
        x.y = fmaf(y[j].y, f, x.y);
        x.z = fmaf(y[j].z, f, x.z);
        x.w = fmaf(y[j].w, f, x.w);
        l = fmaf(kl[j], f, l);
      }
    }
    if (to_partial) {
      // heads' maxima and sums are read by all threads of the head: write
      // them after everyone has read
      float* s = at(k0);
      __syncwarp();
      *reinterpret_cast<float4*>(s + h * D + d) = x;
      if (d == 0) {
        s[HEADS * D + h] = m;
        s[HEADS * D + HEADS + h] = l;
      }
    } else if (h < heads) {
      write_out(a.p, row + h, d, D, x, m, l);
    }
  }
}

template <class C, bool F32ACT, int D, int R>
__global__ void __launch_bounds__(kThreads, Cfg<C, F32ACT, D, R>::kCtas)
    paged_attention_kernel(const __grid_constant__ Launch a) {
  using F = Cfg<C, F32ACT, D, R>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_scan[kWarps];
  __shared__ Cursor s_start;
  __shared__ float s_m[kWarps][8 * R], s_l[kWarps][8 * R];
  __shared__ int s_last;
  const int tid = threadIdx.x, w = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const PagedAttention& p = a.p;

  // ---- this CTA's share of the units
  int64_t mine = 0;
  for (int64_t b = tid; b < p.batch; b += kThreads) {
    Cursor c;
    c.b = b;
    read_length<F::kUnit>(a, c);
    mine += c.units;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_scan[w] = mine;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) total += s_scan[i];
  total *= a.items;
  const int64_t ctas = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= ctas) return;
  const int64_t first = total * blockIdx.x / ctas, last = total * (blockIdx.x + 1) / ctas;
  __syncthreads();
  for (int64_t b0 = 0, before = 0; b0 < p.batch; b0 += kThreads) {
    Cursor c{};
    c.b = b0 + tid;
    if (c.b < p.batch) read_length<F::kUnit>(a, c);
    int64_t upto = c.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s_scan[w] = upto;
    __syncthreads();
    int64_t chunk = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      if (i < w) upto += s_scan[i];
      chunk += s_scan[i];
    }
    const int64_t from = first - (before + upto - c.units) * a.items;
    if (from >= 0 && from < (int64_t)c.units * a.items) {
      c.item = (int)(from / c.units);
      c.unit = (int)(from % c.units);
      s_start = c;
    }
    before += chunk;
    __syncthreads();
    if (before * a.items > first) break;
  }
  Cursor cur = s_start, ahead = cur;

  // ---- the copy side: tiles of this warp, kStages - 1 ahead of the products
  const uint32_t ring = smem_addr(smem) + w * (F::kStages * F::kStageBytes);
  const uint8_t* ring_ptr = smem + w * (F::kStages * F::kStageBytes);
  const bool second = (lane / F::kKeys) & 1;  // this lane addresses V rows, else K rows
  const int my_row = lane % F::kKeys;
  // The lane's part of a copy instruction: row copy_row + i * kCopyRows, chunk
  // lane % kRowChunks.  The row's bits and i's do not meet, so the chunk's
  // position is the xor of a part of each (chunk_pos).
  const int copy_row = lane / F::kRowChunks, copy_chunk = lane % F::kRowChunks;
  const int64_t k_step = p.kv.ks[2] * (int64_t)sizeof(C), v_step = p.kv.vs[2] * (int64_t)sizeof(C);
  const uint8_t* k_lane = (const uint8_t*)p.kv.k + copy_row * k_step + copy_chunk * 16;
  const uint8_t* v_lane = (const uint8_t*)p.kv.v + copy_row * v_step + copy_chunk * 16;
  int64_t to_issue = last - first;
  int next_page = -1, next_slot = 0, next_head = 0;
  bool next_there = false;
  auto look_up = [&]() {  // page and slot of the lane's row of the next tile
    next_there = false;
    if (to_issue <= 0) return;
    const int key = ahead.unit * F::kUnit + w * F::kKeys + my_row;
    next_there = key < ahead.len;
    if (next_there) {
      const int index = a.page_shift >= 0 ? key >> a.page_shift : key / p.kv.page_size;
      next_slot = key - index * p.kv.page_size;
      next_page = p.kv.table[ahead.b * p.kv.table_s + index];
      next_head = ahead.item / a.blocks;
    }
    --to_issue;
    if (to_issue > 0) advance<F::kUnit>(a, ahead);
  };
  auto issue = [&](int stage) {
    const bool fine = next_there && (unsigned)next_page < (unsigned)p.kv.pages;
    const uint32_t base = ring + stage * F::kStageBytes;
    if (a.whole_tiles && __all_sync(0xffffffffu, fine)) {
      // all rows are there and follow one another in one page
      const int slot = next_slot - my_row;
      const uint8_t* src[2] = {
          k_lane + (next_page * p.kv.ks[0] + next_head * p.kv.ks[1]) * (int64_t)sizeof(C) + slot * k_step,
          v_lane + (next_page * p.kv.vs[0] + next_head * p.kv.vs[1]) * (int64_t)sizeof(C) + slot * v_step};
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int64_t step = F::kCopyRows * (kv ? v_step : k_step);
        const uint32_t dst = base + kv * (F::kKeys * F::kRowBytes);
#pragma unroll
        for (int i = 0; i < F::kCopies; ++i)
          cp_async16(dst + chunk_pos<F::kRowBytes>(i * F::kCopyRows + copy_row, copy_chunk),
                     src[kv] + i * step, 16);
      }
    } else if (__any_sync(0xffffffffu, next_there)) {
      int64_t off = -1;  // past the length: zeros
      if (next_there) {
        const int64_t* s = second ? p.kv.vs : p.kv.ks;
        off = !fine ? -2  // no such page: NaN keys
                    : (next_page * s[0] + next_head * s[1] + next_slot * s[2]) * (int64_t)sizeof(C);
      }
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* from = (const uint8_t*)(kv ? p.kv.v : p.kv.k);
#pragma unroll
        for (int i = 0; i < F::kCopies; ++i) {
          const int r = i * F::kCopyRows + copy_row;
          const int64_t o = __shfl_sync(0xffffffffu, off, kv * F::kKeys + r);
          const uint32_t dst =
              base + kv * (F::kKeys * F::kRowBytes) + chunk_pos<F::kRowBytes>(r, copy_chunk);
          if (o == -2)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0x7fc07fc0u)
                         : "memory");  // NaN in each of the three types
          else
            cp_async16(dst, o < 0 ? from : from + o + copy_chunk * 16, o < 0 ? 0 : 16);
        }
      }
    }
    cp_async_commit();
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < F::kStages - 1; ++s) issue(s);

  float* join = reinterpret_cast<float*>(smem + F::kRingBytes);
  uint32_t* q_smem = reinterpret_cast<uint32_t*>(smem + F::kRingBytes);
  uint32_t q_regs[F::kQInRegs ? F::kSteps : 1][F::kQOps][4];
  int stage = 0;

  for (int64_t at = first; at < last;) {
    // ---- one segment: units cur.unit .. end of the item, or of the share
    const int kv_head = cur.item / a.blocks, head0 = (cur.item % a.blocks) * 8 * R;
    const int heads = a.group - head0 < 8 * R ? a.group - head0 : 8 * R;
    const int64_t q_head = (int64_t)kv_head * a.group + head0;
    const int64_t item_first = at - cur.unit;
    const int seg = (int)(last - at < cur.units - cur.unit ? last - at : cur.units - cur.unit);

    // q in the order of the products' A operands: the dims that lane t of step
    // s multiplies; rows g and g + 8 are two terms (R = 1) or two heads.
    using A = std::conditional_t<F32ACT, float, C>;
    const A* q_row[R];
#pragma unroll
    for (int r = 0; r < R; ++r)  // a head past the group's last reads another's row, and then zero
      q_row[r] = (const A*)p.q + cur.b * p.qs[0] +
                 (q_head + (r * 8 + g < heads ? r * 8 + g : 0)) * p.qs[1];
    auto q_at = [&](int r, int d) {
      const float x = to_f32(q_row[r][d * p.qs[2]]);
      return r * 8 + g < heads ? x : 0.0f;
    };
    // FP32 q in f16 terms is scaled by a power of two that brings the head's
    // largest element to 2^14 .. 2^15: what falls below the f16 range is then
    // below 2^-38 of it.  s_mul undoes it, with the softmax scale.
    float s_mul[R], q_mul[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      q_mul[r] = 1.0f;
      s_mul[r] = p.scale * kLog2e;
      if constexpr (!F::kF32 && !F::kBf16 && F32ACT) {
        float top = 0.0f;
#pragma unroll
        for (int d = t; d < D; d += 4) top = fmaxf(top, fabsf(q_at(r, d)));
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
    auto q_ops = [&](int s, uint32_t (&op)[F::kQOps][4]) {
      const int i = s / (F::kVec / (F::kF32 ? 2 : 4)), e = s % (F::kVec / (F::kF32 ? 2 : 4));
      const int d = (t + 4 * i) * F::kVec + e * (F::kF32 ? 2 : 4);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (F::kF32) {
          uint32_t term[2][2];
          split_tf32(q_at(r, d), term[0][0], term[1][0]);
          split_tf32(q_at(r, d + 1), term[0][1], term[1][1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            op[R == 1 ? 0 : k][R == 1 ? k : r] = term[k][0];
            op[R == 1 ? 0 : k][(R == 1 ? k : r) + 2] = term[k][1];
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = q_at(r, d + 2 * h) * q_mul[r];
            float y = q_at(r, d + 2 * h + 1) * q_mul[r];
#pragma unroll
            for (int k = 0; k < F::kQTerms; ++k)
              op[R == 1 ? k / 2 : k][(R == 1 ? k % 2 : r) + 2 * h] = take_term<C>(x, y);
            if (R == 1 && F::kQTerms % 2) op[F::kQTerms / 2][1 + 2 * h] = 0u;
          }
        }
      }
    };
    if constexpr (F::kQInRegs) {
#pragma unroll
      for (int s = 0; s < F::kSteps; ++s) q_ops(s, q_regs[s]);
    } else {
      for (int s = w; s < F::kSteps; s += kWarps) {
        uint32_t op[F::kQOps][4];
        q_ops(s, op);
#pragma unroll
        for (int k = 0; k < F::kQOps; ++k)
          *reinterpret_cast<uint4*>(q_smem + ((s * F::kQOps + k) * 32 + lane) * 4) =
              make_uint4(op[k][0], op[k][1], op[k][2], op[k][3]);
      }
      __syncthreads();
    }

    float o_acc[F::kOTiles][4], m_run[R], l_run[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m_run[r] = -INFINITY;
      l_run[r] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o_acc[j][e] = 0.0f;

    for (int u = 0; u < seg; ++u) {
      cp_async_wait<F::kStages - 2>();
      __syncwarp();
      issue(stage == 0 ? F::kStages - 1 : stage - 1);
      const int key0 = (cur.unit + u) * F::kUnit + w * F::kKeys;
      const uint8_t* tile = ring_ptr + stage * F::kStageBytes;
      stage = stage + 1 == F::kStages ? 0 : stage + 1;
      if (key0 >= cur.len) continue;

      // ---- S = q k^T, in two chains for each 8 keys
      float s_acc[F::kNt][2][4];
#pragma unroll
      for (int n = 0; n < F::kNt; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_acc[n][0][e] = s_acc[n][1][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < F::kKIter; ++i) {
        uint32_t kw[F::kNt][4];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
          *reinterpret_cast<uint4*>(kw[n]) = *reinterpret_cast<const uint4*>(
              tile + chunk_pos<F::kRowBytes>(n * 8 + g, t + 4 * i));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int s = 2 * i + e;
          uint32_t qa[F::kQOps][4];
#pragma unroll
          for (int k = 0; k < F::kQOps; ++k) {
            if constexpr (F::kQInRegs) {
#pragma unroll
              for (int x = 0; x < 4; ++x) qa[k][x] = q_regs[s][k][x];
            } else {
              *reinterpret_cast<uint4*>(qa[k]) =
                  *reinterpret_cast<const uint4*>(q_smem + ((s * F::kQOps + k) * 32 + lane) * 4);
            }
          }
#pragma unroll
          for (int n = 0; n < F::kNt; ++n) {
            if constexpr (F::kF32) {
              uint32_t xh, xl, yh, yl;
              split_tf32(__uint_as_float(kw[n][2 * e]), xh, xl);
              split_tf32(__uint_as_float(kw[n][2 * e + 1]), yh, yl);
              mma<C>(s_acc[n][0], qa[0], xh, yh);
              mma<C>(s_acc[n][1], qa[0], xl, yl);
              if constexpr (R == 2) mma<C>(s_acc[n][1], qa[1], xh, yh);
            } else {
#pragma unroll
              for (int k = 0; k < F::kQOps; ++k)
                mma<C>(s_acc[n][(e + k) & 1], qa[k], kw[n][2 * e], kw[n][2 * e + 1]);
            }
          }
        }
      }

      // ---- probabilities of keys n * 8 + 2 t and + 1; heads g (and g + 8)
      uint32_t pa[F::kPOps][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float v[F::kNt][2], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float(&x)[2][4] = s_acc[n];
            v[n][e] = R == 1 ? (x[0][e] + x[1][e]) + (x[0][e + 2] + x[1][e + 2])
                             : x[0][2 * r + e] + x[1][2 * r + e];
            v[n][e] *= s_mul[r];
            if (key0 + n * 8 + 2 * t + e >= cur.len) v[n][e] = -INFINITY;
            top = fmaxf(top, v[n][e]);
          }
        if (__any_sync(0xffffffffu, top > m_run[r] + (F::kBelow + kMaxSlack))) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top - F::kBelow, m_run[r]);
          const float f = exp2_diff(m_run[r], top);
          m_run[r] = top;
          l_run[r] *= f;
#pragma unroll
          for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (R == 1 || e / 2 == r) o_acc[j][e] *= f;
        }
        const float m = m_run[r] == -INFINITY ? 0.0f : m_run[r];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n) {
          float x = exp2f(v[n][0] - m), y = exp2f(v[n][1] - m);
          l_run[r] += x + y;
          if constexpr (F::kF32) {
            uint32_t term[2][2];
            split_tf32(x, term[0][0], term[1][0]);
            split_tf32(y, term[0][1], term[1][1]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              pa[R == 1 ? 0 : k][R == 1 ? k : r] = term[k][0];
              pa[R == 1 ? 0 : k][(R == 1 ? k : r) + 2] = term[k][1];
            }
          } else {
#pragma unroll
            for (int k = 0; k < F::kPTerms; ++k)
              pa[R == 1 ? k / 2 : k][(R == 1 ? k % 2 : r) + 2 * n] = take_term<C>(x, y);
            if (R == 1 && F::kPTerms % 2) pa[F::kPTerms / 2][1 + 2 * n] = 0u;
          }
        }
      }

      // ---- O += P V.  The tensor cores cut sums off instead of rounding
      // them, which adds up over a long sequence; with FP32 outputs each
      // tile's product is therefore formed by itself and added in FP32.
      const uint8_t* vt = tile + F::kKeys * F::kRowBytes;
#pragma unroll
      for (int i = 0; i < F::kVIter; ++i) {
        uint32_t vw[2 * F::kNt][4];
#pragma unroll
        for (int n = 0; n < 2 * F::kNt; ++n) {
          const int r = (n / 2) * 8 + 2 * t + n % 2;
          if constexpr (F::kVVec == F::kVec)
            *reinterpret_cast<uint4*>(vw[n]) = *reinterpret_cast<const uint4*>(
                vt + chunk_pos<F::kRowBytes>(r, g + 8 * i));
          else  // 64-byte rows: half a chunk to a lane
            *reinterpret_cast<uint2*>(vw[n]) = *reinterpret_cast<const uint2*>(
                vt + chunk_pos<F::kRowBytes>(r, g >> 1) + (g & 1) * 8);
        }
#pragma unroll
        for (int e = 0; e < F::kVVec; ++e) {
          float(&o)[4] = o_acc[i * F::kVVec + e];
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (!F32ACT) {
#pragma unroll
            for (int x = 0; x < 4; ++x) c[x] = o[x];
          } else if constexpr (R == 1) {  // the low part's sum may be cut off
            c[2] = o[2];
            c[3] = o[3];
          }
          if constexpr (F::kF32) {
            uint32_t xh, xl, yh, yl;
            split_tf32(__uint_as_float(vw[0][e]), xh, xl);
            split_tf32(__uint_as_float(vw[1][e]), yh, yl);
            mma<C>(c, pa[0], xh, yh);
            mma<C>(c, pa[0], xl, yl);
            if constexpr (R == 2) mma<C>(c, pa[1], xh, yh);
          } else {
            // element e of keys 2 t and 2 t + 1 (and 8 further) in one word
            const uint32_t pick = e % 2 ? 0x7632u : 0x5410u;
            const uint32_t b0 = __byte_perm(vw[0][e / 2], vw[1][e / 2], pick);
            const uint32_t b1 = __byte_perm(vw[2][e / 2], vw[3][e / 2], pick);
#pragma unroll
            for (int k = 0; k < F::kPOps; ++k) mma<C>(c, pa[k], b0, b1);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) o[x] = F32ACT && (R == 2 || x < 2) ? o[x] + c[x] : c[x];
        }
      }
    }

    // ---- the segment's end: join the warps, then write O or a partial
    const bool whole = cur.unit == 0 && seg == cur.units;
    const bool tail = cur.unit != 0;
    float* slot =
        a.partials + (2 * (int64_t)blockIdx.x + (tail ? 0 : 1)) * partial_floats(8 * R, D);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float l = l_run[r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) {
        s_m[w][r * 8 + g] = m_run[r];
        s_l[w][r * 8 + g] = l;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s_m[i][r * 8 + g]);
      const float f = exp2_diff(m_run[r], top);
      constexpr int J = F::kJoinDims, kPassIter = J / (8 * F::kVVec);
#pragma unroll
      for (int pass = 0; pass < D / J; ++pass) {
        // lane (g, t) holds dims of chunks 2 t and 2 t + 1 (+ 8 i) of head g
#pragma unroll
        for (int i = 0; i < kPassIter; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < F::kVVec; e += 4) {
              float4 x;
              float* xs = reinterpret_cast<float*>(&x);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float(&o)[4] = o_acc[(pass * kPassIter + i) * F::kVVec + e + k];
                xs[k] = (R == 1 ? o[c] + o[c + 2] : o[2 * r + c]) * f;
              }
              *reinterpret_cast<float4*>(join + (w * 8 + g) * J + (2 * t + c + 8 * i) * F::kVVec +
                                         e) = x;
            }
        __syncthreads();
        for (int i = tid; i < 8 * J / 4; i += kThreads) {
          const int h = i / (J / 4), dj = i % (J / 4) * 4, d = pass * J + dj;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          float hm = -INFINITY, hl = 0.0f;
#pragma unroll
          for (int k = 0; k < kWarps; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(join + (k * 8 + h) * J + dj);
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            x.w += y.w;
            hm = fmaxf(hm, s_m[k][r * 8 + h]);
          }
#pragma unroll
          for (int k = 0; k < kWarps; ++k)
            hl += s_l[k][r * 8 + h] * exp2_diff(s_m[k][r * 8 + h], hm);
          if (cur.bad) hl = NAN;
          if (!whole) {
            *reinterpret_cast<float4*>(slot + (r * 8 + h) * D + d) = x;
            if (d == 0) {
              slot[8 * R * D + r * 8 + h] = hm;
              slot[8 * R * D + 8 * R + r * 8 + h] = hl;
            }
          } else if (r * 8 + h < heads) {
            write_out(p, cur.b * p.q_heads + q_head + r * 8 + h, d, D, x, hm, hl);
          }
        }
        __syncthreads();
      }
    }

    if (!whole) {
      // Contributors of this item: CTAs c0 (its first units, odd slot) .. c1.
      // The last of each kGroup to arrive joins the group's partials into the
      // group's first, the last group to arrive joins those: a few loads in
      // flight at a time for one CTA, however many CTAs share the item.
      const int64_t c0 = ((item_first + 1) * ctas - 1) / total;
      const int n = (int)(((item_first + cur.units) * ctas - 1) / total - c0) + 1;
      const int groups = (n + kGroup - 1) / kGroup, mine_at = (int)(blockIdx.x - c0) / kGroup;
      const int members = n - mine_at * kGroup < kGroup ? n - mine_at * kGroup : kGroup;
      // A group of one needs no counter, so a group's first CTA names it alone.
      uint32_t* counter = a.counters + c0 + mine_at * kGroup;
      if (members == 1 || arrive_last(counter, members, &s_last)) {
        if (groups > 1) {
          if (members > 1)
            join_partials<8 * R, D>(a, c0, mine_at * kGroup, 1, members, true, 0, 0);
          __syncthreads();
          if (arrive_last(a.counters + kMaxCtas + c0, groups, &s_last))
            join_partials<8 * R, D>(a, c0, 0, kGroup, groups, false,
                                    cur.b * p.q_heads + q_head, heads);
        } else {
          join_partials<8 * R, D>(a, c0, 0, 1, n, false, cur.b * p.q_heads + q_head, heads);
        }
      }
    }
    at += seg;
    if (at < last) {
      cur.unit = cur.units - 1;  // the segment ended with its item
      advance<F::kUnit>(a, cur);
    }
  }
  cp_async_wait<0>();
}

template <class C, bool F32ACT, int D, int R>
int launch(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  using F = Cfg<C, F32ACT, D, R>;
  auto kernel = paged_attention_kernel<C, F32ACT, D, R>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem) !=
      cudaSuccess)
    return CT_ERR_CUDA;
  Launch b = a;
  b.whole_tiles = a.p.kv.page_size % F::kKeys == 0;
  // no more CTAs than units the table can hold
  const int64_t keys = a.p.kv.max_pages * a.p.kv.page_size;
  const int64_t units = a.p.batch * a.items * (keys > F::kUnit ? (keys + F::kUnit - 1) / F::kUnit : 1);
  int64_t ctas = (int64_t)dev.sm_count * F::kCtas;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (ctas > units) ctas = units;
  kernel<<<(unsigned)ctas, kThreads, F::kSmem, st>>>(b);
  return check_launch();
}

constexpr size_t kCounterBytes = 2 * kMaxCtas * sizeof(uint32_t);
int head_blocks(int64_t q_heads, int64_t kv_heads) { return q_heads / kv_heads > 8 ? 2 : 1; }

template <class C, bool F32ACT>
int launch_dims(const Launch& a, int r, const DeviceInfo& dev, cudaStream_t st) {
  if (a.p.head_dim == 32)
    return r == 1 ? launch<C, F32ACT, 32, 1>(a, dev, st) : launch<C, F32ACT, 32, 2>(a, dev, st);
  if (a.p.head_dim == 64)
    return r == 1 ? launch<C, F32ACT, 64, 1>(a, dev, st) : launch<C, F32ACT, 64, 2>(a, dev, st);
  return r == 1 ? launch<C, F32ACT, 128, 1>(a, dev, st) : launch<C, F32ACT, 128, 2>(a, dev, st);
}

}  // namespace

size_t paged_attention_workspace(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  return kCounterBytes + 2 * kMaxCtas * sizeof(float) *
                             partial_floats(8 * head_blocks(q_heads, kv_heads), (int)head_dim);
}

int launch_paged_attention(const PagedAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  Launch a{};
  a.p = p;
  const int r = head_blocks(p.q_heads, p.kv_heads);
  a.group = (int)(p.q_heads / p.kv_heads);
  a.blocks = (a.group + 8 * r - 1) / (8 * r);
  const int64_t items = p.kv_heads * a.blocks;
  if (items >= (1ll << 31)) return CT_ERR_INVALID_ARGUMENT;
  a.items = (int)items;
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (p.kv.page_size == 1 << s) a.page_shift = s;
  a.counters = static_cast<uint32_t*>(p.ws);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(p.ws) + kCounterBytes);
  return with_dtype(p.kv.dtype, [&](auto c) {
    using C = decltype(c);
    if (p.act_dtype == CT_DTYPE_F32) return launch_dims<C, true>(a, r, dev, st);
    if constexpr (sizeof(C) == 2) return launch_dims<C, false>(a, r, dev, st);
    return (int)CT_ERR_INVALID_ARGUMENT;
  });
}

}  // namespace ct
