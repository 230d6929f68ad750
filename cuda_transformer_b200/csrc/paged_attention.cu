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
constexpr int kCtasPerSm = 2;
constexpr int kMaxCtas = 512;       // counters and partial slots in the workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The running maximum is raised only when a score passes it by this much (in
// powers of two): probabilities stay below 2^8, which FP32 sums hold as well
// as values below 1, and most tiles skip the rescaling of O.
constexpr float kMaxSlack = 8.0f;

template <class C, int D, int MT>
struct Cfg {
  static constexpr int kVec = 16 / (int)sizeof(C);         // elements of a 16-byte chunk
  static constexpr int kKeys = sizeof(C) == 2 ? 16 : 8;     // keys of a warp's tile
  static constexpr int kNt = kKeys / 8;
  static constexpr int kUnit = kWarps * kKeys;              // keys of a work unit
  static constexpr int kRowBytes = D * (int)sizeof(C);
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kStageBytes = 2 * kKeys * kRowBytes; // K tile, V tile
  static constexpr int kStages = 24576 / kStageBytes > 8 ? 8 : 24576 / kStageBytes;
  static constexpr int kKIter = D / (4 * kVec);             // K chunks a lane reads per key
  static constexpr int kVVec = kVec < D / 8 ? kVec : D / 8; // V elements a lane reads at once
  static constexpr int kVIter = D / (8 * kVVec);
  static constexpr int kOTiles = D / 8;
  static constexpr bool kQInRegs = MT == 1;                 // else in shared memory
  static constexpr int kJoinBytes = kWarps * 8 * D * 4;     // also holds q when MT == 2
  static constexpr int kQBytes = kQInRegs ? 0 : MT * (D / 8) * 32 * 16;
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
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = high + low, both TF32 (11 significant bits): the high part is cut off,
// the rest (13 bits) rounded, so the error is below 2^-22 of x.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
}

// Element e of a 16- or 8-byte chunk as FP32 bits.
template <class C>
__device__ __forceinline__ uint32_t chunk_elem(const uint32_t* w, int e);
template <>
__device__ __forceinline__ uint32_t chunk_elem<float>(const uint32_t* w, int e) { return w[e]; }
template <>
__device__ __forceinline__ uint32_t chunk_elem<__nv_bfloat16>(const uint32_t* w, int e) {
  return e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16;
}
template <>
__device__ __forceinline__ uint32_t chunk_elem<__half>(const uint32_t* w, int e) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w[e >> 1]);
  return __float_as_uint(e & 1 ? __high2float(h) : __low2float(h));
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

__device__ __forceinline__ float load_act(const void* p, int64_t i, int dtype) {
  if (dtype == CT_DTYPE_F32) return ((const float*)p)[i];
  if (dtype == CT_DTYPE_BF16) return to_f32(((const __nv_bfloat16*)p)[i]);
  return to_f32(((const __half*)p)[i]);
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

// Floats of a partial: O [8 MT][D], then max and sum [8 MT] each.
constexpr int64_t partial_floats(int heads, int D) { return (int64_t)heads * (D + 2); }

struct Launch {
  PagedAttention p;
  int group, blocks;  // query heads of a key/value head; its blocks of 8 MT heads
  int items;          // (key/value head, block) pairs of a sequence
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

__device__ __forceinline__ float exp2_diff(float m, float top) {
  return m == -INFINITY ? 0.0f : exp2f(m - top);
}

template <class C, int D, int MT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    paged_attention_kernel(const __grid_constant__ Launch a) {
  using F = Cfg<C, D, MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_scan[kWarps + 2];
  __shared__ Cursor s_start;
  __shared__ float s_m[kWarps][8 * MT], s_l[kWarps][8 * MT];
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
  uint8_t* ring = smem + w * (F::kStages * F::kStageBytes);
  const bool second = (lane / F::kKeys) & 1;  // this lane addresses V rows, else K rows
  const int my_row = lane % F::kKeys;
  int64_t to_issue = last - first;
  int next_page = -1, next_slot = 0, next_head = 0;
  bool next_there = false;
  auto look_up = [&]() {  // page and slot of the lane's row of the next tile
    next_there = false;
    if (to_issue <= 0) return;
    const int key = ahead.unit * F::kUnit + w * F::kKeys + my_row;
    next_there = key < ahead.len;
    if (next_there) {
      const int index = key / p.kv.page_size;
      next_slot = key - index * p.kv.page_size;
      next_page = p.kv.table[ahead.b * p.kv.table_s + index];
      next_head = ahead.item / a.blocks;
    }
    --to_issue;
    if (to_issue > 0) advance<F::kUnit>(a, ahead);
  };
  auto issue = [&](int stage) {
    int64_t off = -1;  // past the length: zeros
    if (next_there) {
      const int64_t* s = second ? p.kv.vs : p.kv.ks;
      off = next_page < 0 || next_page >= p.kv.pages
                ? -2  // no such page: NaN keys
                : (next_page * s[0] + next_head * s[1] + next_slot * s[2]) * (int64_t)sizeof(C);
    }
    const uint32_t base = smem_addr(ring + stage * F::kStageBytes);
    constexpr int kCopies = F::kKeys * F::kRowChunks / 32;
    if (__any_sync(0xffffffffu, next_there)) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int flat = i * 32 + lane, r = flat / F::kRowChunks, c = flat % F::kRowChunks;
          const int64_t o = __shfl_sync(0xffffffffu, off, kv * F::kKeys + r);
          const uint32_t dst = base + kv * (F::kKeys * F::kRowBytes) + chunk_pos<F::kRowBytes>(r, c);
          const uint8_t* src = (const uint8_t*)(kv ? p.kv.v : p.kv.k);
          if (o == -2)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0x7fc07fc0u)
                         : "memory");  // NaN in each of the three types
          else
            cp_async16(dst, o < 0 ? src : src + o + c * 16, o < 0 ? 0 : 16);
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
  uint32_t q_regs[F::kQInRegs ? D / 8 : 1][4];
  const float q_scale = p.scale * kLog2e;
  int stage = 0;

  for (int64_t at = first; at < last;) {
    // ---- one segment: units cur.unit .. end of the item, or of the share
    const int kv_head = cur.item / a.blocks, head0 = (cur.item % a.blocks) * 8 * MT;
    const int heads = a.group - head0 < 8 * MT ? a.group - head0 : 8 * MT;
    const int64_t q_head = (int64_t)kv_head * a.group + head0;
    const int64_t item_first = at - cur.unit;
    const int seg = (int)(last - at < cur.units - cur.unit ? last - at : cur.units - cur.unit);

    // q in the order of the products' A operand: rows g (high) and g + 8
    // (low), the two dims that lane t of step s multiplies
    auto q_split = [&](int mt, int s, int gg, int tt, uint32_t (&r)[4]) {
      const int h = mt * 8 + gg;
      const int d = (tt + 4 * (s / (F::kVec / 2))) * F::kVec + 2 * (s % (F::kVec / 2));
      const int64_t o = cur.b * p.qs[0] + (q_head + h) * p.qs[1] + d * p.qs[2];
      const float x = h < heads ? load_act(p.q, o, p.act_dtype) * q_scale : 0.0f;
      const float y = h < heads ? load_act(p.q, o + p.qs[2], p.act_dtype) * q_scale : 0.0f;
      split_tf32(x, r[0], r[1]);
      split_tf32(y, r[2], r[3]);
    };
    if constexpr (F::kQInRegs) {
#pragma unroll
      for (int s = 0; s < D / 8; ++s) q_split(0, s, g, t, q_regs[s]);
    } else {
      for (int i = tid; i < MT * (D / 8) * 32; i += kThreads) {
        uint32_t r[4];
        q_split(i / (D / 8 * 32), i / 32 % (D / 8), (i % 32) / 4, i % 4, r);
        *reinterpret_cast<uint4*>(q_smem + i * 4) = make_uint4(r[0], r[1], r[2], r[3]);
      }
      __syncthreads();
    }

    float o_acc[MT][F::kOTiles][4], m_run[MT], l_run[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m_run[mt] = -INFINITY;
      l_run[mt] = 0.0f;
#pragma unroll
      for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_acc[mt][j][e] = 0.0f;
    }

    for (int u = 0; u < seg; ++u) {
      cp_async_wait<F::kStages - 2>();
      __syncwarp();
      issue(stage == 0 ? F::kStages - 1 : stage - 1);
      const int key0 = (cur.unit + u) * F::kUnit + w * F::kKeys;
      const uint8_t* tile = ring + stage * F::kStageBytes;
      stage = stage + 1 == F::kStages ? 0 : stage + 1;
      if (key0 >= cur.len) continue;

      // ---- S = q k^T, in two chains for each 8 x 8 tile
      float s_acc[MT][F::kNt][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s_acc[mt][n][0][e] = s_acc[mt][n][1][e] = 0.0f;
#pragma unroll
      for (int i = 0; i < F::kKIter; ++i) {
        uint32_t kw[F::kNt][4];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
          *reinterpret_cast<uint4*>(kw[n]) = *reinterpret_cast<const uint4*>(
              tile + chunk_pos<F::kRowBytes>(n * 8 + g, t + 4 * i));
#pragma unroll
        for (int e = 0; e < F::kVec / 2; ++e) {
          const int s = i * (F::kVec / 2) + e;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t qa[4];
            if constexpr (F::kQInRegs) {
#pragma unroll
              for (int x = 0; x < 4; ++x) qa[x] = q_regs[s][x];
            } else {
              *reinterpret_cast<uint4*>(qa) =
                  *reinterpret_cast<const uint4*>(q_smem + ((mt * (D / 8) + s) * 32 + lane) * 4);
            }
#pragma unroll
            for (int n = 0; n < F::kNt; ++n) {
              const uint32_t x = chunk_elem<C>(kw[n], 2 * e), y = chunk_elem<C>(kw[n], 2 * e + 1);
              if constexpr (sizeof(C) == 4) {
                uint32_t xh, xl, yh, yl;
                split_tf32(__uint_as_float(x), xh, xl);
                split_tf32(__uint_as_float(y), yh, yl);
                mma_tf32(s_acc[mt][n][0], qa, xh, yh);
                mma_tf32(s_acc[mt][n][1], qa, xl, yl);
              } else {
                mma_tf32(s_acc[mt][n][e & 1], qa, x, y);
              }
            }
          }
        }
      }

      // ---- probabilities; keys n * 8 + 2 t and + 1 of head mt * 8 + g
      uint32_t pa[MT][F::kNt][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float v[F::kNt][2], top = -INFINITY;
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float(&x)[2][4] = s_acc[mt][n];
            v[n][e] = (x[0][e] + x[1][e]) + (x[0][e + 2] + x[1][e + 2]);
            if (key0 + n * 8 + 2 * t + e >= cur.len) v[n][e] = -INFINITY;
            top = fmaxf(top, v[n][e]);
          }
        if (__any_sync(0xffffffffu, top > m_run[mt] + kMaxSlack)) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top, m_run[mt]);
          const float f = exp2_diff(m_run[mt], top);
          m_run[mt] = top;
          l_run[mt] *= f;
#pragma unroll
          for (int j = 0; j < F::kOTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_acc[mt][j][e] *= f;
        }
        const float m = m_run[mt] == -INFINITY ? 0.0f : m_run[mt];
#pragma unroll
        for (int n = 0; n < F::kNt; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float pr = exp2f(v[n][e] - m);
            l_run[mt] += pr;
            split_tf32(pr, pa[mt][n][2 * e], pa[mt][n][2 * e + 1]);
          }
      }

      // ---- O += P V
      const uint8_t* vt = tile + F::kKeys * F::kRowBytes;
#pragma unroll
      for (int n = 0; n < F::kNt; ++n) {
#pragma unroll
        for (int i = 0; i < F::kVIter; ++i) {
          uint32_t v0[4], v1[4];
          const int r = n * 8 + 2 * t;
          if constexpr (F::kVVec == F::kVec) {
            *reinterpret_cast<uint4*>(v0) = *reinterpret_cast<const uint4*>(
                vt + chunk_pos<F::kRowBytes>(r, g + 8 * i));
            *reinterpret_cast<uint4*>(v1) = *reinterpret_cast<const uint4*>(
                vt + chunk_pos<F::kRowBytes>(r + 1, g + 8 * i));
          } else {  // 64-byte rows: half a chunk to a lane
            *reinterpret_cast<uint2*>(v0) = *reinterpret_cast<const uint2*>(
                vt + chunk_pos<F::kRowBytes>(r, g >> 1) + (g & 1) * 8);
            *reinterpret_cast<uint2*>(v1) = *reinterpret_cast<const uint2*>(
                vt + chunk_pos<F::kRowBytes>(r + 1, g >> 1) + (g & 1) * 8);
          }
#pragma unroll
          for (int e = 0; e < F::kVVec; ++e) {
            const uint32_t x = chunk_elem<C>(v0, e), y = chunk_elem<C>(v1, e);
            uint32_t xh = x, yh = y, xl = 0, yl = 0;
            if constexpr (sizeof(C) == 4) {
              split_tf32(__uint_as_float(x), xh, xl);
              split_tf32(__uint_as_float(y), yh, yl);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_tf32(o_acc[mt][i * F::kVVec + e], pa[mt][n], xh, yh);
              if constexpr (sizeof(C) == 4) mma_tf32(o_acc[mt][i * F::kVVec + e], pa[mt][n], xl, yl);
            }
          }
        }
      }
    }

    // ---- the segment's end: join the warps, then write O or a partial
    const bool whole = cur.unit == 0 && seg == cur.units;
    const bool tail = cur.unit != 0;
    float* slot = a.partials + (2 * (int64_t)blockIdx.x + (tail ? 0 : 1)) *
                                   partial_floats(8 * MT, D);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float l = l_run[mt];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t == 0) {
        s_m[w][mt * 8 + g] = m_run[mt];
        s_l[w][mt * 8 + g] = l;
      }
    }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s_m[i][mt * 8 + g]);
      const float f = exp2_diff(m_run[mt], top);
      // lane (g, t) holds dims of chunks 2 t and 2 t + 1 (+ 8 i) of head g
#pragma unroll
      for (int i = 0; i < F::kVIter; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < F::kVVec; e += 4) {
            float4 x;
            float* xs = reinterpret_cast<float*>(&x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float(&o)[4] = o_acc[mt][i * F::kVVec + e + k];
              xs[k] = (o[c] + o[c + 2]) * f;
            }
            *reinterpret_cast<float4*>(join + (w * 8 + g) * D + (2 * t + c + 8 * i) * F::kVVec + e) = x;
          }
      __syncthreads();
      for (int i = tid; i < 8 * D / 4; i += kThreads) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float hm = -INFINITY, hl = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(join + (k * 8 + h) * D + d);
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
          hm = fmaxf(hm, s_m[k][mt * 8 + h]);
        }
#pragma unroll
        for (int k = 0; k < kWarps; ++k)
          hl += s_l[k][mt * 8 + h] * exp2_diff(s_m[k][mt * 8 + h], hm);
        if (cur.bad) hl = NAN;
        if (!whole) {
          *reinterpret_cast<float4*>(slot + (mt * 8 + h) * D + d) = x;
          if (d == 0) {
            slot[8 * MT * D + mt * 8 + h] = hm;
            slot[8 * MT * D + 8 * MT + mt * 8 + h] = hl;
          }
        } else if (mt * 8 + h < heads) {
          const int64_t row = cur.b * p.q_heads + q_head + mt * 8 + h;
          const float r = hl == 0.0f ? 0.0f : 1.0f / hl;
          store_act4(p.out, row * D + d, p.act_dtype,
                     make_float4(x.x * r, x.y * r, x.z * r, x.w * r));
          if (d == 0 && p.lse) p.lse[row] = (hm + log2f(hl)) * kLn2;
        }
      }
      __syncthreads();
    }

    if (!whole) {
      // contributors of this item: CTAs c0 (its first units, odd slot) .. c1
      const int64_t c0 = ((item_first + 1) * ctas - 1) / total;
      const int64_t c1 = ((item_first + cur.units) * ctas - 1) / total;
      const int n = (int)(c1 - c0 + 1);
      if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(a.counters + c0, 1u) == (uint32_t)(n - 1);
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        if (tid == 0) a.counters[c0] = 0u;
        const int64_t step = partial_floats(8 * MT, D);
        for (int i = tid; i < 8 * MT * D / 4; i += kThreads) {
          const int h = i / (D / 4), d = i % (D / 4) * 4;
          float hm = -INFINITY, hl = 0.0f;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          const float* base = a.partials + 2 * c0 * step;
#pragma unroll 4
          for (int k = 0; k < n; ++k)
            hm = fmaxf(hm, __ldcg(base + (k == 0 ? 1 : 2 * k) * step + 8 * MT * D + h));
#pragma unroll 4
          for (int k = 0; k < n; ++k) {
            const float* s = base + (k == 0 ? 1 : 2 * k) * step;
            const float4 y = __ldcg(reinterpret_cast<const float4*>(s + h * D + d));
            const float km = __ldcg(s + 8 * MT * D + h), kl = __ldcg(s + 8 * MT * D + 8 * MT + h);
            const float f = exp2_diff(km, hm);
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
            hl = fmaf(kl, f, hl);
          }
          if (h < heads) {
            const int64_t row = cur.b * p.q_heads + q_head + h;
            const float r = hl == 0.0f ? 0.0f : 1.0f / hl;
            store_act4(p.out, row * D + d, p.act_dtype,
                       make_float4(x.x * r, x.y * r, x.z * r, x.w * r));
            if (d == 0 && p.lse) p.lse[row] = (hm + log2f(hl)) * kLn2;
          }
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

template <class C, int D, int MT>
int launch(const Launch& a, const DeviceInfo& dev, cudaStream_t st) {
  using F = Cfg<C, D, MT>;
  auto kernel = paged_attention_kernel<C, D, MT>;
  // once per device and process would do; the call costs well under a microsecond
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem) !=
      cudaSuccess)
    return CT_ERR_CUDA;
  // no more CTAs than units the table can hold
  const int64_t keys = a.p.kv.max_pages * a.p.kv.page_size;
  const int64_t units = a.p.batch * a.items * (keys > F::kUnit ? (keys + F::kUnit - 1) / F::kUnit : 1);
  int64_t ctas = (int64_t)dev.sm_count * kCtasPerSm;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (ctas > units) ctas = units;
  kernel<<<(unsigned)ctas, kThreads, F::kSmem, st>>>(a);
  return check_launch();
}

constexpr size_t kCounterBytes = kMaxCtas * sizeof(uint32_t);
int head_tiles(int64_t q_heads, int64_t kv_heads) { return q_heads / kv_heads > 8 ? 2 : 1; }

}  // namespace

size_t paged_attention_workspace(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  return kCounterBytes + 2 * kMaxCtas * sizeof(float) *
                             partial_floats(8 * head_tiles(q_heads, kv_heads), (int)head_dim);
}

int launch_paged_attention(const PagedAttention& p, const DeviceInfo& dev, cudaStream_t st) {
  Launch a;
  a.p = p;
  const int mt = head_tiles(p.q_heads, p.kv_heads);
  a.group = (int)(p.q_heads / p.kv_heads);
  a.blocks = (a.group + 8 * mt - 1) / (8 * mt);
  const int64_t items = p.kv_heads * a.blocks;
  if (items >= (1ll << 31)) return CT_ERR_INVALID_ARGUMENT;
  a.items = (int)items;
  a.counters = static_cast<uint32_t*>(p.ws);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(p.ws) + kCounterBytes);
  return with_dtype(p.kv.dtype, [&](auto c) {
    using C = decltype(c);
    if (p.head_dim == 32)
      return mt == 1 ? launch<C, 32, 1>(a, dev, st) : launch<C, 32, 2>(a, dev, st);
    if (p.head_dim == 64)
      return mt == 1 ? launch<C, 64, 1>(a, dev, st) : launch<C, 64, 2>(a, dev, st);
    return mt == 1 ? launch<C, 128, 1>(a, dev, st) : launch<C, 128, 2>(a, dev, st);
  });
}

}  // namespace ct
