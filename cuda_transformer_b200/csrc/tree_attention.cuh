// tree_attention.cuh -- what the two kernels of tree_attention share: how the
// work is divided, which tokens a row sees, the joining of split items.
//
// Work is cut into tiles of keys of one item (a sequence and a key/value head),
// and every CTA takes an equal share of the tiles, counted on the device from
// the lengths (the host knows none).  Rows that do not fit one CTA are blocks,
// whose CTAs take the same share side by side and meet its keys in L2.  A share
// that starts or ends inside an item leaves a partial (base of the exponents, sum,
// O) in the workspace, and a second kernel joins the partials in their order: the
// results do not depend on timing and nothing has to be cleared.  The join takes 7 to
// 11 us of the calls measured (a CTA for 8 rows each, as first built: 20).
#pragma once

#include <cfloat>

#include "decode_common.cuh"
#include "tc_ptx.cuh"

namespace ct {
namespace tree {
namespace {

constexpr int kMaxCtas = 448;  // partial slots (two each) and records in the workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The base of the exponents is raised only when a score passes it by this much
// (in powers of two): most tiles skip the rescaling of O.  Weights then reach 2^6
// instead of 1, far inside every type's range (f16's too, which adds 2^8).
constexpr float kMaxSlack = 6.0f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Launch {
  TreeAttention p;
  int group, blocks;    // query heads of a key/value head; row blocks of an item
  int block0;           // of this launch: the first of them
  int group_shift;      // log2 of group, -1 when it is no power of two
  int shares;
  bool whole;           // an item a CTA: none is split
  bool q_vectors;       // q's rows are 16-byte vectors
  int page_shift;       // log2 of page_size, -1 when it is no power of two
  float c2;             // |scale| log2 e
  bool negative;        // scale: q's sign turns
  int box;              // slots of a TMA box; 0: copies of single chunks
  uint32_t* status;
  int4* records;        // of each CTA: the split item that begins in it
  float* partials;
};

// The drafted token of an item's row.
__device__ __forceinline__ int token_of(const Launch& a, int row) {
  return a.group_shift >= 0 ? row >> a.group_shift : row / a.group;
}

struct Sequence {
  int context, drafts, tiles;
  bool there, bad;
};
template <class K>
__device__ __forceinline__ Sequence sequence(const TreeAttention& p, int64_t b) {
  Sequence s;
  s.context = p.context_lens[b];
  const int n = p.draft_lens ? p.draft_lens[b] : (int)p.drafts;
  s.drafts = n < 0 ? 0 : n > p.drafts ? (int)p.drafts : n;
  s.there = s.context >= 0 && s.drafts > 0;
  const int64_t len = (int64_t)s.context + s.drafts;
  s.bad = s.there && len > p.kv.max_pages * p.kv.page_size;
  s.tiles = s.there && !s.bad ? (int)((len + K::kKeys - 1) / K::kKeys) : 0;
  return s;
}

template <class K>
__device__ __forceinline__ int64_t units_of(const Launch& a, int tiles) {
  return tiles > 0 ? (int64_t)(tiles + K::kItemCost) * a.p.kv_heads : 0;
}

// A place in the list of tiles.
struct Cursor {
  int64_t b;
  int head, tile, stop, tiles;  // stop: end of this share's part of the item
  int context, drafts;
  int64_t left;                 // units of the share from this item's part on
};

// The item at (c.b, c.head), `within` units into it, or the next one there is that
// has rows behind row0.  All lanes of a warp.
template <class K>
__device__ __forceinline__ bool enter(const Launch& a, Cursor& c, int64_t within, int row0) {
  while (c.left > 0 && c.b < a.p.batch) {
    const Sequence s = sequence<K>(a.p, c.b);
    if (s.tiles == 0 || c.head == (int)a.p.kv_heads) {
      ++c.b;
      c.head = 0;
      within = 0;
      // the next that is there, 32 looked at at once: batches may be padded (2 sequences
      // in 256 places 25 us, one place after the other 48)
      if (s.tiles == 0)
        for (; c.b < a.p.batch; c.b += 32) {
          const int64_t b = c.b + threadIdx.x % 32;
          const uint32_t there =
              __ballot_sync(0xffffffffu, b < a.p.batch && sequence<K>(a.p, b).tiles > 0);
          if (there) {
            c.b += __ffs(there) - 1;
            break;
          }
        }
      continue;
    }
    const int64_t units = s.tiles + K::kItemCost;
    const int64_t end = within + c.left < units ? within + c.left : units;
    c.left -= end - within;
    c.tile = within > K::kItemCost ? (int)(within - K::kItemCost) : 0;
    c.stop = end > K::kItemCost ? (int)(end - K::kItemCost) : 0;
    c.tiles = s.tiles;
    c.context = s.context;
    c.drafts = s.drafts;
    within = 0;
    if (c.tile < c.stop && row0 < c.drafts * a.group) return true;
    ++c.head;
  }
  return false;
}

struct Finder {
  int64_t scan[32];
  int64_t b, x;
};

// Where share `share` of the units begins (all threads of the CTA; the first barrier
// of theirs): `within` units into an item, which `enter` takes.
template <class K>
__device__ __forceinline__ Cursor first_place(const Launch& a, int share, Finder& f,
                                              int64_t& share_units, int64_t& within) {
  const TreeAttention& p = a.p;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid % 32;
  Cursor c;
  c.head = 0;
  share_units = within = 0;
  if (a.whole) {
    c.b = share / (int)p.kv_heads;
    c.head = share % (int)p.kv_heads;
    const int tiles = sequence<K>(p, c.b).tiles;
    c.left = tiles > 0 ? tiles + K::kItemCost : 0;
    return c;
  }
  const int64_t each = (p.batch + threads - 1) / threads;
  const int64_t b0 = tid * each, b1 = b0 + each < p.batch ? b0 + each : p.batch;
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += units_of<K>(a, sequence<K>(p, b).tiles);
  int64_t run = mine;
  for (int w = 1; w < 32; w *= 2) {
    const int64_t y = __shfl_up_sync(0xffffffffu, run, w);
    if (lane >= w) run += y;
  }
  if (lane == 31) f.scan[tid / 32] = run;
  if (tid == 0) f.b = p.batch;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w < tid / 32) before += f.scan[w];
    total += f.scan[w];
  }
  before += run - mine;
  share_units = (total + a.shares - 1) / a.shares;
  if (share_units < K::kMinShare) share_units = K::kMinShare;
  const int64_t begin = share * share_units;
  if (mine > 0 && begin >= before && begin < before + mine) {
    int64_t b = b0;
    for (; b < b1; ++b) {
      const int64_t u = units_of<K>(a, sequence<K>(p, b).tiles);
      if (begin < before + u) break;
      before += u;
    }
    f.b = b;
    f.x = begin - before;
  }
  __syncthreads();
  c.b = f.b;
  c.left = c.b >= p.batch ? 0 : total - begin < share_units ? total - begin : share_units;
  if (c.left > 0) {
    const int64_t units = sequence<K>(p, c.b).tiles + K::kItemCost;
    c.head = (int)(f.x / units);
    within = f.x - c.head * units;
  }
  return c;
}

// The first two words of a row's mask; both rows' and words' ends are looked at where
// they are used.
constexpr int kKeptWords = 2;
__device__ __forceinline__ uint32_t mask_word(const TreeAttention& p, int64_t b, int i, int word) {
  return p.mask && i < p.drafts && word * 32 < p.drafts ? p.mask[b * p.ms[0] + i * p.ms[1] + word] : 0u;
}

// Which of the 32 drafted tokens from number d on (d < 0: some before the draft) the
// drafted token i of sequence b sees, as bits; kept: its first words.
__device__ __forceinline__ uint32_t seen_from(const TreeAttention& p, uint2 kept, int64_t b, int i, int d,
                                           int drafts) {
  if (d <= -32) return ~0u;
  if (i >= drafts || d >= drafts) return d < 0 ? (1u << -d) - 1u : 0u;
  uint32_t w;
  if (p.mask) {
    const int at = d < 0 ? 0 : d >> 5, last = (drafts - 1) >> 5;
    uint32_t low, high;
    if (last < kKeptWords) {
      low = at == 0 ? kept.x : kept.y;
      high = at < last ? kept.y : 0u;
    } else {
      const uint32_t* words = p.mask + b * p.ms[0] + i * p.ms[1];
      low = words[at];
      high = at < last ? words[at + 1] : 0u;
    }
    w = d < 0 ? low << -d | ((1u << -d) - 1u) : __funnelshift_r(low, high, d & 31);
  } else {
    w = i < d ? 0u : i - d >= 31 ? ~0u : (2u << (i - d)) - 1u;
  }
  return drafts - d >= 32 ? w : w & ((1u << (drafts - d)) - 1u);
}

// Eight 16-bit (four 32-bit) elements that lie `stride` apart.
template <class A>
__device__ __noinline__ uint4 gather8(const A* src, int64_t stride) {
  alignas(16) A x[16 / sizeof(A)];
  for (int e = 0; e < 16 / (int)sizeof(A); ++e) x[e] = src[e * stride];
  return *reinterpret_cast<const uint4*>(x);
}

template <class A>
__device__ __forceinline__ void store2(void* out, int64_t i, float x, float y) {
  if constexpr (sizeof(A) == 4) {
    *reinterpret_cast<float2*>((float*)out + i) = make_float2(x, y);
  } else if constexpr (std::is_same<A, __nv_bfloat16>::value) {
    *reinterpret_cast<__nv_bfloat162*>((A*)out + i) = __floats2bfloat162_rn(x, y);
  } else {
    *reinterpret_cast<__half2*>((A*)out + i) = __floats2half2_rn(x, y);
  }
}

// Bytes of workspace of a partial: O [rows][D], then the exponents' base and the
// sum of each row.
constexpr int64_t partial_floats(int rows, int D) { return (int64_t)rows * (D + 4); }

// Rows that are not there: zero; all of a sequence whose length is out of range: NaN.
template <class K>
__device__ __forceinline__ void write_rows_not_there(const TreeAttention& p) {
  using A = typename K::A;
  constexpr int D = K::D;
  for (int64_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const Sequence s = sequence<K>(p, b);
    const int first = s.there && !s.bad ? s.drafts : 0;
    const int64_t row0 = b * p.drafts * p.q_heads;
    for (int64_t e = (int64_t)first * p.q_heads * D + 2 * threadIdx.x; e < p.drafts * p.q_heads * D;
         e += 2 * blockDim.x) {
      const int64_t row = e / D;
      const bool nan = s.bad && row < (int64_t)s.drafts * p.q_heads;
      store2<A>(p.out, row0 * D + e, nan ? NAN : 0.0f, nan ? NAN : 0.0f);
      if (e % D == 0 && p.lse) p.lse[row0 + row] = nan ? NAN : -INFINITY;
    }
  }
}

// Joins the partials of split items.  Every CTA collects the records (most CTAs of the
// first kernel leave one where sequences are short, few where one is long), so that
// the rows there are can be dealt out evenly: a row a warp while that keeps all rows
// on the way at once, 4 or 16 warps a row when there are few (one sequence of 60,000
// tokens, 16 heads on one of 64, 8 drafts: 27 us, a warp a row 51), four rows a warp when
// there are many.
constexpr int kJoinThreads = 512;

// Rows at, at + step, ... of the split items, LANES lanes a row; with W > 1, W warps of
// the CTA that take turns at its parts and meet in shared memory.
template <class A, int D, int LANES, int W = 1>
__device__ __forceinline__ void join_rows(const Launch& a, const int4* record, const int* first_cta,
                                          int all, int rows, int at, int step,
                                          float (*meet)[D + 1] = nullptr) {
  constexpr int N = D / LANES;  // dims of a lane
  const int lane = threadIdx.x % LANES, warp = threadIdx.x / 32;
  const int64_t each = partial_floats(rows, D);
  static_assert(W == 1 || LANES == 32, "");
  // (all rows of a warp, or of the CTA, go through the same number of steps)
  for (; at - (W > 1 ? warp / W : (int)(threadIdx.x % 32) / LANES) < all; at += step) {
    const bool in = at < all;
    const int4 rec = record[in ? at / rows : 0];
    const int cta = first_cta[in ? at / rows : 0], r = at % rows;
    const int block = a.block0 + cta % a.blocks;
    const int i = token_of(a, block * rows + r);
    const int n = in && i < rec.w ? rec.x : 0;
    // the first part ends its CTA's share, the others begin theirs
    auto part = [&](int k) {
      return a.partials + ((int64_t)(cta + k * a.blocks) * 2 + (k == 0)) * each;
    };
    float top = -INFINITY, sum = 0.0f, o[N] = {};
    for (int k = lane; k < n; k += LANES) top = fmaxf(top, part(k)[rows * D + 2 * r]);
    for (int w = LANES / 2; w; w /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    constexpr int kUnroll = N >= 16 ? 2 : N >= 8 ? 4 : 8;
#pragma unroll kUnroll
    for (int k = W > 1 ? warp % W : 0; k < n; k += W) {
      const float2 ml = *reinterpret_cast<const float2*>(part(k) + rows * D + 2 * r);
      const float* src = part(k) + r * D;
      float x[N];
      // (vectors of the lanes side by side)
      constexpr int V = N < 4 ? N : 4;
#pragma unroll
      for (int v = 0; v < N; v += V) {
        const float* from = src + v * LANES + lane * V;
        if constexpr (V == 4) *reinterpret_cast<float4*>(x + v) = *reinterpret_cast<const float4*>(from);
        else if constexpr (V == 2) *reinterpret_cast<float2*>(x + v) = *reinterpret_cast<const float2*>(from);
        else x[v] = *from;
      }
      const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - top);
      sum += ml.x == -INFINITY ? ml.y : ml.y * f;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] += ml.x == -INFINITY ? 0.0f : x[e] * f;
    }
    if constexpr (W > 1) {
      __syncthreads();
      if (warp % W) {
#pragma unroll
        for (int e = 0; e < N; ++e) meet[warp][e * 32 + lane] = o[e];
        if (lane == 0) meet[warp][D] = sum;
      }
      __syncthreads();
      if (warp % W) continue;
#pragma unroll
      for (int w = 1; w < W; ++w) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] += meet[warp + w][e * 32 + lane];
        sum += meet[warp + w][D];
      }
    }
    if (n > 0) {
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int64_t row = ((int64_t)rec.y * a.p.drafts + i) * a.p.q_heads + rec.z * a.group +
                          (block * rows + r) - i * a.group;
      constexpr int V = N < 4 ? N : 4;
#pragma unroll
      for (int v = 0; v < N; v += V) {
        const int64_t to = row * D + v * LANES + lane * V;
        if constexpr (V == 1) {
          ((A*)a.p.out)[to] = from_f32<A>(o[v] * f);
        } else {
#pragma unroll
          for (int e = 0; e < V; e += 2) store2<A>(a.p.out, to + e, o[v + e] * f, o[v + e + 1] * f);
        }
      }
      if (lane == 0 && a.p.lse) a.p.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
    __syncwarp();
  }
}

// FEW: there cannot be more than 4 rows a CTA.  (One kernel for both took 2 us longer
// where rows are many.)
template <class A, int D, bool FEW>
__global__ void __launch_bounds__(kJoinThreads, 2)
    tree_join_kernel(const __grid_constant__ Launch a, const int rows, const int ctas) {
  __shared__ int4 record[kMaxCtas];
  __shared__ int first_cta[kMaxCtas], count[kJoinThreads / 32];
  static_assert(kMaxCtas <= kJoinThreads, "a thread a record");
  const int c = threadIdx.x, warp = c / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (*reinterpret_cast<const volatile uint32_t*>(a.status) != 0u) return;
  // (in the same order in every CTA)
  const int4 own = c < ctas ? a.records[c] : make_int4(0, 0, 0, 0);
  const uint32_t vote = __ballot_sync(0xffffffffu, own.x > 0);
  if (c % 32 == 0) count[warp] = __popc(vote);
  __syncthreads();
  int found = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    if (w < warp) before += count[w];
    found += count[w];
  }
  if (own.x > 0) {
    before += __popc(vote & ((1u << c % 32) - 1));
    record[before] = own;
    first_cta[before] = c;
  }
  __syncthreads();
  const int all = found * rows, warps = gridDim.x * (kJoinThreads / 32);
  const int at = blockIdx.x * (kJoinThreads / 32) + warp;
  if constexpr (FEW) {
    __shared__ float meet[kJoinThreads / 32][D + 1];
    if (all <= (int)gridDim.x)
      join_rows<A, D, 32, 16>(a, record, first_cta, all, rows, at / 16, warps / 16, meet);
    else
      join_rows<A, D, 32, 4>(a, record, first_cta, all, rows, at / 4, warps / 4, meet);
  } else if (all <= warps)
    join_rows<A, D, 32>(a, record, first_cta, all, rows, at, warps);
  else
    join_rows<A, D, 8>(a, record, first_cta, all, rows, 4 * at + c % 32 / 8, 4 * warps);
}

template <class A, int D>
int launch_join(const Launch& a, unsigned grid, int rows, const DeviceInfo& dev, cudaStream_t st) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(2 * dev.sm_count);
  config.blockDim = dim3(kJoinThreads);
  config.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  // (an item is split into blocks of rows, and no more of them end than there are CTAs)
  const int64_t items = a.p.batch * a.p.kv_heads * a.blocks;
  const bool few = (items < grid ? items : grid) * rows <= 4 * (int64_t)config.gridDim.x;
  if (cudaLaunchKernelEx(&config, few ? tree_join_kernel<A, D, true> : tree_join_kernel<A, D, false>, a,
                         rows, (int)grid) != cudaSuccess) {
    cudaGetLastError();
    return CT_ERR_LAUNCH_FAILED;
  }
  return CT_OK;
}

inline Launch begin_launch(const TreeAttention& p, const DeviceInfo& dev) {
  Launch a{};
  a.p = p;
  a.status = dev.status;
  // (not 0, so that scores of -inf, which mark what is not seen, stay so)
  a.c2 = fabsf(p.scale) * kLog2e;
  if (a.c2 < FLT_MIN) a.c2 = FLT_MIN;
  a.negative = p.scale < 0.0f;
  a.group = (int)(p.q_heads / p.kv_heads);
  const int64_t align = 16 / dtype_bytes(p.act_dtype);
  a.q_vectors = aligned16(p.q) && p.qs[0] % align == 0 && p.qs[1] % align == 0 &&
                p.qs[2] % align == 0 && p.qs[3] == 1;
  a.group_shift = -1;
  a.page_shift = -1;
  for (int s = 0; s < 31; ++s) {
      if (p.kv.page_size == 1 << s) a.page_shift = s;
      if (a.group == 1 << s) a.group_shift = s;
    }
  a.records = reinterpret_cast<int4*>(p.ws);
  a.partials = reinterpret_cast<float*>(a.records + kMaxCtas);
  return a;
}

// Boxes of the largest power of two of slots that fills pages and tiles, of 8 at
// least (the swizzle's period); a.box is 0 for pages without one.
inline void make_maps(Launch& a, CUtensorMap* k_map, CUtensorMap* v_map, int keys) {
  const PagedKv& kv = a.p.kv;
  a.box = 1;
  while (kv.page_size % (2 * a.box) == 0 && 2 * a.box <= keys) a.box *= 2;
  if (a.box < 8 || kv.pages == 0 ||
      make_tmap_pages(k_map, kv.k, kv.dtype, kv.pages, a.p.kv_heads, kv.page_size, a.p.head_dim,
                      kv.ks, a.box) != CT_OK ||
      make_tmap_pages(v_map, kv.v, kv.dtype, kv.pages, a.p.kv_heads, kv.page_size, a.p.head_dim,
                      kv.vs, a.box) != CT_OK)
    a.box = 0;
}

}  // namespace

// The call on tcgen05 (tree_attention_tc.cu); kNoTc where that does not take it.
constexpr int kNoTc = -1;
int launch_tc(const TreeAttention& p, const DeviceInfo& dev, cudaStream_t st);

}  // namespace tree
}  // namespace ct
