// kv_pages.cu -- what a cache holds, moved about inside it: the kept ones of a
// sequence's last tokens move up (kv_compact), pages are copied (kv_copy_pages).
// Both work on all caches of a list (keys and values of every layer) at once.
//
// Bound by HBM: every moved value is read once and written once.  A thread
// moves 16 bytes at a time of one cache, head and place in the row (a column);
// where rows are not aligned to that, one element.
//
// Measured (device): the kept quarter of 64 trees of 16, 24 caches of 8 heads of 128,
// BF16: 8 us; a random half of 4 x 8192 tokens, 8 caches of 32 heads of 64: 248 us, 4.3
// TB/s of what has to move, and DRAM moves nothing else (0.54 GB read, 0.48 written while
// it runs): threads wait for their loads and for the lists.  The same caches with the
// first token dropped, which is one chain a sequence: 4.4 ms (the bytes take 0.33), the first
// 4, 64, 512: 2.8, 2.0, 0.43.  512 pages of 16 tokens, 24 caches: 127 us.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kThreads = 256;
// Moves of a thread that are on the way at once.
constexpr int kMoves = 8;

struct Columns {
  int row_units;   // of a head's row
  uint32_t count;  // units of a token: caches * heads * row_units
  uint32_t blocks;  // CTAs for them
};

// A column's base address and strides in units of T.
template <class T>
struct Column {
  T* base;
  int64_t page, slot;
};
template <class T>
__device__ __forceinline__ Column<T> column(const CacheList& caches, int heads, int row_units,
                                            int bytes, uint32_t c) {
  const uint32_t unit = c % (uint32_t)row_units, row = c / (uint32_t)row_units;
  const uint32_t head = row % (uint32_t)heads, t = row / (uint32_t)heads;
  char* base = (char*)caches.base[t] + head * caches.s[t][1] * bytes;
  return {(T*)base + unit, caches.s[t][0] * bytes / (int64_t)sizeof(T),
          caches.s[t][2] * bytes / (int64_t)sizeof(T)};
}

struct Place {
  int page, slot;  // page < 0: none
};
__device__ __forceinline__ Place place_of(const KvCompact& p, int64_t b, int64_t position) {
  Place at{-1, 0};
  if (position < 0 || position >= p.max_pages * p.page_size) return at;
  const int index = (int)position / p.page_size;
  const int page = p.table[b * p.table_s + index];
  if (page >= 0 && page < p.pages) at = {page, (int)position - index * p.page_size};
  return at;
}

// Drafts of at most this many tokens: a thread makes all moves of its column,
// kMoves at a time in their order, which is safe as the kept ones ascend (what a
// later move reads lies behind what the earlier ones wrote).  This way / as below, us,
// one layer (2 caches), 64 drafts of which every other token is kept: 128 tokens 12 /
// 18, 256 20 / 29, 512 50 / 69; 12 layers, 74 / 76, 143 / 144, 281 / 294.
constexpr int kShortDraft = 512;

template <class T>
__global__ void __launch_bounds__(kThreads)
    compact_short_kernel(const __grid_constant__ KvCompact p, const Columns cols, const int bytes) {
  __shared__ Place from[kShortDraft], to[kShortDraft];
  __shared__ int listed;
  const int64_t b = blockIdx.x / cols.blocks;
  const int base = p.context_lens[b];
  int n = p.counts[b];
  n = n > p.drafts ? (int)p.drafts : n;
  if (base < 0 || n <= 0) return;
  if (threadIdx.x < 32) {  // the moves that there are, in their order
    int found = 0;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + threadIdx.x, k = j < n ? p.keep[b * p.keep_ld + j] : 0;
      Place src{-1, 0}, dst{-1, 0};
      if (j < n && k > j) {
        src = place_of(p, b, (int64_t)base + k);
        dst = place_of(p, b, (int64_t)base + j);
      }
      const bool moves = src.page >= 0 && dst.page >= 0;
      const uint32_t vote = __ballot_sync(0xffffffffu, moves);
      if (moves) {
        const int at = found + __popc(vote & ((1u << threadIdx.x) - 1));
        from[at] = src;
        to[at] = dst;
      }
      found += __popc(vote);
    }
    if (threadIdx.x == 0) listed = found;
  }
  __syncthreads();
  const uint32_t c = blockIdx.x % cols.blocks * kThreads + threadIdx.x;
  if (c >= cols.count) return;
  const Column<T> col = column<T>(p.caches, (int)p.kv_heads, cols.row_units, bytes, c);
  const int moves = listed;
  for (int j0 = 0; j0 < moves; j0 += kMoves) {
    T x[kMoves];
#pragma unroll
    for (int k = 0; k < kMoves; ++k)
      if (j0 + k < moves) x[k] = col.base[from[j0 + k].page * col.page + from[j0 + k].slot * col.slot];
#pragma unroll
    for (int k = 0; k < kMoves; ++k)
      if (j0 + k < moves) col.base[to[j0 + k].page * col.page + to[j0 + k].slot * col.slot] = x[k];
  }
}

// Longer drafts: place x takes the value of place keep[x], which then takes that
// of keep[keep[x]], and so on up to a place that nothing moves to.  Such chains
// have no place in common (keep ascends, so no place is kept twice), and each
// begins at a place that is not kept itself.  So the chains run in parallel: a CTA
// has those that begin in kPlaces places, for the columns of its threads.  It lists
// the next moves of each, then makes them, kMoves at a time: what a batch reads is
// read before the batch writes.  keep[x] > x along a chain whatever keep holds, so
// each of them ends.
constexpr int kPlaces = 64;
constexpr int kListed = 256;
static_assert(kListed == kThreads, "a thread an entry");

struct Move {
  Place from, to;  // from.page < 0: none
};

template <class T>
__global__ void __launch_bounds__(kThreads, 4)
    compact_long_kernel(const __grid_constant__ KvCompact p, const Columns cols, const int bytes,
                        const uint32_t pieces) {
  __shared__ alignas(16) Move list[kListed];
  __shared__ int at[kPlaces], chains;  // where the chains are
  __shared__ bool kept[kPlaces];
  __shared__ int found[kThreads / 32];
  __shared__ uint8_t order[kListed];
  const uint32_t piece = blockIdx.x / cols.blocks;
  const int64_t b = piece / pieces;
  const int base = p.context_lens[b];
  const int n = p.counts[b] > p.drafts ? (int)p.drafts : p.counts[b];
  const int x0 = (int)(piece - b * pieces) * kPlaces;
  if (base < 0 || x0 >= n) return;
  const int32_t* keep = p.keep + b * p.keep_ld;
  const int tid = threadIdx.x;
  if (tid == 0) chains = 0;
  if (tid < kPlaces) kept[tid] = false;
  // the first kept one that is not before x0 (kThreads of them looked at at a time)
  int low = 0, high = x0 < n ? x0 : n;  // (keep[j] >= j)
  while (high > low) {
    const int step = (high - low + kThreads - 1) / kThreads, j = low + tid * step;
    const int before = __syncthreads_count(j < high && keep[j] < x0);
    if (before == 0) break;
    const int from = low + (before - 1) * step;  // keep[from] < x0
    high = from + step < high ? from + step : high;
    low = from + 1;
  }
  __syncthreads();
  if (tid < kPlaces && low + tid < n) {
    const int x = keep[low + tid] - x0;
    if (x >= 0 && x < kPlaces) kept[x] = true;
  }
  __syncthreads();
  if (tid < kPlaces && x0 + tid < n && !kept[tid] && keep[x0 + tid] > x0 + tid)
    at[atomicAdd(&chains, 1)] = x0 + tid;
  __syncthreads();
  const uint32_t c = blockIdx.x % cols.blocks * kThreads + tid;
  const bool mine = c < cols.count;
  const Column<T> col = column<T>(p.caches, (int)p.kv_heads, cols.row_units, bytes, mine ? c : 0);
  while (chains > 0) {
    const int active = chains, steps = kListed / active;
    // the next moves of each chain, in their order
    int x = tid < active ? at[tid] : n;
    if (tid < active) {
      Place to = place_of(p, b, (int64_t)base + x);
      for (int k = 0; k < steps; ++k) {
        Move m{{-1, 0}, {-1, 0}};
        const int y = x < n ? keep[x] : -1;
        if (x < n && y > x) {
          const Place from = place_of(p, b, (int64_t)base + y);
          if (to.page >= 0 && from.page >= 0) m = {from, to};
          to = from;
          x = y;
        } else {
          x = n;
        }
        list[tid * steps + k] = m;
      }
    }
    __syncthreads();
    if (tid == 0) chains = 0;
    // those that there are, close together, in their order
    const bool is_move = tid < active * steps && list[tid].from.page >= 0;
    const uint32_t vote = __ballot_sync(0xffffffffu, is_move);
    if (tid % 32 == 0) found[tid / 32] = __popc(vote);
    __syncthreads();
    int moves = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < tid / 32) before += found[w];
      moves += found[w];
    }
    if (is_move) order[before + __popc(vote & ((1u << tid % 32) - 1))] = (uint8_t)tid;
    __syncthreads();
    if (mine)
      for (int j0 = 0; j0 < moves; j0 += kMoves) {
        T value[kMoves];
#pragma unroll
        for (int k = 0; k < kMoves; ++k)
          if (j0 + k < moves) {
            const Place from = list[order[j0 + k]].from;
            value[k] = col.base[from.page * col.page + from.slot * col.slot];
          }
#pragma unroll
        for (int k = 0; k < kMoves; ++k)
          if (j0 + k < moves) {
            const Place to = list[order[j0 + k]].to;
            col.base[to.page * col.page + to.slot * col.slot] = value[k];
          }
      }
    __syncthreads();
    if (x < n) at[atomicAdd(&chains, 1)] = x;
    __syncthreads();
  }
}

// A thread copies kMoves slots of its column, all on the way at once.  (All of the page,
// one after the other: 8 pages of 16 tokens, 24 caches 6.3 us, here 4.2; 8 of 256 tokens
// 138, here 35.)
template <class T>
__global__ void __launch_bounds__(kThreads)
    copy_pages_kernel(const __grid_constant__ KvCopyPages p, const Columns cols, const int bytes,
                      const uint32_t pieces) {
  const uint32_t piece = blockIdx.x / cols.blocks;
  const int64_t i = piece / pieces, slot0 = (piece - i * pieces) * (int64_t)kMoves;
  const int src = p.src[i], dst = p.dst[i];
  if (src < 0 || src >= p.pages || dst < 0 || dst >= p.pages) return;
  const uint32_t c = blockIdx.x % cols.blocks * kThreads + threadIdx.x;
  if (c >= cols.count) return;
  const Column<T> col = column<T>(p.caches, (int)p.kv_heads, cols.row_units, bytes, c);
  T x[kMoves];
#pragma unroll
  for (int k = 0; k < kMoves; ++k)
    if (slot0 + k < p.page_size) x[k] = col.base[src * col.page + (slot0 + k) * col.slot];
#pragma unroll
  for (int k = 0; k < kMoves; ++k)
    if (slot0 + k < p.page_size) col.base[dst * col.page + (slot0 + k) * col.slot] = x[k];
}

// Whether the rows of all caches are whole 16-byte vectors.
bool rows_of_vectors(const CacheList& caches, int head_dim, int bytes) {
  bool ok = head_dim * bytes % 16 == 0;
  for (int t = 0; t < caches.n; ++t) {
    ok = ok && aligned16(caches.base[t]);
    for (int i = 0; i < 3; ++i) ok = ok && caches.s[t][i] * bytes % 16 == 0;
  }
  return ok;
}

// f with the type of a unit (16 bytes, or an element) and the columns.
template <class P, class F>
int with_units(const P& p, F&& f) {
  const int bytes = dtype_bytes(p.dtype);
  const bool vectors = rows_of_vectors(p.caches, p.head_dim, bytes);
  Columns cols;
  cols.row_units = vectors ? p.head_dim * bytes / 16 : p.head_dim;
  const int64_t count = p.caches.n * p.kv_heads * cols.row_units;
  if (count >= 1ll << 32) return CT_ERR_INVALID_ARGUMENT;
  cols.count = (uint32_t)count;
  cols.blocks = (uint32_t)((count + kThreads - 1) / kThreads);
  if (vectors) return f(uint4{}, cols, bytes);
  if (bytes == 4) return f(uint32_t{}, cols, bytes);
  return f(uint16_t{}, cols, bytes);
}

// The CTAs of `n` pieces of work, `each` a piece (0: more than a grid has).
unsigned grid_of(int64_t n, int64_t each) {
  return n * each < 1ll << 31 ? (unsigned)(n * each) : 0u;
}

}  // namespace

int launch_kv_compact(const KvCompact& p, const DeviceInfo&, cudaStream_t st) {
  return with_units(p, [&](auto unit, const Columns& cols, int bytes) {
    using T = decltype(unit);
    const bool is_short = p.drafts <= kShortDraft;
    const int64_t pieces = is_short ? 1 : (p.drafts + kPlaces - 1) / kPlaces;
    if (p.batch * pieces >= 1ll << 31) return (int)CT_ERR_INVALID_ARGUMENT;
    const unsigned grid = grid_of(p.batch * pieces, cols.blocks);
    if (grid == 0) return (int)CT_ERR_INVALID_ARGUMENT;
    if (is_short)
      compact_short_kernel<T><<<grid, kThreads, 0, st>>>(p, cols, bytes);
    else
      compact_long_kernel<T><<<grid, kThreads, 0, st>>>(p, cols, bytes, (uint32_t)pieces);
    return check_launch();
  });
}

int launch_kv_copy_pages(const KvCopyPages& p, const DeviceInfo&, cudaStream_t st) {
  return with_units(p, [&](auto unit, const Columns& cols, int bytes) {
    using T = decltype(unit);
    const int64_t pieces = (p.page_size + kMoves - 1) / kMoves;
    if (p.count * pieces >= 1ll << 31) return (int)CT_ERR_INVALID_ARGUMENT;
    const unsigned grid = grid_of(p.count * pieces, cols.blocks);
    if (grid == 0) return (int)CT_ERR_INVALID_ARGUMENT;
    copy_pages_kernel<T><<<grid, kThreads, 0, st>>>(p, cols, bytes, (uint32_t)pieces);
    return check_launch();
  });
}

}  // namespace ct
