// logits_process.cu -- penalties for repeated tokens, token biases and a
// grammar's bit mask on rows of logits.
//
// For a row with history h[0 .. n) of which the first m tokens are the prompt,
//   seen(i) = i is in h[0 .. n),  count(i) = occurrences of i in h[m .. n)
//   x = logit(i);  if seen(i): x = x > 0 ? x / r : x * r
//   x -= frequency * count(i) + presence * (count(i) > 0)
//   x += each of the row's biases for i;  x = -inf where i's mask bit is 0
// in FP32.  Biases listed twice for a token are added in their order.
//
// Bound by HBM: a logit is read once and written once; all but the mask
// concerns a few thousand tokens of a row.  So one kernel streams the rows
// through with the mask applied and nothing to wait for, and a second one
// counts the histories in shared memory and mends the outputs of the tokens
// that it found.  The second is launched so that it counts while the first
// still streams (programmatic dependent launch) and waits for it before it
// touches an output.  A CTA of the second takes the token ids of a row that
// leave one remainder, so that the small ids, which make up most of a text,
// are spread.  Integer counts do not depend on the order of the atomics.
//
// Device time on a B200 (floor: bytes at the 6.53 TB/s of a copy):
//   256 x 100256 FP32, mask                     33.4 us   floor 31.9 (95 %)
//   the same, histories of 64 / 64 .. 8192 / 8192 tokens, 64 biases
//                            41 / 53 / 72         floor 32 to 34
//   256 x 100256, 300 / 500 biases              42.7 / 47.0
//   33 x 50257 bf16, histories up to 2048, mask 7.7       1.6
//   1 x 100256, history of 256, 16 biases       4.8       0.1
//   1 x 100256, 100256 biases (a row's are gathered 512 at a time) 296
// The mending alone takes 8 / 23 / 52 us: a history of 8192 is counted in 8,
// and its few thousand outputs are single sectors, read and written.  The
// overlap saves 3 (256 x 100256: 54.5 us against 57.7).  What else was tried
// with 256 x 100256 logits and histories of 64 to 8192: counting within the
// streaming kernel, a piece of the vocabulary a CTA (90 us: each waits for its
// own counts); a cluster for each row (103 to 141); and one mending CTA beside
// three streaming ones on an SM, which counts all of its rows while they
// stream and keeps the results in shared memory (73 to 99: the shared memory
// is the L1 that the streaming loads pass through, 33 us becomes 47).  Taking the
// rows with the longest histories first gave less than finding them cost.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kStreamThreads = 256;
constexpr int kVec = 4;    // logits of an access
constexpr int kLoads = 4;  // accesses of a thread that are on the way at once
constexpr int kRounds = 2;  // of loads of a CTA
constexpr int kBlock = kStreamThreads * kVec;

// Bits 0 .. 3 of the result: tokens id .. id + 3 (ids past the row's last word
// read as 0).
template <bool WHOLE>
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* mask, uint32_t id, uint32_t words) {
  const uint32_t w = id >> 5, shift = id & 31;
  const uint32_t low = __ldg(mask + w);
  if (WHOLE) return low >> shift;  // (id a multiple of 4)
  const uint32_t high = shift > 28 && w + 1 < words ? __ldg(mask + w + 1) : 0u;
  return __funnelshift_r(low, high, shift);
}

// out = logits, -inf where the mask has a 0.  Rows start at any multiple of
// the element size: the tokens up to the first whole vector are single
// accesses, and so are all of a row whose logits and outputs are not aligned
// alike (`vectors` false: 39.3 us instead of 33.4 for 256 x 100256).
template <class T>
__device__ __forceinline__ void stream_piece(const LogitsProcess& p, int64_t item, int piece,
                                             int pieces, bool vectors) {
  struct alignas(sizeof(T) * kVec) In {
    T v[kVec];
  };
  const int64_t r = (uint32_t)item / (uint32_t)pieces;
  const T* src = (const T*)p.logits + r * p.ld;
  float* dst = p.out + r * p.out_ld;
  const uint32_t* mask = p.mask ? p.mask + r * p.mask_ld : nullptr;
  const uint32_t vocab = (uint32_t)p.vocab, words = (vocab + 31) / 32;
  const uint32_t begin = (uint32_t)(item - r * pieces) * (uint32_t)piece;
  const uint32_t end = vocab - begin < (uint32_t)piece ? vocab : begin + (uint32_t)piece;
  auto one = [&](uint32_t i) {
    const float x = to_f32(src[i]);
    dst[i] = !mask || (mask[i >> 5] >> (i & 31) & 1u) ? x : -INFINITY;
  };
  if (!vectors) {
    constexpr int kSingles = 2 * kLoads;
    for (uint32_t at = begin + threadIdx.x; at < end; at += kSingles * kStreamThreads) {
      T x[kSingles];
      uint32_t word[kSingles];
#pragma unroll
      for (int k = 0; k < kSingles; ++k) {
        const uint32_t i = at + k * kStreamThreads;
        if (i < end) {
          x[k] = src[i];
          word[k] = mask ? mask[i >> 5] : 0xffffffffu;
        }
      }
#pragma unroll
      for (int k = 0; k < kSingles; ++k) {
        const uint32_t i = at + k * kStreamThreads;
        if (i < end) dst[i] = word[k] >> (i & 31) & 1u ? to_f32(x[k]) : -INFINITY;
      }
    }
    return;
  }
  // tokens before the row's first whole vector; every piece begins and ends
  // that much later, but for the row's own ends
  const uint32_t head = (uint32_t)(-(int64_t)(reinterpret_cast<uintptr_t>(dst) / 4) & (kVec - 1));
  if (begin == 0 && threadIdx.x < head && threadIdx.x < vocab) one(threadIdx.x);
  const uint32_t stop = vocab - end < head ? vocab : end + head;
  // MASK: 0 none, 1 four bits of one word, 2 of one or two
  auto stream = [&](auto kind) {
    constexpr int MASK = decltype(kind)::value;
    for (uint32_t at = begin + head + threadIdx.x * kVec; at < stop; at += kLoads * kBlock) {
      In in[kLoads];
      uint32_t bits[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const uint32_t i = at + k * kBlock;
        if (i + kVec <= stop) {
          in[k] = *reinterpret_cast<const In*>(src + i);
          bits[k] = MASK == 0 ? 0xfu : mask_bits<MASK == 1>(mask, i, words);
        }
      }
#pragma unroll
      for (int k = 0; k < kLoads; ++k) {
        const uint32_t i = at + k * kBlock;
        if (i + kVec <= stop) {
          float4 x;
          x.x = bits[k] & 1u ? to_f32(in[k].v[0]) : -INFINITY;
          x.y = bits[k] & 2u ? to_f32(in[k].v[1]) : -INFINITY;
          x.z = bits[k] & 4u ? to_f32(in[k].v[2]) : -INFINITY;
          x.w = bits[k] & 8u ? to_f32(in[k].v[3]) : -INFINITY;
          *reinterpret_cast<float4*>(dst + i) = x;
        } else {
          for (uint32_t j = i; j < stop; ++j) one(j);
        }
      }
    }
  };
  if (!mask)
    stream(std::integral_constant<int, 0>{});
  else if (head == 0)
    stream(std::integral_constant<int, 1>{});
  else
    stream(std::integral_constant<int, 2>{});
}

template <class T>
__global__ void __launch_bounds__(kStreamThreads, 5)
    logits_stream_kernel(const __grid_constant__ LogitsProcess p, const int piece, const int pieces,
                         const bool vectors) {
  asm volatile("griddepcontrol.launch_dependents;");
  stream_piece<T>(p, blockIdx.x, piece, pieces, vectors);
}

// (256 x 100256, histories of 64 to 8192: 53.3 us; 512 threads and 8 reads 54.6,
// 1024 threads 57 to 59)
constexpr int kMendThreads = 768;
constexpr int kMendShared = 108 * 1024 - 64;  // most of a CTA beside its 5 KB of biases: two an SM
constexpr int kListed = 4096;           // tokens that the list holds
constexpr int kMends = 4;               // tokens of a thread that are on the way at once
constexpr int kBiases = 512;            // of a CTA that are in shared memory at a time
constexpr int kMostEntries = 65536;     // (the list holds 16 bits)

constexpr int kReads = 4;               // of the history, of a thread, likewise
constexpr uint32_t kNoToken = 0xffffffffu;  // (ids are below 2^31)

// A CTA: the tokens of row r with id % 2^shift == part, id >> shift their index;
// `entries` indices.  A mark is the number of times a token was generated,
// times two, plus one if it is in the prompt; in 16 bits where no history is
// longer than they count (WIDE: 32).  Tokens are listed when they are first
// found, so that their outputs are fetched together; should there be more than
// the list holds, the rest are looked for among the marks.
template <bool WIDE>
__global__ void __launch_bounds__(kMendThreads, 2)
    logits_mend_kernel(const __grid_constant__ LogitsProcess p, const int shift, const int entries,
                       const bool dependent) {
  extern __shared__ __align__(16) uint32_t marks[];
  constexpr int kPerWord = WIDE ? 1 : 2;
  const int words = (entries + 4 * kPerWord - 1) / (4 * kPerWord) * 4;
  uint16_t* const list = reinterpret_cast<uint16_t*>(marks + words);
  __shared__ alignas(16) uint32_t bias_id[kBiases];
  __shared__ float bias_value[kBiases];
  __shared__ int16_t bias_link[kBiases];  // the token's next entry, -1: none
  __shared__ int listed, biases;
  __shared__ int64_t bias_next;
  const int64_t r = blockIdx.x >> shift;
  const uint32_t part = blockIdx.x & ((1u << shift) - 1);
  const uint32_t vocab = (uint32_t)p.vocab;
  const int lane = threadIdx.x % 32;
  const uint32_t* mask = p.mask ? p.mask + r * p.mask_ld : nullptr;
  float* dst = p.out + r * p.out_ld;
  int64_t n = 0, m = 0;
  if (p.tokens) {
    n = p.lens ? p.lens[r] : p.max_len;
    n = n < 0 ? 0 : n > p.max_len ? p.max_len : n;
    m = p.prompt_lens ? p.prompt_lens[r] : 0;
  }
  auto is_mine = [&](uint32_t token) {
    return token != kNoToken && (token & ((1u << shift) - 1)) == part;
  };
  auto known = [&](int64_t id) { return (uint64_t)id < vocab ? (uint32_t)id : kNoToken; };
  auto allowed = [&](uint32_t id) { return !mask || (mask[id >> 5] >> (id & 31) & 1u); };

  if (n > 0)
    for (int i = threadIdx.x; i < words / 4; i += kMendThreads)
      reinterpret_cast<uint4*>(marks)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();

  // ---- the biases of these tokens in their order: from entry j0 on, as many as
  // surely fit, by the last warp
  const int64_t* ids = p.bias_ids + r * p.bias_ld;
  const float* values = p.bias_values + r * p.bias_values_ld;
  auto gather = [&](int64_t j0) {
    int found = 0;
    for (; j0 < p.bias_n && found + 32 * kReads <= kBiases; j0 += 32 * kReads) {
      uint32_t id[kReads];
      float value[kReads];
#pragma unroll
      for (int k = 0; k < kReads; ++k) {
        const int64_t j = j0 + lane + k * 32;
        id[k] = j < p.bias_n ? known(ids[j]) : kNoToken;
        value[k] = j < p.bias_n ? values[j] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kReads; ++k) {
        const bool mine = is_mine(id[k]);
        const uint32_t vote = __ballot_sync(0xffffffffu, mine);
        if (mine) {
          const int at = found + __popc(vote & ((1u << lane) - 1));
          bias_id[at] = id[k];
          bias_value[at] = value[k];
        }
        found += __popc(vote);
      }
    }
    if (found + lane < (found + 3) / 4 * 4) bias_id[found + lane] = kNoToken;  // (read in fours)
    if (lane == 0) {
      biases = found;
      bias_next = j0;
    }
  };
  const bool gathers = threadIdx.x >= kMendThreads - 32;
  if (p.bias_n > 0 && gathers) gather(0);
  // ---- the history
  const int64_t* history = p.tokens + r * p.tokens_ld;
  for (int64_t j0 = threadIdx.x; j0 - threadIdx.x < n; j0 += kReads * kMendThreads) {
    uint32_t token[kReads];
#pragma unroll
    for (int k = 0; k < kReads; ++k) {
      const int64_t j = j0 + k * kMendThreads, id = j < n ? history[j] : -1;
      token[k] = known(id);
    }
#pragma unroll
    for (int k = 0; k < kReads; ++k) {
      if (j0 - threadIdx.x + k * kMendThreads >= n) break;
      bool first = false;
      const uint32_t i = token[k] >> shift;
      if (is_mine(token[k])) {
        const uint32_t up = WIDE ? 0u : 16u * (i & 1u);
        const uint32_t old = j0 + k * kMendThreads < m
                                 ? atomicOr(&marks[i / kPerWord], 1u << up)
                                 : atomicAdd(&marks[i / kPerWord], 2u << up);
        first = WIDE ? old == 0u : (old >> up & 0xffffu) == 0u;
      }
      const uint32_t vote = __ballot_sync(0xffffffffu, first);
      if (vote == 0u) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(&listed, __popc(vote));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(vote & ((1u << lane) - 1));
      if (first && at < kListed) list[at] = (uint16_t)i;
    }
  }
  __syncthreads();
  // the first of a token's gathered entries adds them all to its output, in their
  // order (so that it does not matter how many are gathered at a time)
  bool leads = false;
  auto look_around = [&]() {
    const int kept = biases, mine = threadIdx.x;
    leads = mine < kept;
    if (!leads) return;
    const uint32_t id = bias_id[mine];
    int link = -1;
    for (int i = (kept + 3) / 4 * 4 - 4; i >= 0; i -= 4) {
      const uint4 four = *reinterpret_cast<const uint4*>(bias_id + i);
      if (four.x != id && four.y != id && four.z != id && four.w != id) continue;
      const uint32_t each[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        if (each[e] != id || i + e == mine) continue;
        if (i + e > mine)
          link = i + e;
        else
          leads = false;
      }
    }
    bias_link[mine] = (int16_t)link;
  };
  if (p.bias_n > 0) look_around();
  if (dependent) asm volatile("griddepcontrol.wait;" ::: "memory");

  if (n > 0) {
    const float rep = p.repetition ? p.repetition[r] : 1.0f;
    const float freq = p.frequency ? p.frequency[r] : 0.0f;
    const float pres = p.presence ? p.presence[r] : 0.0f;
    using Mark = std::conditional_t<WIDE, uint32_t, uint16_t>;
    Mark* const mark_of = reinterpret_cast<Mark*>(marks);
    auto mended = [&](float x, uint32_t mark) {
      const uint32_t count = mark >> 1;
      // (the roundings are spelled out: a row's result does not depend on
      // which of the two places mends it)
      const float y = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      return count ? __fsub_rn(y, fmaf(freq, (float)count, pres)) : y;
    };
    const int in_list = listed < kListed ? listed : kListed;
    for (int k0 = threadIdx.x; k0 < in_list; k0 += kMends * kMendThreads) {
      uint32_t id[kMends], mark[kMends];
      float x[kMends];
#pragma unroll
      for (int k = 0; k < kMends; ++k) {
        mark[k] = 0u;
        if (k0 + k * kMendThreads >= in_list) continue;
        const uint32_t i = list[k0 + k * kMendThreads];
        id[k] = i << shift | part;
        if (allowed(id[k])) {  // (else it stays -inf)
          mark[k] = mark_of[i];
          x[k] = dst[id[k]];
        }
        if (listed > kListed) mark_of[i] = 0;
      }
#pragma unroll
      for (int k = 0; k < kMends; ++k)
        if (mark[k] != 0u) dst[id[k]] = mended(x[k], mark[k]);
    }
    if (listed > kListed) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < (uint32_t)entries; i += kMendThreads) {
        const uint32_t id = i << shift | part;
        if (mark_of[i] != 0 && allowed(id)) dst[id] = mended(dst[id], mark_of[i]);
      }
    }
  }
  if (p.bias_n == 0) return;
  while (true) {
    __syncthreads();
    if (leads && allowed(bias_id[threadIdx.x])) {
      const uint32_t id = bias_id[threadIdx.x];
      float x = dst[id];
      for (int i = threadIdx.x; i >= 0; i = bias_link[i]) x += bias_value[i];
      dst[id] = x;
    }
    const int64_t next = bias_next;
    if (next >= p.bias_n) return;
    __syncthreads();
    if (gathers) gather(next);
    __syncthreads();
    look_around();
  }
}

template <class T>
int launch_stream(const LogitsProcess& p, const DeviceInfo& dev, cudaStream_t st) {
  // Some rounds of loads a CTA, one or less where that would leave SMs without
  // work (1 x 100256: 1.8 us against 2.4).
  int piece = kRounds * kLoads * kBlock;
  while (piece > kBlock && p.rows * ((p.vocab + piece - 1) / piece) < 4 * dev.sm_count) piece /= 2;
  const int64_t pieces = (p.vocab + piece - 1) / piece;
  if (p.rows * pieces > 0x7fffffffll) return CT_ERR_INVALID_ARGUMENT;
  // vectors of logits and of outputs start at the same tokens, in every row
  const uintptr_t x = reinterpret_cast<uintptr_t>(p.logits), y = reinterpret_cast<uintptr_t>(p.out);
  const bool vectors = x % sizeof(T) == 0 && y % 4 == 0 && (x / sizeof(T) - y / 4) % kVec == 0 &&
                       (p.ld - p.out_ld) % kVec == 0;
  logits_stream_kernel<T><<<(unsigned)(p.rows * pieces), kStreamThreads, 0, st>>>(p, piece,
                                                                                (int)pieces, vectors);
  return check_launch();
}

template <bool WIDE>
int launch_mend(const LogitsProcess& p, bool dependent, const DeviceInfo& dev, cudaStream_t st) {
  // The fewest parts of a row (each reads its history) whose marks and list fit
  // and that give every SM a CTA (64 x 100256: 13.1 us, with the fewest that fit
  // 13.8; 1 x 100256: 5.0 and 5.3).
  const int64_t most = p.tokens ? p.max_len : 0;
  int shift = 0;
  int64_t entries = p.vocab, bytes = 0;
  for (;; ++shift) {
    entries = (p.vocab + (1ll << shift) - 1) >> shift;
    const int64_t words = WIDE ? (entries + 3) / 4 * 4 : (entries + 7) / 8 * 4;
    bytes = most == 0 ? 0 : 4 * words + 2 * (most < kListed ? most : kListed);
    if (bytes <= kMendShared && entries <= kMostEntries &&
        (p.rows << shift >= dev.sm_count || entries <= 4096))
      break;
  }
  if (p.rows << shift > 0x7fffffffll) return CT_ERR_INVALID_ARGUMENT;
  constexpr auto kernel = logits_mend_kernel<WIDE>;
  const int rc = allow_shared<kernel>(kMendShared, dev);
  if (rc != CT_OK) return rc;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(p.rows << shift));
  config.blockDim = dim3(kMendThreads);
  config.dynamicSmemBytes = (size_t)bytes;
  config.stream = st;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p, shift, (int)entries, dependent);
  return e == cudaSuccess ? check_launch() : (int)CT_ERR_LAUNCH_FAILED;
}

}  // namespace

int launch_logits_process(const LogitsProcess& p, const DeviceInfo& dev, cudaStream_t st) {
  // in place and without a mask there is nothing to stream
  const bool stream = p.logits != p.out || p.mask;
  if (stream) {
    const int rc =
        with_dtype(p.dtype, [&](auto t) { return launch_stream<decltype(t)>(p, dev, st); });
    if (rc != CT_OK) return rc;
  }
  const int64_t most = p.tokens ? p.max_len : 0;
  if (most == 0 && p.bias_n == 0) return CT_OK;
  return most > 32767 ? launch_mend<true>(p, stream, dev, st) : launch_mend<false>(p, stream, dev, st);
}

}  // namespace ct
