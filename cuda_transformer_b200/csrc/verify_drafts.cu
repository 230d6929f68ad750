// verify_drafts.cu -- which tokens of a draft (a tree or a chain) are kept, by
// the target's and the drafter's probabilities and given random numbers, and
// the token after them.
//
// From node 0 on, the children i of the last kept node are tried in their order.
// With r the target's row of that node, q the drafter's, Z = 1 at first:
//   kept when u_i q(x_i) Z < r(x_i);  refused: r <- max(r / Z - q, 0), Z <- sum r
// After k refusals r = max(a p - c q, 0) with a and c that follow from the sums,
//   a <- a / Z,  c <- c / Z + 1,
// so a row is never written: each sum is one pass over p and q.  Where proposals
// are certain (no q), q(x_i) counts as 1 and a refusal takes x_i out of r.  When
// no child is kept, the next token is where the running sum of r passes u_0 of
// the whole.  Without random numbers the best token decides at each place.
//
// All sums and products are FP64: a running sum of 100256 FP32 values would be off
// by more than many of the values, and the token drawn with it.
//
// A cluster of CTAs works on a sequence, each on a part of the vocabulary.  The
// probabilities of the proposals themselves are gathered first, all at once, so
// that the walk through the tree reads shared memory only, but for the passes.
//
// Bound by HBM where sequences are many (each pass reads a row of p, and of q), by the
// passes' latencies, each an exchange of the cluster, where they are few.  Measured
// (device; sampling with a drafter, n = 8): one sequence of 100,256 tokens 14 us, 64 of
// 50,257 18 us, 128 27 us; best tokens only: 8, 12 and 16 us.
#include <cooperative_groups.h>

#include "decode_common.cuh"

namespace ct {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kCtasSm = 4;
constexpr int kWarps = kThreads / 32;
constexpr int kMostCtas = 16;  // of a cluster
constexpr int kPortableCtas = 8;

struct Best {
  float value;
  int index;  // -1: none yet, -2: a NaN was met
};
__device__ __forceinline__ Best better(Best a, Best b) {
  if (a.index == -2 || b.index == -2) return {0.0f, -2};
  if (b.index == -1) return a;
  if (a.index == -1) return b;
  if (a.value != b.value) return a.value > b.value ? a : b;
  return a.index < b.index ? a : b;
}

// What a node of the tree is, for its place among its parent's children.
struct Node {
  int parent, token;  // token < 0: not tried
  float u, p, q;      // its number; probabilities of its token in its parent's rows
};

template <class T>
__global__ void __launch_bounds__(kThreads, kCtasSm) verify_kernel(const __grid_constant__ VerifyDrafts p) {
  extern __shared__ __align__(16) char shared[];
  Node* const node = reinterpret_cast<Node*>(shared);
  __shared__ double warp_sum[kWarps], cta_sum[2][kMostCtas];
  __shared__ Best warp_best[kWarps], cta_best[2][kMostCtas];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / ctas;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int n = p.draft_lens ? p.draft_lens[b] : (int)p.drafts;
  n = n < 0 ? 0 : n > p.drafts ? (int)p.drafts : n;
  const T* const target = (const T*)p.target + b * p.ts[0];
  const T* const drafter = p.draft_probs ? (const T*)p.draft_probs + b * p.ds[0] : nullptr;
  const bool greedy = p.uniform == nullptr;

  for (int i = 1 + threadIdx.x; i < n; i += kThreads) {
    Node x{p.parents ? p.parents[b * p.parents_ld + i] : i - 1, -1, 0.0f, 0.0f, 1.0f};
    const int64_t token = p.tokens[b * p.tokens_ld + i];
    if (token >= 0 && token < p.vocab && x.parent >= 0 && x.parent < i) {
      x.token = (int)token;
      if (!greedy) {
        x.u = p.uniform[b * p.uniform_ld + i];
        x.p = to_f32(target[x.parent * p.ts[1] + token]);
        if (drafter) x.q = to_f32(drafter[x.parent * p.ds[1] + token]);
      }
    }
    node[i] = x;
  }
  cluster.sync();  // (all of its CTAs run before one writes into another's memory)

  // This warp's part of a row: whole 16-byte vectors, evenly; the elements before the
  // first of them are the first warp's, those behind the last one the last warp's.
  const int vocab = (int)p.vocab;
  constexpr int VEC = 16 / (int)sizeof(T);
  const int part = rank * kWarps + warp, parts = ctas * kWarps;
  struct Vec {
    T v[VEC];
  };
  int head, first, last, tail;  // elements before the vectors; this warp's vectors
  const T *p_row, *q_row;
  auto set_row = [&](int at) {
    p_row = target + at * p.ts[1];
    q_row = drafter ? drafter + at * p.ds[1] : nullptr;
    head = (int)((16 - reinterpret_cast<uintptr_t>(p_row) % 16) % 16 / sizeof(T));
    // (rows that are aligned differently are read element by element)
    const bool alike = !drafter || (reinterpret_cast<uintptr_t>(p_row) -
                                    reinterpret_cast<uintptr_t>(q_row)) % 16 == 0;
    const int vectors = !alike || head > vocab ? 0 : (vocab - head) / VEC;
    if (vectors == 0) head = 0;
    first = (int)((int64_t)vectors * part / parts);
    last = (int)((int64_t)vectors * (part + 1) / parts);
    tail = head + vectors * VEC;
  };
  int parity = 0;

  int current = 0, last_refused = 0, refused = 0;
  double a = 1.0, c = 0.0, total = 1.0;
  bool summed = false;  // warp_sum and cta_sum are those of r
  // r(t) with the refused proposals of `current` taken out, where they are certain
  auto mass = [&](int t, float pt, float qt) -> double {
    if (drafter) {
      const double x = a * (double)pt - c * (double)qt;
      return x > 0.0 ? x : x != x ? x : 0.0;
    }
    if (refused > 0)
      for (int i = current + 1; i <= last_refused; ++i)
        if (node[i].token == t && node[i].parent == current) return 0.0;
    return (double)pt;
  };
  auto mass_at = [&](int t) -> double {
    return mass(t, to_f32(p_row[t]), drafter ? to_f32(q_row[t]) : 0.0f);
  };
  // single elements of this warp: [0, head) before its vectors, [tail, vocab) behind
  // them.  Without vectors a warp's elements are a part of [0, vocab).
  auto singles = [&](bool behind, int& from, int& to) {
    if (tail == 0) {
      from = behind ? 0 : (int)((int64_t)vocab * part / parts);
      to = behind ? 0 : (int)((int64_t)vocab * (part + 1) / parts);
    } else if (behind) {
      from = part == parts - 1 ? tail : vocab;
      to = vocab;
    } else {
      from = 0;
      to = part == 0 ? head : 0;
    }
  };
  constexpr int kLoads = 4;  // vectors of a lane that are on the way at once
  // the sum of r; the parts of warps and CTAs stay in shared memory
  auto sum_row = [&]() -> double {
    set_row(current);
    double sum = 0.0;
    for (int side = 0; side < 2; ++side) {
      int from, to;
      singles(side == 1, from, to);
      for (int t = from + lane; t < to; t += 32) sum += mass_at(t);
    }
    for (int i = first + lane; i < last; i += 32 * kLoads) {
      Vec pv[kLoads], qv[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        if (i + 32 * k < last) {
          *reinterpret_cast<uint4*>(&pv[k]) =
              *reinterpret_cast<const uint4*>(p_row + head + (int64_t)(i + 32 * k) * VEC);
          if (drafter)
            *reinterpret_cast<uint4*>(&qv[k]) =
                *reinterpret_cast<const uint4*>(q_row + head + (int64_t)(i + 32 * k) * VEC);
        }
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        if (i + 32 * k < last) {
          double each = 0.0;
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            each += mass(head + (i + 32 * k) * VEC + e, to_f32(pv[k].v[e]),
                         drafter ? to_f32(qv[k].v[e]) : 0.0f);
          sum += each;
        }
    }
    for (int w = 16; w; w /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    __syncthreads();  // (the last pass's sums have been read)
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    parity ^= 1;
    if (threadIdx.x < ctas) {
      double all = 0.0;
      for (int w = 0; w < kWarps; ++w) all += warp_sum[w];
      cluster.map_shared_rank(&cta_sum[parity][rank], threadIdx.x)[0] = all;
    }
    cluster.sync();
    double all = 0.0;
    for (int w = 0; w < ctas; ++w) all += cta_sum[parity][w];
    return all;
  };
  auto best_of_row = [&]() -> Best {
    set_row(current);
    // the largest value of a lane, its place (the lowest, as they come in order), NaN
    float top = -INFINITY;
    int where = -1;
    bool nan = false;
    auto take = [&](int t, float x) {
      nan = nan || x != x;
      if (x > top) {
        top = x;
        where = t;
      }
    };
    int from, to;
    singles(false, from, to);
    for (int t = from + lane; t < to; t += 32) take(t, to_f32(p_row[t]));
    for (int i = first + lane; i < last; i += 32 * kLoads) {
      Vec pv[kLoads];
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        if (i + 32 * k < last)
          *reinterpret_cast<uint4*>(&pv[k]) =
              *reinterpret_cast<const uint4*>(p_row + head + (int64_t)(i + 32 * k) * VEC);
#pragma unroll
      for (int k = 0; k < kLoads; ++k)
        if (i + 32 * k < last) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) take(head + (i + 32 * k) * VEC + e, to_f32(pv[k].v[e]));
        }
    }
    singles(true, from, to);
    for (int t = from + lane; t < to; t += 32) take(t, to_f32(p_row[t]));
    Best best{top, nan ? -2 : where};
    for (int w = 16; w; w /= 2)
      best = better(best, Best{__shfl_xor_sync(0xffffffffu, best.value, w),
                               __shfl_xor_sync(0xffffffffu, best.index, w)});
    __syncthreads();
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    parity ^= 1;
    if (threadIdx.x < ctas) {
      Best all{0.0f, -1};
      for (int w = 0; w < kWarps; ++w) all = better(all, warp_best[w]);
      cluster.map_shared_rank(&cta_best[parity][rank], threadIdx.x)[0] = all;
    }
    cluster.sync();
    Best all{0.0f, -1};
    for (int w = 0; w < ctas; ++w) all = better(all, cta_best[parity][w]);
    return all;
  };

  int64_t* const new_tokens = p.new_tokens + b * p.drafts;
  int32_t* const path = p.path + b * p.drafts;
  const bool writes = rank == 0 && threadIdx.x == 0;
  int count = n > 0 ? 1 : 0;
  if (writes && n > 0) path[0] = 0;
  auto keep = [&](int i) {
    if (writes) {
      new_tokens[count - 1] = node[i].token;
      path[count] = i;
    }
    ++count;
    current = i;
  };

  if (greedy) {
    while (count > 0) {
      const Best best = best_of_row();
      int next = 0;
      for (int i = current + 1; i < n && next == 0; ++i)
        if (node[i].parent == current && node[i].token >= 0 && node[i].token == best.index) next = i;
      if (next > 0) {
        keep(next);
        continue;
      }
      if (writes) new_tokens[count - 1] = best.index < 0 ? -1 : best.index;
      break;
    }
  } else if (n > 0) {
    for (int i = 1; i < n; ++i) {
      const Node x = node[i];
      if (x.parent != current || x.token < 0) continue;
      const double here = mass(x.token, x.p, x.q);
      if ((double)x.u * (double)x.q * total < here) {
        keep(i);
        a = total = 1.0;
        c = 0.0;
        refused = 0;
        summed = false;
        continue;
      }
      if (drafter) {
        const double old_a = a, old_c = c;
        a = a / total;
        c = c / total + 1.0;
        const double sum = sum_row();
        summed = sum > 0.0;
        if (summed) {
          total = sum;
        } else {
          a = old_a;
          c = old_c;
        }
      } else if (total - here > 0.0) {
        total -= here;
        ++refused;
        last_refused = i;
      }
    }
    if (!summed) total = sum_row();
    // the CTA, then the warp, in whose part the running sum passes the mark
    const double mark = (double)p.uniform[b * p.uniform_ld] * total;
    double before = 0.0, upto = 0.0;
    int owner = -1;
    for (int w = 0; w < ctas; ++w) {
      const double s = cta_sum[parity][w];
      if (s > 0.0 && (owner < 0 || upto <= mark)) {
        owner = w;
        before = upto;
      }
      upto += s;
    }
    if (!(total > 0.0)) {
      if (writes) new_tokens[count - 1] = -1;
    } else if (owner == rank) {
      int mine = -1;
      upto = before;
      for (int w = 0; w < kWarps; ++w) {
        if (warp_sum[w] > 0.0 && (mine < 0 || upto <= mark)) {
          mine = w;
          before = upto;
        }
        upto += warp_sum[w];
      }
      if (mine == warp) {
        int found = -1, last_one = -1;
        // the next elements in their order, N of each lane from t0 + lane N on
        auto look = [&](int t0, int end, auto count) {
          constexpr int N = decltype(count)::value;
          double x[N], run = 0.0;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int t = t0 + lane * N + e;
            x[e] = t < end ? mass_at(t) : 0.0;
            run += x[e];
          }
          const double own = run;
          for (int w = 1; w < 32; w *= 2) {
            const double y = __shfl_up_sync(0xffffffffu, run, w);
            if (lane >= w) run += y;
          }
          int hit = -1, any = -1;
          double upto_here = before + (run - own);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            upto_here += x[e];
            if (x[e] > 0.0) {
              any = t0 + lane * N + e;
              if (hit < 0 && upto_here > mark) hit = any;
            }
          }
          const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
          const uint32_t some = __ballot_sync(0xffffffffu, any >= 0);
          if (hits) found = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
          if (some) last_one = __shfl_sync(0xffffffffu, any, 31 - __clz(some));
          before += __shfl_sync(0xffffffffu, run, 31);
        };
        int from, to;
        singles(false, from, to);
        for (int t = from; t < to && found < 0; t += 32)
          look(t, to, std::integral_constant<int, 1>{});
        for (int i = first; i < last && found < 0; i += 32)
          look(head + i * VEC, head + last * VEC, std::integral_constant<int, VEC>{});
        singles(true, from, to);
        for (int t = from; t < to && found < 0; t += 32)
          look(t, to, std::integral_constant<int, 1>{});
        // (roundings can leave the mark behind the last of them)
        if (lane == 0) new_tokens[count - 1] = found >= 0 ? found : last_one;
      }
    }
  }
  if (rank == 0) {
    if (threadIdx.x == 0) p.counts[b] = count;
    for (int i = count + threadIdx.x; i < p.drafts; i += kThreads) {
      new_tokens[i] = -1;
      path[i] = -1;
    }
  }
}

template <class T>
int launch(const VerifyDrafts& p, const DeviceInfo& dev, cudaStream_t st) {
  // As many as one wave holds, each with 2048 tokens at least; two also in more than a
  // wave, which then ends more evenly.  Sampling, us: 8 sequences of 100,256 tokens with
  // 16 / 8 / 4 CTAs 14 / 20 / 29; 64 of 50,257 with 8 / 4 18 / 21; 128 of them in one
  // wave / half a wave / two 27 / 35 / 27 (best tokens 16 / 18 / 19); 512 of 32,000 with
  // two / one 54 / 62.  64 of 8192 with at least 2048 / 512 tokens a CTA 10.3 / 11.6.
  int ctas = kMostCtas;
  while (ctas > 1 && (p.vocab < ctas * 2048 ||
                      (ctas > 2 && p.batch * ctas > kCtasSm * dev.sm_count)))
    ctas /= 2;
  if (ctas > kPortableCtas) {
    static std::atomic<bool> done[64];
    if (dev.device >= 64 || !done[dev.device].load(std::memory_order_acquire)) {
      if (cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) !=
          cudaSuccess) {
        cudaGetLastError();
        return CT_ERR_CUDA;
      }
      if (dev.device < 64) done[dev.device].store(true, std::memory_order_release);
    }
  }
  if (p.batch * ctas >= 1ll << 31) return CT_ERR_INVALID_ARGUMENT;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)(p.batch * ctas));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = sizeof(Node) * p.drafts;
  config.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  if (cudaLaunchKernelEx(&config, verify_kernel<T>, p) != cudaSuccess) {
    cudaGetLastError();
    return CT_ERR_LAUNCH_FAILED;
  }
  return CT_OK;
}

}  // namespace

int launch_verify_drafts(const VerifyDrafts& p, const DeviceInfo& dev, cudaStream_t st) {
  return with_dtype(p.dtype, [&](auto t) { return launch<decltype(t)>(p, dev, st); });
}

}  // namespace ct
