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
#include <cooperative_groups.h>

#include "decode_common.cuh"

namespace ct {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostCtas = 8;  // of a cluster

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
__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyDrafts p) {
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

  // this CTA's part of the vocabulary, and this warp's of that
  const int vocab = (int)p.vocab;
  const int per_cta = (vocab + ctas - 1) / ctas;
  const int per_warp = (per_cta + kWarps - 1) / kWarps;
  const int cta_end = min(vocab, (rank + 1) * per_cta);
  const int begin = min(cta_end, rank * per_cta + warp * per_warp);
  const int end = min(cta_end, begin + per_warp);
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
    return mass(t, to_f32(target[current * p.ts[1] + t]),
                drafter ? to_f32(drafter[current * p.ds[1] + t]) : 0.0f);
  };
  // the sum of r; the parts of warps and CTAs stay in shared memory
  auto sum_row = [&]() -> double {
    double sum = 0.0;
    for (int t = begin + lane; t < end; t += 32) sum += mass_at(t);
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
    Best best{0.0f, -1};
    for (int t = begin + lane; t < end; t += 32) {
      const float x = to_f32(target[current * p.ts[1] + t]);
      best = better(best, x != x ? Best{0.0f, -2} : x == -INFINITY ? Best{0.0f, -1} : Best{x, t});
    }
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
        int found = -1, last = -1;
        for (int t0 = begin; t0 < end && found < 0; t0 += 32) {
          const double x = t0 + lane < end ? mass_at(t0 + lane) : 0.0;
          double run = x;
          for (int w = 1; w < 32; w *= 2) {
            const double y = __shfl_up_sync(0xffffffffu, run, w);
            if (lane >= w) run += y;
          }
          const uint32_t hit = __ballot_sync(0xffffffffu, x > 0.0 && before + run > mark);
          const uint32_t any = __ballot_sync(0xffffffffu, x > 0.0);
          if (hit) found = t0 + __ffs(hit) - 1;
          if (any) last = t0 + 31 - __clz(any);
          before += __shfl_sync(0xffffffffu, run, 31);
        }
        // (roundings can leave the mark behind the last of them)
        if (lane == 0) new_tokens[count - 1] = found >= 0 ? found : last;
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
int launch(const VerifyDrafts& p, cudaStream_t st) {
  int ctas = kMostCtas;
  while (ctas > 1 && p.vocab < ctas * 2048) ctas /= 2;
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

int launch_verify_drafts(const VerifyDrafts& p, const DeviceInfo&, cudaStream_t st) {
  return with_dtype(p.dtype, [&](auto t) { return launch<decltype(t)>(p, st); });
}

}  // namespace ct
