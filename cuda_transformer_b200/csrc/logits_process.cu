// logits_process.cu -- penalties for repeated tokens, token biases and a
// grammar's bit mask on rows of logits.
//
// For a row with history h[0 .. n) of which the first m tokens are the prompt,
//   seen(i) = i is in h[0 .. n),  count(i) = occurrences of i in h[m .. n)
//   x = logit(i);  if seen(i): x = x > 0 ? x / r : x * r
//   x -= frequency * count(i) + presence * (count(i) > 0)
//   x += sum of the row's biases for i;  x = -inf where i's mask bit is 0
// in FP32.  Biases listed twice for a token are added in their order.
#include "decode_common.cuh"

namespace ct {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // vocabulary entries a CTA holds counters for

template <class T>
__global__ void __launch_bounds__(kThreads) logits_process_kernel(const LogitsProcess p) {
  __shared__ uint32_t hist[kChunk];  // bit 0: in the prompt; above: generated count
  const int64_t chunks = (p.vocab + kChunk - 1) / kChunk;
  const int64_t r = blockIdx.x / chunks, first = (blockIdx.x % chunks) * kChunk;
  const int width = (int)(p.vocab - first < kChunk ? p.vocab - first : kChunk);
  for (int i = threadIdx.x; i < kChunk; i += kThreads) hist[i] = 0u;
  __syncthreads();
  if (p.tokens) {
    int64_t n = p.lens ? p.lens[r] : p.max_len;
    n = n < 0 ? 0 : n > p.max_len ? p.max_len : n;
    const int64_t m = p.prompt_lens ? p.prompt_lens[r] : 0;
    for (int64_t j = threadIdx.x; j < n; j += kThreads) {
      const int64_t id = p.tokens[r * p.tokens_ld + j] - first;
      if (id >= 0 && id < width) {
        if (j < m)
          atomicOr(&hist[id], 1u);
        else
          atomicAdd(&hist[id], 2u);
      }
    }
  }
  __syncthreads();
  const float rep = p.repetition ? p.repetition[r] : 1.0f;
  const float freq = p.frequency ? p.frequency[r] : 0.0f;
  const float pres = p.presence ? p.presence[r] : 0.0f;
  const T* src = (const T*)p.logits + r * p.ld + first;
  float* dst = p.out + r * p.out_ld + first;
  const uint32_t* mask = p.mask ? p.mask + r * p.mask_ld : nullptr;
  for (int i = threadIdx.x; i < width; i += kThreads) {
    float x = to_f32(src[i]);
    const uint32_t w = hist[i];
    if (w) {
      x = x > 0.0f ? x / rep : x * rep;
      if (w >> 1) x -= freq * (float)(w >> 1) + pres;
    }
    if (mask && !(mask[(first + i) >> 5] >> ((first + i) & 31) & 1u)) x = -INFINITY;
    dst[i] = x;
  }
  if (p.bias_n == 0) return;
  __syncthreads();
  const int64_t* ids = p.bias_ids + r * p.bias_ld;
  const float* values = p.bias_values + r * p.bias_values_ld;
  for (int64_t j = threadIdx.x; j < p.bias_n; j += kThreads) {
    const int64_t id = ids[j];
    if (id < first || id >= first + width) continue;
    if (mask && !(mask[id >> 5] >> (id & 31) & 1u)) continue;
    // the first entry of a token adds all of its entries
    float x = dst[id - first];
    bool earlier = false;
    for (int64_t i = 0; i < j && !earlier; ++i) earlier = ids[i] == id;
    if (earlier) continue;
    for (int64_t i = j; i < p.bias_n; ++i)
      if (ids[i] == id) x += values[i];
    dst[id - first] = x;
  }
}

}  // namespace

int launch_logits_process(const LogitsProcess& p, cudaStream_t st) {
  const int64_t blocks = p.rows * ((p.vocab + kChunk - 1) / kChunk);
  if (blocks > 0x7fffffffll) return CT_ERR_INVALID_ARGUMENT;
  return with_dtype(p.dtype, [&](auto t) {
    logits_process_kernel<decltype(t)><<<(unsigned)blocks, kThreads, 0, st>>>(p);
    return check_launch();
  });
}

}  // namespace ct
