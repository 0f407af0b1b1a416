// Penalties, bias and token mask on a step's logits, before the sampler or the argmax.
//
//   z = x                                               fp32, whatever the logits' type
//   z = z > 0 ? z / r : z * r     if the token is in the row's history   (repetition penalty r)
//   z = z - (f * c + p * [c > 0]) c: times the token stands in the history from output_start on
//   z = z + bias[token]
//   z = -inf                      if the token's bit in the mask is 0
//
// History entries outside [0, vocab) are padding. The argmax takes the lowest token among equal
// scores; NaN scores are never taken (as the sampler never draws them), a row with nothing left
// gives token 0.
#pragma once

#include "common.cuh"

namespace one {

struct LogitsParams {
  const void* logits;
  int64_t ld;
  int B, V;
  const void* history;
  int64_t hist_ld;
  int T;
  const int* starts;
  const float *rep, *pres, *freq;  // per row, or null: the scalars
  float rep1, pres1, freq1;
  const float* bias;
  int64_t bias_ld;
  const uint32_t* mask;
  int64_t mask_ld;
  float* out;
  int64_t out_ld;
  int* best;
};

constexpr int kLogitsChunk = 8192;  // tokens whose counts are held at a time

// One CTA per row, the vocabulary in chunks: counts of the row's history in shared memory (bit 31:
// the token occurred at all), then one pass over the chunk.
template <typename T, typename I>
__global__ void __launch_bounds__(512) logits_simple_kernel(const LogitsParams p) {
  pdl_wait();
  __shared__ uint32_t cnt[kLogitsChunk];
  __shared__ float bv[512];
  __shared__ int bi[512];
  const int b = blockIdx.x, tid = threadIdx.x;
  const I* hist = (const I*)p.history + b * p.hist_ld;
  const int start = p.starts ? p.starts[b] : 0;
  const float r = p.rep ? p.rep[b] : p.rep1, pr = p.pres ? p.pres[b] : p.pres1, f = p.freq ? p.freq[b] : p.freq1;
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int v0 = 0; v0 < p.V; v0 += kLogitsChunk) {
    const int n = min(kLogitsChunk, p.V - v0);
    for (int i = tid; i < n; i += blockDim.x) cnt[i] = 0;
    __syncthreads();
    for (int t = tid; t < p.T; t += blockDim.x) {
      const int64_t id = (int64_t)hist[t] - v0;
      if (id >= 0 && id < n) {
        if (t >= start) atomicAdd(&cnt[id], 1u);
        atomicOr(&cnt[id], 0x80000000u);
      }
    }
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
      const int v = v0 + i;
      float x = ld<T>((const T*)p.logits + b * p.ld + v);
      const uint32_t u = cnt[i], c = u & 0x7fffffffu;
      if (u) x = x > 0.f ? x / r : x * r;
      if (c) x -= f * (float)c + pr;
      if (p.bias) x += p.bias[b * p.bias_ld + v];
      if (p.mask && !((p.mask[b * p.mask_ld + (v >> 5)] >> (v & 31)) & 1u)) x = -INFINITY;
      p.out[b * p.out_ld + v] = x;
      if (x > best) {
        best = x;
        at = v;
      }
    }
    __syncthreads();
  }
  if (!p.best) return;
  bv[tid] = best;
  bi[tid] = at;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < (int)blockDim.x; ++i)
      if (bv[i] > best || (bv[i] == best && bi[i] < at)) {
        best = bv[i];
        at = bi[i];
      }
    p.best[b] = at == 0x7fffffff ? 0 : at;
  }
}

}  // namespace one
