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

constexpr int kLogitsThreads = 512;
constexpr int kLogitsCounts = 16384;  // counts held at a time (64 KB)

// A cluster of CTAs per row, each with a slice of the vocabulary (a multiple of 32 tokens). Per up to
// kLogitsCounts tokens of it: the history's counts in shared memory (bit 31: the token occurs before the output;
// integer atomics, so the order does not matter), then one pass over the logits. The best token goes
// through the CTAs' shared memory to the cluster's first one. Bound by HBM (one read, one write) when
// there are many rows, by the chain history -> counts -> logits for a single one.
// VEC: eight tokens per thread and step, all rows on 16-byte boundaries.
template <typename T, typename I, bool VEC>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const __grid_constant__ LogitsParams p, int slice, int ctas) {
  extern __shared__ __align__(16) uint32_t cnt[];
  __shared__ float bv[kLogitsThreads / 32];
  __shared__ int bi[kLogitsThreads / 32];
  __shared__ unsigned long long mine;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int vbeg = rank * slice, vend = min(p.V, vbeg + slice);
  pdl_wait();
  const I* hist = (const I*)p.history + b * p.hist_ld;
  const int start = p.starts ? p.starts[b] : 0;
  const float r = p.rep ? p.rep[b] : p.rep1, pr = p.pres ? p.pres[b] : p.pres1, f = p.freq ? p.freq[b] : p.freq1;
  const T* x = (const T*)p.logits + b * p.ld;
  float* z = p.out + b * p.out_ld;
  const float* bias = p.bias ? p.bias + b * p.bias_ld : nullptr;
  const uint32_t* mask = p.mask ? p.mask + b * p.mask_ld : nullptr;
  float best = -INFINITY;
  int at = 0x7fffffff;
  auto one_token = [&](float v, uint32_t u, int tok, float add, bool allowed) -> float {
    if (u) {
      v = v > 0.f ? v / r : v * r;
      const uint32_t n = u & 0x7fffffffu;
      if (n) v -= f * (float)n + pr;
    }
    if (bias) v += add;
    if (!allowed) v = -INFINITY;
    if (v > best) {
      best = v;
      at = tok;
    }
    return v;
  };
  for (int v0 = vbeg; v0 < vend; v0 += kLogitsCounts) {
    const int n = min(kLogitsCounts, vend - v0);
    if (p.T) {
      if (v0 != vbeg) __syncthreads();
      for (int i = tid * 4; i < n; i += kLogitsThreads * 4) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
#pragma unroll 4
      for (int t = tid; t < p.T; t += kLogitsThreads) {
        const uint64_t id = (uint64_t)(int64_t)hist[t] - (uint64_t)v0;
        if (id < (uint64_t)n) {
          if (t >= start) atomicAdd(&cnt[id], 1u);
          else atomicOr(&cnt[id], 0x80000000u);
        }
      }
      __syncthreads();
    }
    if (VEC) {
      for (int i = tid * 8; i < n; i += kLogitsThreads * 8) {
        float v[8], add[8];
        load8(x + v0 + i, v);
        if (bias) load8(bias + v0 + i, add);
        const uint32_t bits = mask ? mask[(v0 + i) >> 5] >> (i & 31) : 0xffu;
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (p.T) {
          u0 = *reinterpret_cast<const uint4*>(cnt + i);
          u1 = *reinterpret_cast<const uint4*>(cnt + i + 4);
        }
        const uint32_t u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = one_token(v[k], u[k], v0 + i + k, bias ? add[k] : 0.f, bits >> k & 1);
        store8(z + v0 + i, v);
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < n; i += kLogitsThreads)
        z[v0 + i] = one_token(ld<T>(x + v0 + i), p.T ? cnt[i] : 0u, v0 + i, bias ? bias[v0 + i] : 0.f,
                              mask ? mask[(v0 + i) >> 5] >> (i & 31) & 1 : 1);
    }
  }
  if (!p.best) return;
  auto better = [&](float v, int i) {
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (lane == 0) {
    bv[warp] = best;
    bi[warp] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLogitsThreads / 32; ++w) better(bv[w], bi[w]);
    mine = (unsigned long long)__float_as_uint(best) << 32 | (uint32_t)at;
  }
  if (ctas > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && tid == 0)
      for (int k = 1; k < ctas; ++k) {
        uint32_t far;
        unsigned long long o;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(smem_u32(&mine)), "r"(k));
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(o) : "r"(far) : "memory");
        better(__uint_as_float((uint32_t)(o >> 32)), (int)(uint32_t)o);
      }
    // nobody leaves while the first CTA reads
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (rank == 0 && tid == 0) p.best[b] = at == 0x7fffffff ? 0 : at;
}

}  // namespace one
