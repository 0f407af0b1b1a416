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
constexpr int kLogitsBytes = 65536;   // counts held at a time
constexpr int kLogitsAhead = 2;       // vectors per thread, and
constexpr int kLogitsIds = 4;         // history entries per thread, that are asked for at once at the start

template <typename T> struct LogitsVec;  // four logits as they lie in memory
template <> struct LogitsVec<__nv_bfloat16> {
  using Raw = uint2;
  ONE_DEVINL static void open(Raw u, float (&v)[4]) {
    v[0] = bf2_lo(u.x); v[1] = bf2_hi(u.x); v[2] = bf2_lo(u.y); v[3] = bf2_hi(u.y);
  }
};
template <> struct LogitsVec<float> {
  using Raw = float4;
  ONE_DEVINL static void open(Raw u, float (&v)[4]) {
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
};

// How often the tokens of a slice stand in the history, as words of shared memory: 16 bits per token, or
// 32 for histories whose counts might not fit; the top bit says that the token occurs before the output.
template <bool WIDE> struct LogitsCounts;
template <> struct LogitsCounts<false> {
  static constexpr int N = kLogitsBytes / 2, kTop = 0x8000;
  ONE_DEVINL static void add(uint32_t* w, int i, bool output) {
    const int s = 16 * (i & 1);
    if (output) atomicAdd(w + (i >> 1), 1u << s);
    else atomicOr(w + (i >> 1), 0x8000u << s);
  }
  ONE_DEVINL static uint32_t get(const uint32_t* w, int i) { return w[i >> 1] >> 16 * (i & 1) & 0xffffu; }
  ONE_DEVINL static uint4 get4(const uint32_t* w, int i) {  // i a multiple of 4
    const uint2 u = *reinterpret_cast<const uint2*>(w + (i >> 1));
    return make_uint4(u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16);
  }
};
template <> struct LogitsCounts<true> {
  static constexpr int N = kLogitsBytes / 4;
  static constexpr uint32_t kTop = 0x80000000u;
  ONE_DEVINL static void add(uint32_t* w, int i, bool output) {
    if (output) atomicAdd(w + i, 1u);
    else atomicOr(w + i, 0x80000000u);
  }
  ONE_DEVINL static uint32_t get(const uint32_t* w, int i) { return w[i]; }
  ONE_DEVINL static uint4 get4(const uint32_t* w, int i) { return *reinterpret_cast<const uint4*>(w + i); }
};

// A cluster of CTAs per row, each with a slice of the vocabulary. Per up to Counts::N tokens of it: the
// history's counts in shared memory (integer atomics, so the order does not matter), then one pass over
// the logits. Bound by HBM (one read, one write) when there are many rows, by the chain history -> counts
// -> scores for a single one, so the first history entries and logits are asked for together, before
// anything waits. Between the two the chain of each row and the rows left over in the last wave count:
// 256 rows of 32000 tokens with 2176 ids take 20.5 us, 22 with 32-bit counts.
//
// PER_SM: CTAs that the registers leave room for. Two where the grid fits so, three where it does not; with
// two and three: 256 x 32000 18.8 and 19.9 us (back to back), 318 x 15021 16.2 and 12.4, 2048 x 32000 106
// and 92, 300 x 128000 137 and 86.
//
// Four tokens per thread and step, starting at the row's first 16-byte boundary of the scores: rows of
// an odd vocabulary start anywhere, but logits and scores are off by the same number of tokens unless
// the caller's strides differ (then: token by token).
//
// Each CTA's best token goes into the shared memory of the cluster's first CTA, which alone waits.
template <typename T, typename I, bool WIDE, int PER_SM>
__global__ void __launch_bounds__(kLogitsThreads, PER_SM) logits_kernel(const __grid_constant__ LogitsParams p, int slice, int ctas) {
  using V4 = LogitsVec<T>;
  using Counts = LogitsCounts<WIDE>;
  constexpr int kLogitsCounts = Counts::N, kPer16 = WIDE ? 4 : 8;  // tokens; in 16 bytes
  extern __shared__ __align__(16) uint32_t cnt[];
  __shared__ float bv[kLogitsThreads / 32];
  __shared__ int bi[kLogitsThreads / 32];
  __shared__ unsigned long long theirs[8];  // of the cluster's first CTA: every CTA's best
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA exists
  pdl_wait();
  const T* x = (const T*)p.logits + b * p.ld;
  float* z = p.out + b * p.out_ld;
  const float* bias = p.bias ? p.bias + b * p.bias_ld : nullptr;
  const uint32_t* mask = p.mask ? p.mask + b * p.mask_ld : nullptr;
  const int phase = (int)(reinterpret_cast<uintptr_t>(z) >> 2 & 3), head = min((4 - phase) & 3, p.V);
  const bool vec = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) & 3) == phase;
  const bool bias_vec = bias && (int)(reinterpret_cast<uintptr_t>(bias) >> 2 & 3) == phase;
  const int beg = head + rank * slice, end = min(p.V, beg + slice);  // the first CTA takes [0, head) too
  const I* hist = (const I*)p.history + b * p.hist_ld;
  I ids[kLogitsIds];
#pragma unroll
  for (int k = 0; k < kLogitsIds; ++k) ids[k] = k * kLogitsThreads + tid < p.T ? __ldg(hist + k * kLogitsThreads + tid) : I(-1);
  // logits of the next kLogitsAhead vectors: the scores may overwrite the logits, so the compiler would
  // not move a load above the stores before it
  typename V4::Raw ahead[kLogitsAhead];
  auto ask = [&](int i0, int v0, int n) {
#pragma unroll
    for (int k = 0; k < kLogitsAhead; ++k) {
      const int i = i0 + (k * kLogitsThreads + tid) * 4;
      if (i + 4 <= n) ahead[k] = *reinterpret_cast<const typename V4::Raw*>(x + v0 + i);
    }
  };
  if (vec) ask(0, beg, min(kLogitsCounts, end - beg));
  const int start = p.starts ? p.starts[b] : 0;
  const float r = p.rep ? p.rep[b] : p.rep1, pr = p.pres ? p.pres[b] : p.pres1, f = p.freq ? p.freq[b] : p.freq1;
  float best = -INFINITY;
  int at = 0x7fffffff;
  auto penalise = [&](float v, uint32_t u) -> float {
    v = v > 0.f ? v / r : v * r;
    const uint32_t n = u & (Counts::kTop - 1);
    return n ? v - (f * (float)n + pr) : v;
  };
  auto one_token = [&](int v, uint32_t u) {
    float y = ld<T>(x + v);
    if (u) y = penalise(y, u);
    if (bias) y += bias[v];
    if (mask && !(mask[v >> 5] >> (v & 31) & 1)) y = -INFINITY;
    z[v] = y;
    if (y > best) {
      best = y;
      at = v;
    }
  };
  for (int v0 = beg; v0 < end || (v0 == beg && rank == 0); v0 += kLogitsCounts) {
    const int n = max(0, min(kLogitsCounts, end - v0)), lo = v0 == 0 + head ? -head : 0;  // counts of [v0 + lo, v0 + n)
    if (p.T) {
      if (v0 != beg) __syncthreads();
      for (int i = tid; i * kPer16 < n + 4; i += kLogitsThreads) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      auto count = [&](I x, int t) {
        const uint64_t id = (uint64_t)(int64_t)x - (uint64_t)(int64_t)(v0 + lo);
        if (id < (uint64_t)(n - lo)) Counts::add(cnt, 4 + lo + (int)id, t >= start);
      };
#pragma unroll
      for (int k = 0; k < kLogitsIds; ++k) count(ids[k], k * kLogitsThreads + tid);
#pragma unroll 4
      for (int t = kLogitsIds * kLogitsThreads + tid; t < p.T; t += kLogitsThreads) count(__ldg(hist + t), t);
      __syncthreads();
    }
    if (lo < 0 && tid < -lo) one_token(tid, p.T ? Counts::get(cnt, 4 + lo + tid) : 0u);
    if (vec) {
      constexpr int kStep = kLogitsAhead * kLogitsThreads * 4;
      for (int i0 = 0; i0 < n; i0 += kStep) {
        typename V4::Raw now[kLogitsAhead];
#pragma unroll
        for (int k = 0; k < kLogitsAhead; ++k) now[k] = ahead[k];
        if (i0 + kStep < n) ask(i0 + kStep, v0, n);
        else if (v0 + n < end) ask(0, v0 + n, min(kLogitsCounts, end - v0 - n));
#pragma unroll
        for (int k = 0; k < kLogitsAhead; ++k) {
          const int i = i0 + (k * kLogitsThreads + tid) * 4, v = v0 + i;
          if (i + 4 > n) {
            for (int e = i; e < n; ++e) one_token(v0 + e, p.T ? Counts::get(cnt, 4 + e) : 0u);
            continue;
          }
          float y[4];
          V4::open(now[k], y);
          if (p.T) {
            const uint4 u = Counts::get4(cnt, 4 + i);
            if (u.x | u.y | u.z | u.w) {
              if (u.x) y[0] = penalise(y[0], u.x);
              if (u.y) y[1] = penalise(y[1], u.y);
              if (u.z) y[2] = penalise(y[2], u.z);
              if (u.w) y[3] = penalise(y[3], u.w);
            }
          }
          if (bias_vec) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(bias + v));
            y[0] += a.x; y[1] += a.y; y[2] += a.z; y[3] += a.w;
          } else if (bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += __ldg(bias + v + e);
          }
          if (mask) {
            const int w = v >> 5;
            const uint32_t bits = __funnelshift_r(__ldg(mask + w), (v & 31) > 28 ? __ldg(mask + w + 1) : 0u, v & 31);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(bits >> e & 1)) y[e] = -INFINITY;
          }
          *reinterpret_cast<float4*>(z + v) = make_float4(y[0], y[1], y[2], y[3]);
          const float top = fmaxf(fmax3(y[0], y[1], y[2]), y[3]);
          if (top > best) {
            best = top;
            at = v + (y[0] == top ? 0 : y[1] == top ? 1 : y[2] == top ? 2 : 3);
          }
        }
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < n; i += kLogitsThreads) one_token(v0 + i, p.T ? Counts::get(cnt, 4 + i) : 0u);
    }
  }
  if (!p.best) {
    if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    return;
  }
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
  if (warp == 0) {
    best = lane < kLogitsThreads / 32 ? bv[lane] : -INFINITY;
    at = lane < kLogitsThreads / 32 ? bi[lane] : 0x7fffffff;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  }
  if (ctas > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA exists
    if (tid == 0) {
      uint32_t far;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(far) : "r"(smem_u32(theirs + rank)));
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(far), "l"((unsigned long long)__float_as_uint(best) << 32 | (uint32_t)at)
                   : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0)
      for (int k = 1; k < ctas; ++k) better(__uint_as_float((uint32_t)(theirs[k] >> 32)), (int)(uint32_t)theirs[k]);
  }
  if (tid == 0) p.best[b] = at == 0x7fffffff ? 0 : at;
}

}  // namespace one
