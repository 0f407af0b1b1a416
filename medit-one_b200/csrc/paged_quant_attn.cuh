// Attention of one new token per sequence over a paged cache held in 4 or 8 bits (paged_quant.cuh):
//   s_t = q . k_t * scale * log2(e)    o = sum_t 2^(s_t - m) v_t / l    mass_t += sum over heads 2^(s_t - m) / l
#pragma once

#include "paged_quant.cuh"

namespace one {

struct QuantAttnParams {
  PagedQuant m;
  const void* q;
  int64_t q_bs, q_hs;
  int G;
  float scale_log2;
  float* mass;
  int64_t mass_width;
  void* out;
  float* scores;
  int64_t score_ld;
};

// One CTA of four warps per (sequence, kv head), its query heads one after the other; a warp takes every
// fourth slot, a lane the dims lane + 32 g.
template <typename T, int BITS>
__global__ void __launch_bounds__(128) quant_attn_kernel(const __grid_constant__ QuantAttnParams p) {
  __shared__ float so[4][128], sm[4], sl[4];
  pdl_wait();
  const PagedCache& c = p.m.c;
  const int b = blockIdx.x / c.Hkv, h = blockIdx.x % c.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = paged_length(c, b, SITE_QUANT_ATTN), groups = p.m.groups;
  auto value = [&](const uint8_t* codes, int d) {
    return (float)((BITS == 4 ? codes[d >> 1] >> (d & 1) * 4 & 15 : codes[d]) - QuantCode<BITS>::kZero);
  };
  for (int g = 0; g < p.G; ++g) {
    const int64_t hq = ((int64_t)b * c.Hkv + h) * p.G + g;
    const T* q = (const T*)p.q + b * p.q_bs + (int64_t)(h * p.G + g) * p.q_hs;
    float* scores = p.scores ? p.scores + hq * p.score_ld : nullptr;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < groups; ++i)
      if (i * 32 + lane < c.Dh) x[i] = ld<T>(q + i * 32 + lane);
    for (int t = warp; t < len; t += 4) {
      const int index = t / c.page_size, page = paged_page(c, c.table, b * c.table_stride, index, SITE_QUANT_ATTN);
      if (page < 0) {
        if (scores && lane == 0) scores[t] = -INFINITY;
        continue;
      }
      const int64_t r = (int64_t)h * c.page_size + t - index * c.page_size;
      const uint8_t* kc = (const uint8_t*)c.k + page * c.k_stride + r * p.m.row;
      const uint8_t* vc = (const uint8_t*)c.v + page * c.v_stride + r * p.m.row;
      const __nv_bfloat16* sc = (const __nv_bfloat16*)p.m.scales + page * p.m.s_stride + r * 2 * groups;
      float s = 0.f;
      for (int i = 0; i < groups; ++i)
        if (i * 32 + lane < c.Dh) s += x[i] * value(kc, i * 32 + lane) * __bfloat162float(sc[i]);
      s = warp_sum(s) * p.scale_log2;
      if (scores && lane == 0) scores[t] = s;
      const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.f : mn, a = exp2f(m - ms), w = exp2f(s - ms);
      m = mn;
      l = l * a + w;
      for (int i = 0; i < groups; ++i)
        if (i * 32 + lane < c.Dh) o[i] = o[i] * a + w * (value(vc, i * 32 + lane) * __bfloat162float(sc[groups + i]));
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    for (int i = 0; i < 4; ++i) so[warp][i * 32 + lane] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, y = 0.f;
    for (int k = 0; k < 4; ++k) {
      const float f = exp2f(sm[k] - Ms);
      L += f * sl[k];
      y += f * so[k][threadIdx.x];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if ((int)threadIdx.x < c.Dh) st<T>((T*)p.out + hq * c.Dh + threadIdx.x, y * inv);
    if (p.mass)
      for (int t = threadIdx.x; t < len; t += 128) p.mass[((int64_t)b * c.Hkv + h) * p.mass_width + t] += exp2f(scores[t] - Ms) * inv;
    __syncthreads();
  }
}

}  // namespace one
