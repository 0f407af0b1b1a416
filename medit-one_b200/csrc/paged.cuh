// A paged key-value cache and the operators of one serving step over it.
//
//   pages        k_pages, v_pages [num_pages][Hkv][page_size][Dh], model dtype (the page stride may
//                be larger than Hkv * page_size * Dh)
//   block table  [B][max_pages] int32: the pages of each sequence in order; slot t of sequence b is
//                row t % page_size of page table[b][t / page_size]
//   lengths      [B] int32: slots in use
//
// Pages that a sequence does not use are not read. A page number outside [0, num_pages) where one
// is used, a negative length, and a length beyond the table are recorded (ERR_BAD_ARG); the rows
// they name are neither read nor written.
#pragma once

#include "common.cuh"

namespace one {

enum : int { SITE_PAGED_ATTN = 41, SITE_PAGED_APPEND = 42, SITE_PAGED_EVICT = 43 };

struct PagedCache {
  void* k;
  void* v;
  int64_t k_stride, v_stride;  // elements from one page to the next
  const int* table;
  int64_t table_stride;
  const int* lengths;
  int num_pages, page_size, max_pages, B, Hkv, Dh;
  DevErr* err;
};

ONE_DEVINL int paged_length(const PagedCache& c, int b, int site) {
  const int n = c.lengths[b], cap = c.max_pages * c.page_size;
  if (n < 0 || n > cap) set_err(c.err, ERR_BAD_ARG, site);
  return min(max(n, 0), cap);
}

// Page of slot t, or -1 (recorded) when the table names no page of the pool.
ONE_DEVINL int paged_page(const PagedCache& c, const int* table, int64_t row, int index, int site) {
  const int pg = table[row + index];
  if (pg < 0 || pg >= c.num_pages) {
    set_err(c.err, ERR_BAD_ARG, site);
    return -1;
  }
  return pg;
}

struct PagedAttnParams {
  PagedCache c;
  const void* q;
  int64_t q_bs, q_hs;
  int G;
  float scale_log2;
  float* mass;
  int64_t mass_width;
  void* out;  // [B][Hq][Dh]
};

// One CTA per (kv head, sequence): its query heads one after the other, every warp over its share
// of the slots with the online softmax (running maximum and sum in base 2).
template <typename T>
__global__ void __launch_bounds__(256) paged_attn_simple_kernel(const PagedAttnParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = blockDim.x >> 5;
  const int n = paged_length(c, b, SITE_PAGED_ATTN);
  __shared__ float sm_m[8], sm_l[8], sm_o[8][128];
  auto row = [&](int t) -> int64_t {
    const int pg = paged_page(c, c.table, b * c.table_stride, t / c.page_size, SITE_PAGED_ATTN);
    return pg < 0 ? -1 : ((int64_t)h * c.page_size + t % c.page_size) * c.Dh + pg * c.k_stride;
  };
  auto vrow = [&](int t) -> int64_t {
    const int pg = c.table[b * c.table_stride + t / c.page_size];
    return ((int64_t)h * c.page_size + t % c.page_size) * c.Dh + pg * c.v_stride;
  };
  for (int g = 0; g < p.G; ++g) {
    const int hq = h * p.G + g;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 32 * i;
      q[i] = d < c.Dh ? ld<T>((const T*)p.q + b * p.q_bs + hq * p.q_hs + d) * p.scale_log2 : 0.f;
    }
    auto score = [&](int64_t at) {
      float s = 0.f;
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 32 * i;
        if (d < c.Dh) s += q[i] * ld<T>((const T*)c.k + at + d);
      }
      return warp_sum(s);
    };
    float m = -INFINITY, l = 0.f;
    for (int t = warp; t < n; t += W) {
      const int64_t at = row(t);
      if (at < 0) continue;
      const float s = score(at), mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.f : mn;
      const float a = exp2f(m - ms), e = exp2f(s - ms);
      const int64_t va = vrow(t);
      l = l * a + e;
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 32 * i;
        if (d < c.Dh) o[i] = o[i] * a + e * ld<T>((const T*)c.v + va + d);
      }
      m = mn;
    }
    if (lane == 0) {
      sm_m[warp] = m;
      sm_l[warp] = l;
    }
    for (int i = 0; i < 4; ++i) sm_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm_m[w]);
    const float Ms = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < W; ++w) L += sm_l[w] * exp2f(sm_m[w] - Ms);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int d = threadIdx.x; d < c.Dh; d += blockDim.x) {
      float acc = 0.f;
      for (int w = 0; w < W; ++w) acc += sm_o[w][d] * exp2f(sm_m[w] - Ms);
      st<T>((T*)p.out + ((int64_t)b * c.Hkv * p.G + hq) * c.Dh + d, acc * inv);
    }
    if (p.mass) {
      for (int t = warp; t < n; t += W) {
        const int64_t at = row(t);
        if (at < 0) continue;
        const float s = score(at);
        if (lane == 0) p.mass[((int64_t)b * c.Hkv + h) * p.mass_width + t] += exp2f(s - Ms) * inv;
      }
    }
    __syncthreads();
  }
}

struct PagedAppendParams {
  PagedCache c;
  const void *k, *v, *q;
  int64_t ks[3], vs[3], qs[3];  // element strides: batch, head, token
  const void *cosv, *sinv;      // [cos_batch][N][Dh] or null
  int64_t cos_bs;
  const int* counts;
  float* mass;
  int64_t mass_width;
  void* q_out;  // [B][Hq][N][Dh]
  int N, Hq;
};

// One warp per row of q, k or v.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_simple_kernel(const PagedAppendParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 31, half = c.Dh / 2, heads = 2 * c.Hkv + (p.q ? p.Hq : 0);
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (i >= (int64_t)c.B * p.N * heads) return;
  const int hh = (int)(i % heads), t = (int)(i / heads % p.N), b = (int)(i / heads / p.N);
  const bool is_q = hh >= 2 * c.Hkv, is_v = !is_q && hh >= c.Hkv;
  const int h = is_q ? hh - 2 * c.Hkv : is_v ? hh - c.Hkv : hh;
  const int64_t* s = is_q ? p.qs : is_v ? p.vs : p.ks;
  const T* x = (const T*)(is_q ? p.q : is_v ? p.v : p.k) + b * s[0] + h * s[1] + t * s[2];
  T* y;
  if (is_q) {
    y = (T*)p.q_out + (((int64_t)b * p.Hq + h) * p.N + t) * c.Dh;
  } else {
    const int cnt = p.counts ? min(p.counts[b], p.N) : p.N;
    if (t >= cnt) return;
    const int64_t slot = (int64_t)c.lengths[b] + t;
    if (c.lengths[b] < 0 || slot >= (int64_t)c.max_pages * c.page_size) {
      set_err(c.err, ERR_BAD_ARG, SITE_PAGED_APPEND);
      return;
    }
    const int pg = paged_page(c, c.table, b * c.table_stride, (int)(slot / c.page_size), SITE_PAGED_APPEND);
    if (pg < 0) return;
    y = (T*)(is_v ? c.v : c.k) + pg * (is_v ? c.v_stride : c.k_stride) + ((int64_t)h * c.page_size + slot % c.page_size) * c.Dh;
    if (!is_v && p.mass && lane == 0) p.mass[((int64_t)b * c.Hkv + h) * p.mass_width + slot] = 0.f;
  }
  const int64_t cs = b * p.cos_bs + (int64_t)t * c.Dh;
  for (int d = lane; d < c.Dh; d += 32) {
    float r = ld<T>(x + d);
    if (p.cosv && !is_v) {
      const float o = d < half ? -ld<T>(x + d + half) : ld<T>(x + d - half);
      r = r * ld<T>((const T*)p.cosv + cs + d) + o * ld<T>((const T*)p.sinv + cs + d);
    }
    st<T>(y + d, r);
  }
}

struct PagedEvictParams {
  PagedCache c;
  const int* dst;
  int64_t dst_stride;
  const float* mass;
  int64_t mass_width;
  int budget, recent, sink;
  float* mass_out;
  int64_t out_width;
  int* kept;  // [B][Hkv][budget]
};

// Rank of a mass, larger first: order-preserving bits of the float, -0 as 0, NaN below all.
ONE_DEVINL uint32_t mass_key(float f) {
  if (isnan(f)) return 0u;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One CTA per (kv head, sequence): a slot survives when fewer than the free places rank before it.
__global__ void __launch_bounds__(256) paged_select_simple_kernel(const PagedEvictParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = paged_length(c, b, SITE_PAGED_EVICT);
  const float* mass = p.mass + ((int64_t)b * c.Hkv + h) * p.mass_width;
  int* kept = p.kept + ((int64_t)b * c.Hkv + h) * p.budget;
  __shared__ uint32_t sh_thr;
  __shared__ int sh_count, sh_at;
  const int lo = n > p.budget ? p.sink : 0, hi = n > p.budget ? n - p.recent : 0;  // slots that are ranked
  const int places = p.budget - p.sink - p.recent;
  // the smallest key that survives, bit by bit
  uint32_t thr = 0;
  for (int bit = 31; bit >= 0; --bit) {
    if (threadIdx.x == 0) sh_count = 0;
    __syncthreads();
    int mine = 0;
    for (int t = lo + threadIdx.x; t < hi; t += blockDim.x) mine += mass_key(mass[t]) >= (thr | 1u << bit);
    atomicAdd(&sh_count, mine);
    __syncthreads();
    if (sh_count >= places) thr |= 1u << bit;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    int above = 0, at = 0;
    for (int t = lo; t < hi; ++t) above += mass_key(mass[t]) > thr;
    int equal = places - above;
    for (int t = 0; t < n; ++t) {
      bool keep = t < lo || t >= hi;
      if (!keep) {
        const uint32_t k = mass_key(mass[t]);
        keep = k > thr || (k == thr && equal-- > 0);
      }
      if (keep) kept[at++] = t;
    }
    for (; at < p.budget; ++at) kept[at] = -1;
  }
}

// One warp per survivor's place.
template <typename T>
__global__ void __launch_bounds__(256) paged_move_simple_kernel(const PagedEvictParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 31, h = blockIdx.y % c.Hkv, b = blockIdx.y / c.Hkv;
  const int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (i >= p.out_width) return;
  const int64_t bh = (int64_t)b * c.Hkv + h;
  const int src = i < p.budget ? p.kept[bh * p.budget + i] : -1;
  if (lane == 0) p.mass_out[bh * p.out_width + i] = src < 0 ? 0.f : p.mass[bh * p.mass_width + src];
  if (src < 0) return;
  const int ps = paged_page(c, c.table, b * c.table_stride, src / c.page_size, SITE_PAGED_EVICT);
  const int pd = paged_page(c, p.dst, b * p.dst_stride, (int)(i / c.page_size), SITE_PAGED_EVICT);
  if (ps < 0 || pd < 0) return;
  const int64_t so = ((int64_t)h * c.page_size + src % c.page_size) * c.Dh;
  const int64_t to = ((int64_t)h * c.page_size + i % c.page_size) * c.Dh;
  for (int d = lane; d < c.Dh; d += 32) {
    ((T*)c.k)[pd * c.k_stride + to + d] = ((const T*)c.k)[ps * c.k_stride + so + d];
    ((T*)c.v)[pd * c.v_stride + to + d] = ((const T*)c.v)[ps * c.v_stride + so + d];
  }
}

}  // namespace one
