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

// Where token t of sequence b goes in head h of `pages` (stride: elements per page), or null. A slot
// beyond the table and a page outside the pool are recorded.
template <typename T>
ONE_DEVINL T* append_row(const PagedAppendParams& p, void* pages, int64_t stride, int b, int h, int t, int64_t& slot) {
  const PagedCache& c = p.c;
  if (p.counts && t >= p.counts[b]) return nullptr;
  const int len = c.lengths[b];
  slot = (int64_t)len + t;
  if (len < 0 || slot >= (int64_t)c.max_pages * c.page_size) {
    set_err(c.err, ERR_BAD_ARG, SITE_PAGED_APPEND);
    return nullptr;
  }
  const int index = (int)slot / c.page_size;
  const int pg = paged_page(c, c.table, b * c.table_stride, index, SITE_PAGED_APPEND);
  if (pg < 0) return nullptr;
  return (T*)pages + pg * stride + ((int64_t)h * c.page_size + ((int)slot - index * c.page_size)) * c.Dh;
}

// New tokens into the pages, rotated: y = x cos + rotate_half(x) sin. A copy with two products per
// element, bound by HBM (prompts) or by one round trip to it (single tokens).
//
// One thread per 8 elements of a row's first half and the matching 8 of its second, so the rotation
// needs no exchange; the threads of a token's heads are neighbours and share its cos and sin in L1.
// For rows whose halves are whole 16-byte pieces (Dh a multiple of 16, aligned strides);
// paged_append_any_kernel takes the rest. Sequence blockIdx.y.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int units = c.Dh / 16, heads = 2 * c.Hkv + (p.q ? p.Hq : 0), half = c.Dh / 2, b = blockIdx.y;
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t row = i / units;
  const int e = (int)(i - row * units) * 8, t = (int)(row / heads), hh = (int)(row - (uint32_t)t * heads);
  if (t >= p.N) return;
  const bool is_q = hh >= 2 * c.Hkv, is_v = !is_q && hh >= c.Hkv;
  const int h = is_q ? hh - 2 * c.Hkv : is_v ? hh - c.Hkv : hh;
  const T* x;
  if (is_q) x = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
  else if (is_v) x = (const T*)p.v + b * p.vs[0] + h * p.vs[1] + t * p.vs[2];
  else x = (const T*)p.k + b * p.ks[0] + h * p.ks[1] + t * p.ks[2];
  float x1[8], x2[8];
  load8(x + e, x1);
  load8(x + half + e, x2);
  T* y;
  if (is_q) {
    y = (T*)p.q_out + (((int64_t)b * p.Hq + h) * p.N + t) * c.Dh;
  } else {
    int64_t slot;
    y = append_row<T>(p, is_v ? c.v : c.k, is_v ? c.v_stride : c.k_stride, b, h, t, slot);
    if (!y) return;
    if (!is_v && p.mass && e == 0) p.mass[((int64_t)b * c.Hkv + h) * p.mass_width + slot] = 0.f;
  }
  if (p.cosv && !is_v) {
    const int64_t cs = b * p.cos_bs + (int64_t)t * c.Dh + e;
    float c1[8], c2[8], s1[8], s2[8];
    load8((const T*)p.cosv + cs, c1);
    load8((const T*)p.cosv + cs + half, c2);
    load8((const T*)p.sinv + cs, s1);
    load8((const T*)p.sinv + cs + half, s2);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float a = x1[k], o = x2[k];
      x1[k] = a * c1[k] - o * s1[k];
      x2[k] = o * c2[k] + a * s2[k];
    }
  }
  store8(y + e, x1);
  store8(y + half + e, x2);
}

// The same for rows of any alignment: one warp per row of q, k or v.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_any_kernel(const __grid_constant__ PagedAppendParams p) {
  pdl_wait();
  const PagedCache& c = p.c;
  const int lane = threadIdx.x & 31, half = c.Dh / 2, heads = 2 * c.Hkv + (p.q ? p.Hq : 0), b = blockIdx.y;
  const uint32_t row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int t = (int)(row / heads), hh = (int)(row - (uint32_t)t * heads);
  if (t >= p.N) return;
  const bool is_q = hh >= 2 * c.Hkv, is_v = !is_q && hh >= c.Hkv;
  const int h = is_q ? hh - 2 * c.Hkv : is_v ? hh - c.Hkv : hh;
  const int64_t* s = is_q ? p.qs : is_v ? p.vs : p.ks;
  const T* x = (const T*)(is_q ? p.q : is_v ? p.v : p.k) + b * s[0] + h * s[1] + t * s[2];
  T* y;
  if (is_q) {
    y = (T*)p.q_out + (((int64_t)b * p.Hq + h) * p.N + t) * c.Dh;
  } else {
    int64_t slot;
    y = append_row<T>(p, is_v ? c.v : c.k, is_v ? c.v_stride : c.k_stride, b, h, t, slot);
    if (!y) return;
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

// Which slots survive: one CTA per (sequence, kv head) finds the smallest surviving key by radix
// selection (digits of 11, 11 and 10 bits, counted in shared memory), then writes the surviving slots
// in order: every warp counts its run of slots, and the counts before it say where its survivors go.
// Keys are read from HBM once and kept in shared memory up to `cached` of them; longer sequences are
// read again in each of the five passes. Bound by the passes over shared memory, not by HBM.
constexpr int kSelThreads = 1024;
constexpr int kSelCached = 48 * 1024;

__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const __grid_constant__ PagedEvictParams p, int cached) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[2048];
  __shared__ int wsum[2][32];
  __shared__ uint32_t sh_digit;
  __shared__ int sh_above;
  pdl_wait();
  pdl_launch_dependents();
  const PagedCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t bh = blockIdx.x;
  const int n = paged_length(c, (int)(bh / c.Hkv), SITE_PAGED_EVICT);
  int* kept = p.kept + bh * p.budget;
  if (n <= p.budget) {
    for (int t = tid; t < p.budget; t += kSelThreads) kept[t] = t < n ? t : -1;
    return;
  }
  const float* mass = p.mass + bh * p.mass_width + p.sink;
  const int nc = n - p.sink - p.recent, places = p.budget - p.sink - p.recent;  // candidates, and room for them
  for (int t = tid; t < p.sink; t += kSelThreads) kept[t] = t;
  for (int t = tid; t < p.recent; t += kSelThreads) kept[p.budget - p.recent + t] = n - p.recent + t;
  if (places == 0) return;
  const bool in_smem = nc <= cached;
  uint32_t prefix = 0, mask = 0;
  int above = 0;  // candidates above the prefix
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < nc; i += kSelThreads) {
      const uint32_t k = pass > 0 && in_smem ? keys[i] : mass_key(mass[i]);
      if (pass == 0 && in_smem) keys[i] = k;
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread t holds digits 2047 - 2 t and 2046 - 2 t; sums from the top
    const int d0 = 2047 - 2 * tid, h0 = (int)hist[d0], h1 = (int)hist[d0 - 1];
    int incl = h0 + h1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) wsum[0][warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int v = wsum[0][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
      }
      wsum[0][lane] = v;
    }
    __syncthreads();
    const int before = above + (warp ? wsum[0][warp - 1] : 0) + incl - h0 - h1;
    if (before < places && before + h0 + h1 >= places) {
      const bool first = before + h0 >= places;
      sh_digit = (uint32_t)(first ? d0 : d0 - 1);
      sh_above = first ? before : before + h0;
    }
    __syncthreads();
    prefix |= sh_digit << shift;
    mask |= ((1u << bits) - 1) << shift;
    above = sh_above;
    __syncthreads();
  }
  // survivors: keys above `prefix`, and the first `ties` that equal it
  const int ties = places - above;
  const int run = ((nc + 31) / 32 + 31) / 32 * 32, i0 = warp * run, i1 = min(nc, i0 + run);
  int gt = 0, eq = 0;
  for (int i = i0; i < i1; i += 32) {
    const uint32_t k = i + lane < i1 ? (in_smem ? keys[i + lane] : mass_key(mass[i + lane])) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && k > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, i + lane < i1 && k == prefix));
  }
  if (lane == 0) {
    wsum[0][warp] = gt;
    wsum[1][warp] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < warp; ++w) {
    gt += wsum[0][w];
    eq += wsum[1][w];
  }
  const uint32_t below = (1u << lane) - 1;
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? (in_smem ? keys[i + lane] : mass_key(mass[i + lane])) : 0u;
    const unsigned bg = __ballot_sync(0xffffffffu, in && k > prefix), be = __ballot_sync(0xffffffffu, in && k == prefix);
    const int myeq = eq + __popc(be & below), at = gt + __popc(bg & below) + min(myeq, ties);
    if (in && (k > prefix || (k == prefix && myeq < ties))) kept[p.sink + at] = p.sink + i + lane;
    gt += __popc(bg);
    eq += __popc(be);
  }
}

// The survivors' rows and masses to their places, 64 places of one (sequence, kv head) per CTA: the
// rows' addresses first, then 16 bytes per thread and copy. A gather, bound by HBM.
constexpr int kMovePlaces = 64;

__global__ void __launch_bounds__(256) paged_move_kernel(const __grid_constant__ PagedEvictParams p, int per_bh, int pieces) {
  __shared__ int64_t from[2][kMovePlaces], to[2][kMovePlaces];  // 16-byte units; -1: nothing to copy
  pdl_wait();
  const PagedCache& c = p.c;
  const int tid = threadIdx.x;
  const int64_t bh = blockIdx.x / per_bh;
  const int i0 = (int)(blockIdx.x % per_bh) * kMovePlaces, b = (int)(bh / c.Hkv), h = (int)(bh % c.Hkv);
  const int64_t i = (int64_t)i0 + tid;
  if (tid < kMovePlaces) {
    const int src = i < p.budget ? p.kept[bh * p.budget + i] : -1;
    int ps = -1, pd = -1;
    if (src >= 0) {
      ps = paged_page(c, c.table, b * c.table_stride, src / c.page_size, SITE_PAGED_EVICT);
      pd = paged_page(c, p.dst, b * p.dst_stride, (int)i / c.page_size, SITE_PAGED_EVICT);
    }
    const bool there = ps >= 0 && pd >= 0;
    const int64_t row = (int64_t)c.Dh, per16 = row / pieces;  // elements of a row; of 16 bytes
    const int64_t so = ((int64_t)h * c.page_size + src % c.page_size) * row;
    const int64_t dt = ((int64_t)h * c.page_size + (int)i % c.page_size) * row;
    from[0][tid] = there ? (ps * c.k_stride + so) / per16 : -1;
    from[1][tid] = there ? (ps * c.v_stride + so) / per16 : -1;
    to[0][tid] = there ? (pd * c.k_stride + dt) / per16 : -1;
    to[1][tid] = there ? (pd * c.v_stride + dt) / per16 : -1;
    if (i < p.out_width) p.mass_out[bh * p.out_width + i] = src < 0 ? 0.f : p.mass[bh * p.mass_width + src];
  }
  __syncthreads();
  if (i0 >= p.budget) return;
  uint4* kp = (uint4*)c.k;
  uint4* vp = (uint4*)c.v;
  for (int e = tid; e < kMovePlaces * pieces; e += blockDim.x) {
    const int place = e / pieces, piece = e - place * pieces;
    if (from[0][place] < 0) continue;
    const uint4 a = kp[from[0][place] + piece], v = vp[from[1][place] + piece];
    kp[to[0][place] + piece] = a;
    vp[to[1][place] + piece] = v;
  }
}

}  // namespace one
