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

enum : int {
  SITE_PAGED_ATTN = 41, SITE_PAGED_APPEND = 42, SITE_PAGED_EVICT = 43,
  SITE_QUANT_APPEND = 44, SITE_QUANT_READ = 45, SITE_QUANT_ATTN = 46, SITE_QUANT_EVICT = 47
};

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
  const void *cosv, *sinv;      // [cos_batch][N][Dh] or null, in the cache's type or fp32
  int64_t cos_bs;
  const int* counts;
  float* mass;
  int64_t mass_width;
  void* q_out;  // [B][Hq][N][Dh]
  int N, Hq;
};

// The page and the row in it (head 0) of token t of sequence b; false: the token is not stored. A slot
// beyond the table and a page outside the pool are recorded.
ONE_DEVINL bool append_place(const PagedAppendParams& p, int b, int t, int64_t& slot, int& page, int& row,
                             int site = SITE_PAGED_APPEND) {
  const PagedCache& c = p.c;
  if (p.counts && t >= p.counts[b]) return false;
  const int len = c.lengths[b];
  slot = (int64_t)len + t;
  if (len < 0 || slot >= (int64_t)c.max_pages * c.page_size) {
    set_err(c.err, ERR_BAD_ARG, site);
    return false;
  }
  const int index = (int)slot / c.page_size;
  page = paged_page(c, c.table, b * c.table_stride, index, site);
  row = (int)slot - index * c.page_size;
  return page >= 0;
}

// 16 bytes of elements <-> pairs of floats
template <typename T> struct Piece;
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  ONE_DEVINL static void open(const uint4& u, float2 (&v)[4]) {
    v[0] = make_float2(bf2_lo(u.x), bf2_hi(u.x)); v[1] = make_float2(bf2_lo(u.y), bf2_hi(u.y));
    v[2] = make_float2(bf2_lo(u.z), bf2_hi(u.z)); v[3] = make_float2(bf2_lo(u.w), bf2_hi(u.w));
  }
  ONE_DEVINL static uint4 close(const float2 (&v)[4]) {
    return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y),
                      pack_bf16x2(v[3].x, v[3].y));
  }
};
template <> struct Piece<float> {
  static constexpr int N = 4;
  ONE_DEVINL static void open(const uint4& u, float2 (&v)[2]) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  ONE_DEVINL static uint4 close(const float2 (&v)[2]) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
// cos or sin, of type C, of a piece of T
template <typename T, typename C>
ONE_DEVINL void open_table(const C* at, float2 (&v)[Piece<T>::N / 2]) {
  constexpr int N = Piece<C>::N / 2;  // pairs per load
#pragma unroll
  for (int i = 0; i < Piece<T>::N / 2; i += N)
    Piece<C>::open(__ldg(reinterpret_cast<const uint4*>(at + 2 * i)), *reinterpret_cast<float2(*)[N]>(v + i));
}
ONE_DEVINL float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_from(d);
}

// New tokens into the pages, rotated: y = x cos + rotate_half(x) sin, in fp32 with one rounding; C is the
// type of cos and sin, that of the tokens or fp32. A copy with two products per element, bound by HBM
// (prompts) or by one round trip to it (single tokens).
//
// One thread per token, group of kAppendRows heads of its keys, queries or values, and 16-byte piece:
// consecutive lanes read and write whole rows, the group's loads are in flight together and share cos
// and sin. The piece half a row away, which the rotation needs, comes from its lane (PAIR false: rows of
// a power of two of pieces), or the thread has both (PAIR: halves of whole pieces).
// paged_append_any_kernel takes the rest. Sequence blockIdx.y.
//
// 8 prompts of up to 4096 tokens, 12 heads x 64: 68 us with one row per thread, 72 with pairs, 54 as here,
// 51 with five CTAs per SM (73 % of the copy rate; two thirds of the issue slots are taken, and what the
// warps wait for most is loads: cos and sin are asked for only when the page is known); without rotation it
// runs at the rate of a plain copy. 170 x 4 tokens of 367 heads x 80: 100 us one element at a time, 35 by
// halves.
constexpr int kAppendRows = 4;

template <typename T, typename C, bool PAIR>
__global__ void __launch_bounds__(256, PAIR ? 3 : 5) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  using P = Piece<T>;
  pdl_wait();
  const PagedCache& c = p.c;
  const int pieces = c.Dh / P::N, units = PAIR ? pieces / 2 : pieces, half = PAIR ? c.Dh / 2 : 0, hq = p.q ? p.Hq : 0, b = blockIdx.y;
  const int kvg = (c.Hkv + kAppendRows - 1) / kAppendRows, qg = (hq + kAppendRows - 1) / kAppendRows, groups = 2 * kvg + qg;
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x, item = i / units;
  const int piece = (int)(i - item * units), e = piece * P::N, t = (int)(item / groups);
  int g = (int)(item - (uint32_t)t * groups);
  if (t >= p.N) return;  // whole rows of lanes
  const T* from;
  int64_t step;
  int heads = c.Hkv, kind = 0;  // keys, queries, values
  if (g < kvg) {
    from = (const T*)p.k + b * p.ks[0] + t * p.ks[2];
    step = p.ks[1];
  } else if (g < kvg + qg) {
    g -= kvg;
    kind = 1;
    heads = hq;
    from = (const T*)p.q + b * p.qs[0] + t * p.qs[2];
    step = p.qs[1];
  } else {
    g -= kvg + qg;
    kind = 2;
    from = (const T*)p.v + b * p.vs[0] + t * p.vs[2];
    step = p.vs[1];
  }
  const int r0 = g * kAppendRows, rows = min(kAppendRows, heads - r0);
  from += r0 * step + e;
  uint4 x[kAppendRows], o[PAIR ? kAppendRows : 1];  // the other piece of a pair
#pragma unroll
  for (int k = 0; k < kAppendRows; ++k)
    if (k < rows) {
      x[k] = *reinterpret_cast<const uint4*>(from + k * step);
      if (PAIR) o[PAIR ? k : 0] = *reinterpret_cast<const uint4*>(from + k * step + half);
    }
  T* y;
  int64_t ystep;
  if (kind == 1) {
    y = (T*)p.q_out + (((int64_t)b * hq + r0) * p.N + t) * c.Dh + e;
    ystep = (int64_t)p.N * c.Dh;
  } else {
    int64_t slot;
    int page, row;
    if (!append_place(p, b, t, slot, page, row)) return;
    y = (kind ? (T*)c.v + page * c.v_stride : (T*)c.k + page * c.k_stride) + (r0 * c.page_size + row) * c.Dh + e;
    ystep = c.page_size * c.Dh;
    if (kind == 0 && p.mass)
      for (int k = piece; k < rows; k += units) p.mass[((int64_t)b * c.Hkv + r0 + k) * p.mass_width + slot] = 0.f;
  }
  if (kind < 2 && p.cosv) {
    const int64_t at = b * p.cos_bs + (int64_t)t * c.Dh + e;
    float2 cs[P::N / 2], sn[P::N / 2], cs2[PAIR ? P::N / 2 : 1], sn2[PAIR ? P::N / 2 : 1];
    open_table<T>((const C*)p.cosv + at, cs);
    open_table<T>((const C*)p.sinv + at, sn);
    if constexpr (PAIR) {
      open_table<T>((const C*)p.cosv + at + half, cs2);
      open_table<T>((const C*)p.sinv + at + half, sn2);
    }
    if (PAIR || 2 * piece < pieces) {
#pragma unroll
      for (int d = 0; d < P::N / 2; ++d) sn[d] = make_float2(-sn[d].x, -sn[d].y);
    }
    // the lanes of this row take this branch together
    const uint32_t lanes = PAIR ? 0u : (0xffffffffu >> (32 - pieces)) << ((threadIdx.x & 31) & ~(pieces - 1));
#pragma unroll
    for (int k = 0; k < kAppendRows; ++k) {
      if (k >= rows) break;
      uint4 other;
      if (PAIR) {
        other = o[PAIR ? k : 0];
      } else {
        other.x = __shfl_xor_sync(lanes, x[k].x, pieces / 2);
        other.y = __shfl_xor_sync(lanes, x[k].y, pieces / 2);
        other.z = __shfl_xor_sync(lanes, x[k].z, pieces / 2);
        other.w = __shfl_xor_sync(lanes, x[k].w, pieces / 2);
      }
      float2 u[P::N / 2], w[P::N / 2], r[P::N / 2];
      P::open(x[k], u);
      P::open(other, w);
#pragma unroll
      for (int d = 0; d < P::N / 2; ++d) r[d] = fma2(u[d], cs[d], mul2(w[d], sn[d]));
      *reinterpret_cast<uint4*>(y + k * ystep) = P::close(r);
      if constexpr (PAIR) {
#pragma unroll
        for (int d = 0; d < P::N / 2; ++d) r[d] = fma2(w[d], cs2[d], mul2(u[d], sn2[d]));
        *reinterpret_cast<uint4*>(y + k * ystep + half) = P::close(r);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kAppendRows; ++k)
      if (k < rows) {
        *reinterpret_cast<uint4*>(y + k * ystep) = x[k];
        if (PAIR) *reinterpret_cast<uint4*>(y + k * ystep + half) = o[PAIR ? k : 0];
      }
  }
}

// The same for rows of any alignment: one warp per row of q, k or v.
template <typename T, typename C>
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
    int page, at;
    if (!append_place(p, b, t, slot, page, at)) return;
    y = (T*)(is_v ? c.v : c.k) + page * (is_v ? c.v_stride : c.k_stride) + (h * c.page_size + at) * c.Dh;
    if (!is_v && p.mass && lane == 0) p.mass[((int64_t)b * c.Hkv + h) * p.mass_width + slot] = 0.f;
  }
  const int64_t cs = b * p.cos_bs + (int64_t)t * c.Dh;
  for (int d = lane; d < c.Dh; d += 32) {
    float r = ld<T>(x + d);
    if (p.cosv && !is_v) {
      const float o = d < half ? -ld<T>(x + d + half) : ld<T>(x + d - half);
      r = r * ld<C>((const C*)p.cosv + cs + d) + o * ld<C>((const C*)p.sinv + cs + d);
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
  uint32_t* scales;  // of a quantised cache: `words` words per row, pages s_stride words apart
  int64_t s_stride;
  int words;
};

// Rank of a mass, larger first: order-preserving bits of the float, -0 as 0, NaN below all.
ONE_DEVINL uint32_t mass_key(float f) {
  if (isnan(f)) return 0u;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Eviction. A CTA finds which slots of a (sequence, kv head) survive:
//  - the smallest surviving key by radix selection (digits of 9, 12 and 11 bits, counted in shared
//    memory; the first, sign and exponent, in eight copies, since masses crowd in few exponents); then
//    the survivors' ranks, from counts of runs of 32 candidates.
// Bound by latency: one read of the masses and a dozen barriers.
// MOVE: each of `parts` CTAs selects for itself and copies a part of the survivors: the slots whose rank
// lies in it go into a list in shared memory, and their rows and masses to their places, kEvictAhead
// pairs of a thread's 16-byte pieces in flight together. One launch, for as many CTAs as the SMs hold at
// once (4 x 1040 slots to 1024, 12 heads x 64: 12.3 us in two launches, 10.3 in one; 16 x 8192 to 2048:
// 51 in two, 70 in one). Otherwise one CTA writes the survivors' list and paged_move_kernel copies.
// KPT > 0: a thread keeps the keys of candidates tid, tid + 512, .. in KPT registers, read together and
// before the length is known; the smallest KPT that holds the table, since every pass goes over all of them
// (200 x 16 heads of 4096 slots to 512: 251 us in all with 16, 218 with 8). KPT = 0, for tables of more than
// 32768 slots: the masses are read again in each pass (16 x 12 heads of 30000 to 2048: 102 us, 84 with 64).
// CTAs per SM as the keys' registers allow: 3 rather than 2 up to KPT = 8 (100 x 16 heads of 781 slots to
// 200, 80 dims: 74.6 -> 70.3 us), 2 rather than 1 up to 32 (16 x 12 heads of 16000 to 2048: 60 us; with 64
// keys and one CTA 78), although the 64 registers of two spill: 8 bytes with KPT = 32, and with MOVE 176
// (KPT = 32) and 48 (KPT = 16).
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictList = 512;  // places listed at a time, one per thread
constexpr int kEvictAhead = 4;

template <int N>
struct Int {
  static constexpr int value = N;
};

template <int KPT, bool MOVE, typename U = uint4>
__global__ void __launch_bounds__(kEvictThreads, KPT > 32 ? 1 : KPT && KPT <= 8 && !MOVE ? 3 : 2)
    paged_evict_kernel(const __grid_constant__ PagedEvictParams p, int parts, int pieces) {
  // digit counts [512][8], [4096], [2048]; the first part's room then holds the listed rows' addresses in
  // 16 bytes: [from, to][keys, values][places], from -1: nothing to copy
  __shared__ __align__(16) uint32_t hist[10240];
  static_assert(sizeof(int64_t) * 4 * kEvictList <= 4 * 4096, "addresses");
  int64_t* from = reinterpret_cast<int64_t*>(hist);
  int64_t* to = from + 2 * kEvictList;
  constexpr bool SCALES = sizeof(U) == 8;  // a cache in 4 or 8 bits: rows of 8-byte units, and scales
  constexpr int SITE = SCALES ? SITE_QUANT_EVICT : SITE_PAGED_EVICT;
  // the third part's: the listed rows' scales, in words
  int64_t* from_s = reinterpret_cast<int64_t*>(hist + 8192);
  static_assert(sizeof(int64_t) * 2 * kEvictList <= 4 * 2048, "addresses");
  __shared__ int wsum[kEvictWarps];
  __shared__ uint32_t sh_digit[3];
  __shared__ int sh_above[3];
  // the second part's: survivors above << 32 | equal of runs of candidates, then what is before each
  unsigned long long* runs = reinterpret_cast<unsigned long long*>(hist + 4096);
  static_assert(sizeof(unsigned long long) * (KPT + 1) * kEvictWarps <= 4 * 4096, "runs");
  __shared__ unsigned long long part_sum[kEvictWarps];
  __shared__ int list[kEvictList];
  pdl_wait();
  if (!MOVE) pdl_launch_dependents();
  const PagedCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t bh = blockIdx.x / parts;
  const int part = blockIdx.x % parts, b = (int)(bh / c.Hkv), h = (int)(bh % c.Hkv);
  const float* row_mass = p.mass + bh * p.mass_width;
  const int cap = c.max_pages * c.page_size, slots = max(1, cap - p.sink);
  const float* mass = row_mass + min(p.sink, cap - 1);  // a budget may exceed the table; then nothing is selected
  uint32_t key[KPT ? KPT : 1];
#pragma unroll
  for (int k = 0; k < KPT; ++k) key[k] = __float_as_uint(__ldg(mass + min(k * kEvictThreads + tid, slots - 1)));
  const int n = paged_length(c, b, SITE), all = min(n, p.budget);
  // this part's places; the last part also clears the masses behind the survivors
  const int per = (p.budget + parts - 1) / parts, beg = min(part * per, p.budget), end = min(beg + per, p.budget);
  int* kept = p.kept + bh * p.budget;
  float* mass_out = p.mass_out + bh * p.out_width;
  for (int i = max(beg, all) + tid; i < end; i += kEvictThreads) {
    kept[i] = -1;
    if (MOVE) mass_out[i] = 0.f;
  }
  if (MOVE && part == parts - 1)
    for (int64_t i = p.budget + tid; i < p.out_width; i += kEvictThreads) mass_out[i] = 0.f;
  if (beg >= all) return;
  const int nc = n - p.sink - p.recent, places = p.budget - p.sink - p.recent;  // candidates, and room for them
  const bool select = n > p.budget && places > 0;
  uint32_t prefix = 0;
  int above = 0;  // candidates above the prefix
  if (select) {
#pragma unroll
    for (int k = 0; k < KPT; ++k) key[k] = mass_key(__uint_as_float(key[k]));
    // f(key) for the thread's candidates
    auto each = [&](auto&& f) {
      if (KPT) {
#pragma unroll
        for (int k = 0; k < KPT; ++k)
          if (k * kEvictThreads + tid < nc) f(key[k]);
      } else {
#pragma unroll 4
        for (int i = tid; i < nc; i += kEvictThreads) f(mass_key(__ldg(mass + i)));
      }
    };
    for (int i = tid * 4; i < 10240; i += kEvictThreads * 4) *reinterpret_cast<uint4*>(hist + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t mask = 0;
    // one digit: PER of its values per thread, thread t from the top; COPIES counts of each, side by side
    auto pass = [&](auto which, uint32_t* hs, int shift, int bits, auto per, auto copies) {
      constexpr int P = decltype(which)::value, PER = decltype(per)::value, COPIES = decltype(copies)::value;
      const uint32_t digits = (1u << bits) - 1;
      each([&](uint32_t k) {
        if ((k & mask) == prefix) atomicAdd(hs + (k >> shift & digits) * COPIES + (COPIES > 1 ? lane % COPIES : 0), 1u);
      });
      __syncthreads();
      const int d0 = (int)digits - PER * tid;
      int at[PER], sum = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        at[k] = 0;
#pragma unroll
        for (int j = 0; j < COPIES; ++j) at[k] += (int)hs[(d0 - k) * COPIES + j];
        sum += at[k];
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      if (lane == 31) wsum[warp] = incl;
      __syncthreads();
      int w = lane < warp ? wsum[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      int before = above + w + incl - sum;
      if (before < places && before + sum >= places) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          if (before < places && before + at[k] >= places) {
            sh_digit[P] = (uint32_t)(d0 - k);
            sh_above[P] = before;
          }
          before += at[k];
        }
      }
      __syncthreads();
      prefix |= sh_digit[P] << shift;
      mask |= digits << shift;
      above = sh_above[P];
    };
    pass(Int<0>{}, hist, 23, 9, Int<1>{}, Int<8>{});
    pass(Int<1>{}, hist + 4096, 11, 12, Int<8>{}, Int<1>{});
    pass(Int<2>{}, hist + 8192, 0, 11, Int<4>{}, Int<1>{});
  }
  // survivors: keys above `prefix`, and the first `ties` that equal it. Runs of 32 candidates (KPT) or a
  // warp's share of them all are counted, and the counts before each summed.
  const int ties = places - above;
  const uint32_t below = (1u << lane) - 1;
  const int run = ((nc + kEvictWarps - 1) / kEvictWarps + 31) / 32 * 32, i0 = warp * run, i1 = min(nc, i0 + run);  // KPT = 0
  if (select) {
    if (KPT) {
#pragma unroll
      for (int k = 0; k < KPT; ++k) {
        const bool in = k * kEvictThreads + tid < nc;
        const unsigned bg = __ballot_sync(0xffffffffu, in && key[k] > prefix), be = __ballot_sync(0xffffffffu, in && key[k] == prefix);
        if (lane == 0) runs[k * kEvictWarps + warp] = (unsigned long long)__popc(bg) << 32 | __popc(be);
      }
    } else {
      int gt = 0, eq = 0;
      for (int i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const uint32_t k = in ? mass_key(__ldg(mass + i + lane)) : 0u;
        gt += __popc(__ballot_sync(0xffffffffu, in && k > prefix));
        eq += __popc(__ballot_sync(0xffffffffu, in && k == prefix));
      }
      if (lane == 0) runs[warp] = (unsigned long long)gt << 32 | (uint32_t)eq;
    }
    __syncthreads();
    constexpr int kRuns = KPT ? KPT * kEvictWarps : kEvictWarps, kPer = (kRuns + kEvictThreads - 1) / kEvictThreads;
    unsigned long long v[kPer], sum = 0, incl;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      v[k] = tid * kPer + k < kRuns ? runs[tid * kPer + k] : 0ull;
      sum += v[k];
    }
    incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) part_sum[warp] = incl;
    __syncthreads();
    unsigned long long w = lane < warp ? part_sum[lane] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    w += incl - sum;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (tid * kPer + k < kRuns) runs[tid * kPer + k] = w;
      w += v[k];
    }
  }
  U* kp = (U*)c.k;
  U* vp = (U*)c.v;
  const int unit = SCALES ? sizeof(U) : c.Dh / pieces, head = h * c.page_size;  // elements of a unit; the head's first row in a page
  const int64_t ks = c.k_stride / unit, vs = c.v_stride / unit;
  const int step = MOVE ? kEvictList : p.budget;
  for (int lo = beg; lo < min(end, all); lo += step) {
    const int hi = MOVE ? min(lo + step, min(end, all)) : all;
    int* to_list = MOVE ? list : kept;
    __syncthreads();
    // list the survivors of places [lo, hi)
    auto put = [&](int place, int slot) {
      if (place >= lo && place < hi) to_list[place - lo] = slot;
    };
    if (!select) {  // all of them, or the first and the last ones alone
      for (int i = lo + tid; i < hi; i += kEvictThreads) to_list[i - lo] = n <= p.budget || i < p.sink ? i : n - p.budget + i;
    } else {
      for (int i = tid; i < p.sink; i += kEvictThreads) put(i, i);
      for (int i = tid; i < p.recent; i += kEvictThreads) put(p.budget - p.recent + i, n - p.recent + i);
      auto candidate = [&](bool in, uint32_t k, int i, int gt, int eq, unsigned bg, unsigned be) {
        const int mine = eq + __popc(be & below);
        if (in && (k > prefix || (k == prefix && mine < ties))) put(p.sink + gt + __popc(bg & below) + min(mine, ties), p.sink + i);
      };
      if (KPT) {
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
          const int i = k * kEvictThreads + tid;
          const bool in = i < nc;
          const unsigned bg = __ballot_sync(0xffffffffu, in && key[k] > prefix), be = __ballot_sync(0xffffffffu, in && key[k] == prefix);
          const unsigned long long r = runs[k * kEvictWarps + warp];
          candidate(in, key[k], i, (int)(r >> 32), (int)(uint32_t)r, bg, be);
        }
      } else {
        int gt = (int)(runs[warp] >> 32), eq = (int)(uint32_t)runs[warp];
        for (int i = i0; i < i1; i += 32) {
          const bool in = i + lane < i1;
          const uint32_t k = in ? mass_key(__ldg(mass + i + lane)) : 0u;
          const unsigned bg = __ballot_sync(0xffffffffu, in && k > prefix), be = __ballot_sync(0xffffffffu, in && k == prefix);
          candidate(in, k, i + lane, gt, eq, bg, be);
          gt += __popc(bg);
          eq += __popc(be);
        }
      }
    }
    if (!MOVE) return;
    __syncthreads();
    static_assert(kEvictList == kEvictThreads, "one place per thread");
    if (tid < hi - lo) {
      const int i = lo + tid, src = list[tid], si = src / c.page_size, di = i / c.page_size;
      kept[i] = src;
      mass_out[i] = row_mass[src];
      const int ps = paged_page(c, c.table, b * c.table_stride, si, SITE);
      const int pd = paged_page(c, p.dst, b * p.dst_stride, di, SITE);
      const bool there = ps >= 0 && pd >= 0;
      const int64_t sr = (int64_t)(head + src - si * c.page_size) * pieces, dr = (int64_t)(head + i - di * c.page_size) * pieces;
      from[tid] = there ? ps * ks + sr : -1;
      from[kEvictList + tid] = there ? ps * vs + sr : -1;
      to[tid] = pd * ks + dr;
      to[kEvictList + tid] = pd * vs + dr;
      if (SCALES) {
        from_s[tid] = ps * p.s_stride + (int64_t)(head + src - si * c.page_size) * p.words;
        from_s[kEvictList + tid] = pd * p.s_stride + (int64_t)(head + i - di * c.page_size) * p.words;
      }
    }
    __syncthreads();
    if (SCALES)
      for (int e = tid; e < (hi - lo) * p.words; e += kEvictThreads) {
        const int place = e / p.words, w = e - place * p.words;
        if (from[place] >= 0) p.scales[from_s[kEvictList + place] + w] = p.scales[from_s[place] + w];
      }
    const int count = (hi - lo) * pieces;
    for (int e0 = tid; e0 < count; e0 += kEvictAhead * kEvictThreads) {
      U a[kEvictAhead], v[kEvictAhead];
      int place[kEvictAhead];
#pragma unroll
      for (int k = 0; k < kEvictAhead; ++k) {
        const int e = e0 + k * kEvictThreads;
        place[k] = e < count ? e / pieces : -1;
        if (place[k] < 0 || from[place[k]] < 0) {
          place[k] = -1;
          continue;
        }
        a[k] = kp[from[place[k]] + (e - place[k] * pieces)];
        v[k] = vp[from[kEvictList + place[k]] + (e - place[k] * pieces)];
      }
#pragma unroll
      for (int k = 0; k < kEvictAhead; ++k) {
        if (place[k] < 0) continue;
        const int piece = e0 + k * kEvictThreads - place[k] * pieces;
        kp[to[place[k]] + piece] = a[k];
        vp[to[kEvictList + place[k]] + piece] = v[k];
      }
    }
  }
}

// The survivors' rows and masses to their places, 64 places of one (sequence, kv head) per CTA: the
// rows' addresses first, then 16 bytes per copy, kMoveAhead pairs of a thread's in flight together. A
// gather, bound by HBM.
constexpr int kMovePlaces = 64;
constexpr int kMoveAhead = 4;
constexpr int kMoveThreads = 128;

template <typename U = uint4>
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const __grid_constant__ PagedEvictParams p, int per_bh, int pieces) {
  constexpr bool SCALES = sizeof(U) == 8;
  constexpr int SITE = SCALES ? SITE_QUANT_EVICT : SITE_PAGED_EVICT;
  __shared__ int64_t from[2][kMovePlaces], to[2][kMovePlaces];  // units of U; -1: nothing to copy
  __shared__ int64_t from_s[SCALES ? kMovePlaces : 1], to_s[SCALES ? kMovePlaces : 1];  // the rows' scales, in words
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
      ps = paged_page(c, c.table, b * c.table_stride, src / c.page_size, SITE);
      pd = paged_page(c, p.dst, b * p.dst_stride, (int)i / c.page_size, SITE);
    }
    const bool there = ps >= 0 && pd >= 0;
    const int64_t unit = SCALES ? sizeof(U) : c.Dh / pieces;  // elements of a unit
    const int64_t sr = (int64_t)h * c.page_size + src % c.page_size, dr = (int64_t)h * c.page_size + (int)i % c.page_size;
    from[0][tid] = there ? ps * c.k_stride / unit + sr * pieces : -1;
    from[1][tid] = there ? ps * c.v_stride / unit + sr * pieces : -1;
    to[0][tid] = there ? pd * c.k_stride / unit + dr * pieces : -1;
    to[1][tid] = there ? pd * c.v_stride / unit + dr * pieces : -1;
    if constexpr (SCALES) {
      from_s[tid] = there ? ps * p.s_stride + sr * p.words : -1;
      to_s[tid] = there ? pd * p.s_stride + dr * p.words : -1;
    }
    if (i < p.out_width) p.mass_out[bh * p.out_width + i] = src < 0 ? 0.f : p.mass[bh * p.mass_width + src];
  }
  __syncthreads();
  if (i0 >= p.budget) return;
  if constexpr (SCALES)
    for (int e = tid; e < kMovePlaces * p.words; e += blockDim.x) {
      const int place = e / p.words, w = e - place * p.words;
      if (from_s[place] >= 0) p.scales[to_s[place] + w] = p.scales[from_s[place] + w];
    }
  U* kp = (U*)c.k;
  U* vp = (U*)c.v;
  const int all = kMovePlaces * pieces;
  for (int e0 = tid; e0 < all; e0 += kMoveAhead * blockDim.x) {
    U a[kMoveAhead], v[kMoveAhead];
#pragma unroll
    for (int k = 0; k < kMoveAhead; ++k) {
      const int e = e0 + k * blockDim.x, place = e / pieces;
      if (e < all && from[0][place] >= 0) {
        a[k] = kp[from[0][place] + (e - place * pieces)];
        v[k] = vp[from[1][place] + (e - place * pieces)];
      }
    }
#pragma unroll
    for (int k = 0; k < kMoveAhead; ++k) {
      const int e = e0 + k * blockDim.x, place = e / pieces;
      if (e < all && from[0][place] >= 0) {
        kp[to[0][place] + (e - place * pieces)] = a[k];
        vp[to[1][place] + (e - place * pieces)] = v[k];
      }
    }
  }
}

}  // namespace one
