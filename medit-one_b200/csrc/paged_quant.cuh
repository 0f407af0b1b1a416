// A paged key-value cache held in 4 or 8 bits: quantising tokens into it and reading them back.
//
//   codes     k, v [num_pages][Hkv][page_size][Dh * bits / 8] bytes: 4 bits hold code + 8, the even dim in
//             the low half of a byte; 8 bits hold code + 128
//   scales    bf16 [num_pages][Hkv][page_size][2][groups]: of the keys, then of the values
//
// A row of Dh values is cut into groups of 32 (the last may be shorter) of scale * code:
//   scale = bf16(max |x| / m), m = 7 or 127       code = rint(x / scale)
// where x is the value in fp32. Codes do not depend on how the quotient is computed as long as it is
// rounded correctly: scale has 8 significant bits and x 24, so that x / scale, when it is no multiple
// of 1/2, is at least an ulp away from one. The same holds for max |x| / m and the bf16 rounding.
// Symmetric codes, so that a product with a code needs no second sum for an offset of its own; 32
// values to a scale, so that a large channel spoils few others, for half a bit per value.
#pragma once

#include "paged.cuh"

namespace one {

constexpr int kQuantGroup = 32;
constexpr float kQuantLeast = 7.888609052210118e-31f;  // 2^-100: smaller scales are held as 0

struct PagedQuant {
  PagedCache c;  // k, v: bytes, strides in bytes
  void* scales;
  int64_t s_stride;  // elements from one page to the next
  int row, groups;   // bytes of a row of codes; scales of a row
};

template <int BITS>
struct QuantCode {
  static constexpr float kTop = BITS == 4 ? 7.f : 127.f;
  static constexpr int kZero = BITS == 4 ? 8 : 128;
};

// The scale (as a float that bf16 holds), its reciprocal and whether codes count, from the bits of max |x|.
template <int BITS>
ONE_DEVINL void quant_scale(uint32_t largest, float& scale, float& inv) {
  const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__uint_as_float(largest), QuantCode<BITS>::kTop)));
  const bool finite = largest < 0x7f800000u, there = finite && s >= kQuantLeast;
  scale = there ? s : finite ? 0.f : __uint_as_float(0x7fc00000u);
  inv = there ? __frcp_rn(s) : 0.f;
}

// x cos + y sin in fp32 with one rounding: products of bf16 values are exact in fp32, those of fp32 in fp64.
ONE_DEVINL float quant_rotate(__nv_bfloat16, __nv_bfloat16, float x, float y, float cs, float sn) { return fmaf(x, cs, y * sn); }
template <typename T, typename C>
ONE_DEVINL float quant_rotate(T, C, float x, float y, float cs, float sn) {
  return (float)fma((double)x, (double)cs, (double)y * (double)sn);
}

struct QuantAppendParams {
  PagedAppendParams a;
  void* scales;
  int64_t s_stride;
  int row, groups;
};

// New tokens, one warp per row of q, k or v, any alignment; a lane holds dim 32 g + lane of group g.
template <typename T, typename C, int BITS>
__global__ void __launch_bounds__(256) quant_append_any_kernel(const __grid_constant__ QuantAppendParams p) {
  pdl_wait();
  const PagedAppendParams& a = p.a;
  const PagedCache& c = a.c;
  const int lane = threadIdx.x & 31, half = c.Dh / 2, heads = 2 * c.Hkv + (a.q ? a.Hq : 0), b = blockIdx.y;
  const uint32_t row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int t = (int)(row / heads), hh = (int)(row - (uint32_t)t * heads);
  if (t >= a.N) return;
  const bool is_q = hh >= 2 * c.Hkv, is_v = !is_q && hh >= c.Hkv;
  const int h = is_q ? hh - 2 * c.Hkv : is_v ? hh - c.Hkv : hh;
  const int64_t* s = is_q ? a.qs : is_v ? a.vs : a.ks;
  const T* x = (const T*)(is_q ? a.q : is_v ? a.v : a.k) + b * s[0] + h * s[1] + t * s[2];
  uint8_t* codes = nullptr;
  __nv_bfloat16* scales = nullptr;
  if (!is_q) {
    int64_t slot;
    int page, at;
    if (!append_place(a, b, t, slot, page, at, SITE_QUANT_APPEND)) return;
    codes = (uint8_t*)(is_v ? c.v : c.k) + page * (is_v ? c.v_stride : c.k_stride) + ((int64_t)h * c.page_size + at) * p.row;
    scales = (__nv_bfloat16*)p.scales + page * p.s_stride + (((int64_t)h * c.page_size + at) * 2 + is_v) * p.groups;
    if (!is_v && a.mass && lane == 0) a.mass[((int64_t)b * c.Hkv + h) * a.mass_width + slot] = 0.f;
  }
  const int64_t cs = b * a.cos_bs + (int64_t)t * c.Dh;
  for (int g = 0; g < p.groups; ++g) {
    const int d = g * kQuantGroup + lane;
    float r = 0.f;
    if (d < c.Dh) {
      r = ld<T>(x + d);
      if (a.cosv && !is_v) {
        const float o = d < half ? -ld<T>(x + d + half) : ld<T>(x + d - half);
        r = quant_rotate(T(), C(), r, o, ld<C>((const C*)a.cosv + cs + d), ld<C>((const C*)a.sinv + cs + d));
      }
      if (is_q) st<T>((T*)a.q_out + (((int64_t)b * a.Hq + h) * a.N + t) * c.Dh + d, r);
    }
    if (is_q) continue;
    float scale, inv;
    quant_scale<BITS>(__reduce_max_sync(0xffffffffu, __float_as_uint(r) & 0x7fffffffu), scale, inv);
    const int code = inv == 0.f ? 0 : __float2int_rn(__fdiv_rn(r, scale));
    const uint32_t u = (uint32_t)(code + QuantCode<BITS>::kZero);
    if (BITS == 4) {
      const uint32_t next = __shfl_down_sync(0xffffffffu, u, 1);
      if (d < c.Dh && !(lane & 1)) codes[d >> 1] = (uint8_t)(u | next << 4);
    } else if (d < c.Dh) {
      codes[d] = (uint8_t)u;
    }
    if (lane == 0) scales[g] = __float2bfloat16_rn(scale);
  }
}

struct QuantReadParams {
  PagedQuant m;
  const int* starts;  // or null: 0
  void *k, *v;        // [B][Hkv][N][Dh]
  int N;
};

// Slots starts[b] .. starts[b] + N - 1 of every sequence, those not below lengths[b] as zeros; a thread
// has 8 dims of a slot's key and value.
template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_read_kernel(const __grid_constant__ QuantReadParams p) {
  pdl_wait();
  const PagedCache& c = p.m.c;
  const int pieces = c.Dh / 8, b = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, row = i / pieces;
  if (row >= (int64_t)c.Hkv * p.N) return;
  const int piece = (int)(i - row * pieces), h = (int)(row / p.N), t = (int)(row - (int64_t)h * p.N);
  const int len = paged_length(c, b, SITE_QUANT_READ), first = p.starts ? p.starts[b] : 0;
  const int64_t slot = (int64_t)first + t;
  int page = -1, at = 0;
  if (first < 0) set_err(c.err, ERR_BAD_ARG, SITE_QUANT_READ);
  if (slot >= 0 && slot < len) {
    const int index = (int)slot / c.page_size;
    page = paged_page(c, c.table, b * c.table_stride, index, SITE_QUANT_READ);
    at = (int)slot - index * c.page_size;
  }
  T* to[2] = {(T*)p.k, (T*)p.v};
  const int64_t out = (((int64_t)b * c.Hkv + h) * p.N + t) * c.Dh + piece * 8;
  for (int w = 0; w < 2; ++w) {
    float x[8];
    if (page >= 0) {
      const int64_t r = (int64_t)h * c.page_size + at;
      const uint8_t* codes = (const uint8_t*)(w ? c.v : c.k) + page * (w ? c.v_stride : c.k_stride) + r * p.m.row + piece * BITS;
      const float s = __bfloat162float(((const __nv_bfloat16*)p.m.scales)[page * p.m.s_stride + (r * 2 + w) * p.m.groups + piece / 4]);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const int u = BITS == 4 ? codes[d >> 1] >> (d & 1) * 4 & 15 : codes[d];
        x[d] = s * (float)(u - QuantCode<BITS>::kZero);
      }
    } else {
#pragma unroll
      for (int d = 0; d < 8; ++d) x[d] = 0.f;
    }
    store8(to[w] + out, x);
  }
}

}  // namespace one
