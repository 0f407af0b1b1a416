// A paged key-value cache held in 4 or 8 bits: quantising tokens into it and reading them back.
//
//   codes     k, v [num_pages][Hkv][page_size][Dh * bits / 8] bytes: 4 bits hold code + 8, the even dim in
//             the low half of a byte; 8 bits hold code + 128
//   scales    bf16 [num_pages][Hkv][page_size][2][groups]: of the keys, then of the values
//
// A row of Dh values is cut into groups of 32 (the last may be shorter) of scale * code:
//   scale = bf16(max |x| / m), m = 7 or 127       code = rint(x / scale)
// where x is the value in fp32. Codes do not depend on how the quotient is computed as long as its error
// stays well below 2^-24: scale has at most 8 significant bits and x 24, so that (n + 1/2) scale is an fp32, x
// differs from it by an ulp or not at all, and x / scale from n + 1/2 by more than half an ulp (by 1 / 1.992
// of one; the rounding of a quotient off by 2^-40 is therefore the exact one's). The same holds for max |x| /
// m and the halfway points of bf16.
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

// The scale (as a float that bf16 holds) and about its reciprocal, 0 where codes do not count, from max |x|. The
// quotient is one by a rounded reciprocal with one residual (Markstein, IBM J. Res. Dev. 34(1), 1990).
template <int BITS>
ONE_DEVINL void quant_scale(float largest, float& scale, float& inv) {
  constexpr float m = QuantCode<BITS>::kTop, by = 1.f / m;
  const float q = largest * by;
  const float s = __bfloat162float(__float2bfloat16_rn(fmaf(fmaf(-q, m, largest), by, q)));
  const bool finite = largest < INFINITY, there = finite && s >= kQuantLeast;
  scale = there ? s : finite ? 0.f : __uint_as_float(0x7fc00000u);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));  // 2^-125 at least
  if (!there) inv = 0.f;
}
// max |.| of three, NaN if one is
ONE_DEVINL float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// x cos + y sin, rounded to fp32: products of bf16 values are exact in fp32, so that there is one rounding; those of
// fp32 in fp64, whose sum is rounded to fp64 first.
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
  int per, lane_m;  // rows of lanes per warp; lane / (Dh / 8) = lane * lane_m >> 10
};

// 8 values as codes, 4 (8) bits each, the first lowest. The quotient is x inv with one residual; adding 1.5 *
// 2^23 rounds it to a whole number, halves to even, in the low bits of the sum.
template <int BITS>
ONE_DEVINL void quant_codes(const float2 (&x)[4], float scale, float inv, uint32_t (&out)[BITS / 4]) {
  const float2 by = make_float2(inv, inv), minus = make_float2(-scale, -scale);
  const float magic = 12582912.f + QuantCode<BITS>::kZero;
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t = mul2(x[i], by);
    t = fma2(fma2(t, minus, x[i]), by, t);
    t = add2(t, make_float2(magic, magic));
    u[2 * i] = __float_as_uint(t.x);
    u[2 * i + 1] = __float_as_uint(t.y);
  }
  auto bytes = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  };
  constexpr uint32_t kNone = BITS == 4 ? 0x88888888u : 0x80808080u;
  if constexpr (BITS == 4) {
    out[0] = bytes(u[0] + 16 * u[1], u[2] + 16 * u[3], u[4] + 16 * u[5], u[6] + 16 * u[7]);
    if (inv == 0.f) out[0] = kNone;
  } else {
    out[0] = bytes(u[0], u[1], u[2], u[3]);
    out[1] = bytes(u[4], u[5], u[6], u[7]);
    if (inv == 0.f) out[0] = out[1] = kNone;
  }
}

// 8 values of T, 16-byte aligned
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
  uint4 u;
  ONE_DEVINL void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  ONE_DEVINL void ldg(const __nv_bfloat16* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  ONE_DEVINL void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
  ONE_DEVINL void open(float2 (&v)[4]) const { Piece<__nv_bfloat16>::open(u, v); }
  ONE_DEVINL void close(const float2 (&v)[4]) { u = Piece<__nv_bfloat16>::close(v); }
  ONE_DEVINL Eight from_lane(int lane) const {
    return {make_uint4(__shfl_sync(0xffffffffu, u.x, lane), __shfl_sync(0xffffffffu, u.y, lane), __shfl_sync(0xffffffffu, u.z, lane),
                       __shfl_sync(0xffffffffu, u.w, lane))};
  }
};
template <> struct Eight<float> {
  float4 a, b;
  ONE_DEVINL void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
  ONE_DEVINL void ldg(const float* p) { a = __ldg(reinterpret_cast<const float4*>(p)); b = __ldg(reinterpret_cast<const float4*>(p + 4)); }
  ONE_DEVINL void store(float* p) const { *reinterpret_cast<float4*>(p) = a; *reinterpret_cast<float4*>(p + 4) = b; }
  ONE_DEVINL void open(float2 (&v)[4]) const {
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
  }
  ONE_DEVINL void close(const float2 (&v)[4]) {
    a = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    b = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  }
  ONE_DEVINL Eight from_lane(int lane) const {
    auto s = [&](float x) { return __shfl_sync(0xffffffffu, x, lane); };
    return {make_float4(s(a.x), s(a.y), s(a.z), s(a.w)), make_float4(s(b.x), s(b.y), s(b.z), s(b.w))};
  }
};

// New tokens into the pages, rotated and quantised: a copy of 2 or 4 bytes per value in and a half or one
// out, with some eight instructions per value in between; bound by HBM (prompts) or by the chain lengths ->
// page -> store (single tokens).
//
// 8 prompts of up to 4096 tokens, 12 heads x 64, bf16 to 4 bits: 46 us, 60 % of the copy rate; with four heads per lane
// and four CTAs per SM (that and the read: 66 us; three CTAs 74, two 86; two heads 74 to 78).
//
// A lane has 8 dims of kQuantRows heads of a token's keys, queries or values, which share cos and sin; a
// row's lanes lie side by side in a warp, as many tokens as fit. CTAs of one kind and group of heads each
// (blockIdx.z), so that warps do not diverge. The half that the rotation needs and the largest value of a
// group come from the row's other lanes. All loads are asked for before the first is used. Rows must be
// whole 16-byte pieces; quant_append_any_kernel takes the rest. Sequence blockIdx.y.
template <typename T>
constexpr int kQuantRows = sizeof(T) == 2 ? 4 : 2;

template <typename T, typename C, int BITS>
__global__ void __launch_bounds__(256, 4) quant_append_kernel(const __grid_constant__ QuantAppendParams p) {
  constexpr int ROWS = kQuantRows<T>;
  pdl_wait();
  const PagedAppendParams& a = p.a;
  const PagedCache& c = a.c;
  const int lane = threadIdx.x & 31, pieces = c.Dh / 8, b = blockIdx.y;
  const int sub = lane * p.lane_m >> 10, piece = lane - sub * pieces;  // lane / pieces
  int t = (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * p.per + sub;
  const int kvg = (c.Hkv + ROWS - 1) / ROWS, z = blockIdx.z;
  const int kind = z < kvg ? 0 : z < 2 * kvg ? 2 : 1;  // keys, values, queries
  const int r0 = (z - (kind == 0 ? 0 : kind == 2 ? kvg : 2 * kvg)) * ROWS;
  const bool there = sub < p.per && t < a.N && (kind == 1 || !a.counts || t < a.counts[b]);
  if (!__any_sync(0xffffffffu, there)) return;
  if (!there) t = 0;
  const int rows = there ? min(ROWS, (kind == 1 ? a.Hq : c.Hkv) - r0) : 0;
  const int64_t* s = kind == 0 ? a.ks : kind == 1 ? a.qs : a.vs;
  const T* from = (const T*)(kind == 0 ? a.k : kind == 1 ? a.q : a.v) + b * s[0] + r0 * s[1] + t * s[2] + piece * 8;
  Eight<T> x[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    if (k < rows) x[k].load(from + k * s[1]);
    else x[k] = Eight<T>{};
  }
  const bool turn = kind != 2 && a.cosv;
  Eight<C> cs{}, sn{};
  if (turn) {
    const int64_t at = b * a.cos_bs + (int64_t)t * c.Dh + piece * 8;
    cs.ldg((const C*)a.cosv + at);
    sn.ldg((const C*)a.sinv + at);
  }
  const int base = lane - piece, half = pieces / 2, other = base + (piece < half ? piece + half : piece - half);
  float2 co[4], si[4];
  cs.open(co);
  sn.open(si);
  if (piece < half) {
#pragma unroll
    for (int d = 0; d < 4; ++d) si[d] = make_float2(-si[d].x, -si[d].y);
  }
  auto rotate = [&](const Eight<T>& in, float2 (&v)[4]) {
    in.open(v);
    if (!turn) return;
    float2 w[4];
    in.from_lane(other).open(w);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if constexpr (sizeof(T) == 2 && sizeof(C) == 2)
        v[d] = fma2(v[d], co[d], mul2(w[d], si[d]));  // products of bf16 values are exact
      else
        v[d] = make_float2(quant_rotate(T(), C(), v[d].x, w[d].x, co[d].x, si[d].x),
                           quant_rotate(T(), C(), v[d].y, w[d].y, co[d].y, si[d].y));
    }
  };
  if (kind == 1) {
    T* to = (T*)a.q_out + (((int64_t)b * a.Hq + r0) * a.N + t) * c.Dh + piece * 8;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      float2 v[4];
      rotate(x[k], v);
      Eight<T> y;
      y.close(v);
      if (k < rows) y.store(to + k * ((int64_t)a.N * c.Dh));
    }
    return;
  }
  int64_t slot;
  int page = 0, row = 0;
  const bool stored = there && append_place(a, b, t, slot, page, row, SITE_QUANT_APPEND);
  const int64_t head = (int64_t)r0 * c.page_size + row;  // row of the first head in the page
  uint8_t* codes = (uint8_t*)(kind ? c.v : c.k) + page * (kind ? c.v_stride : c.k_stride) + head * p.row + piece * BITS;
  __nv_bfloat16* scales = (__nv_bfloat16*)p.scales + page * p.s_stride + (head * 2 + (kind != 0)) * p.groups + piece / 4;
  const int64_t code_step = (int64_t)c.page_size * p.row, scale_step = (int64_t)c.page_size * 2 * p.groups;
  if (stored && kind == 0 && a.mass)
    for (int k = piece; k < rows; k += pieces) a.mass[((int64_t)b * c.Hkv + r0 + k) * a.mass_width + slot] = 0.f;
  const int next = base + (piece ^ 1), over = base + ((piece ^ 2) < pieces ? piece ^ 2 : piece);  // of the same group
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    float2 v[4];
    rotate(x[k], v);
    float largest = max_abs(v[0].x, v[0].y, v[1].x);
    largest = max_abs(max_abs(largest, v[1].y, v[2].x), max_abs(v[2].y, v[3].x, v[3].y), 0.f);
    largest = max_abs(largest, __shfl_sync(0xffffffffu, largest, next), 0.f);
    largest = max_abs(largest, __shfl_sync(0xffffffffu, largest, over), 0.f);
    float scale, inv;
    quant_scale<BITS>(largest, scale, inv);
    uint32_t out[BITS / 4];
    quant_codes<BITS>(v, scale, inv, out);
    if (!stored || k >= rows) continue;
    if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(codes + k * code_step) = out[0];
    else *reinterpret_cast<uint2*>(codes + k * code_step) = make_uint2(out[0], out[1]);
    if (piece % 4 == 0) scales[k * scale_step] = __float2bfloat16_rn(scale);
  }
}

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
    quant_scale<BITS>(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r) & 0x7fffffffu)), scale, inv);
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

// 8 codes of 4 or 8 bits times their scale. bf16 from 4 bits: 128 + u is a bf16 with u in its last bits, and
// its difference to 136 and the product are one rounding each, the first exact.
template <int BITS>
ONE_DEVINL void quant_open(const uint32_t (&w)[BITS / 4], __nv_bfloat16 scale, Eight<__nv_bfloat16>& out) {
  const uint32_t s = __bfloat16_as_ushort(scale) * 0x10001u;
  if constexpr (BITS == 4) {
    uint32_t x[4];  // dims j and j + 4
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = bf2_mul(bf2_add((w[0] >> 4 * j & 0x000f000fu) | 0x43004300u, 0xc308c308u), s);
    out.u = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632),
                       __byte_perm(x[2], x[3], 0x7632));
  } else {
    const float f = __bfloat162float(scale);
    float2 v[4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      (&v[j / 2].x)[j & 1] = (__uint_as_float(__byte_perm(w[j / 4], 0x4b000000u, 0x7540 + j % 4)) - 8388736.f) * f;
    out.close(v);
  }
}
template <int BITS>
ONE_DEVINL void quant_open(const uint32_t (&w)[BITS / 4], __nv_bfloat16 scale, Eight<float>& out) {
  const float f = __bfloat162float(scale);
  float2 v[4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = BITS == 4 ? (w[0] >> 4 * j & 15u) | 0x4b000000u : __byte_perm(w[j / 4 % (BITS / 4)], 0x4b000000u, 0x7540 + j % 4);
    (&v[j / 2].x)[j & 1] = (__uint_as_float(u) - (8388608.f + QuantCode<BITS>::kZero)) * f;
  }
  out.close(v);
}

// Slots starts[b] .. starts[b] + N - 1 of every sequence, those not below lengths[b] as zeros. A lane has 8
// dims of a slot's keys and values of kReadHeads heads, which share the page; its loads are in flight
// together. A copy that grows fourfold: bound by HBM, that is by what it writes: 16 x up to 4096 slots, 12
// heads x 64, 4 bits to bf16: 40 us, 89 % of the copy rate.
constexpr int kReadHeads = 4;

template <typename T, int BITS>
__global__ void __launch_bounds__(256) quant_read_kernel(const __grid_constant__ QuantReadParams p) {
  pdl_wait();
  const PagedCache& c = p.m.c;
  const int pieces = c.Dh / 8, b = blockIdx.y, hg = blockIdx.z * kReadHeads;
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;
  const int t = (int)(i / pieces), piece = (int)(i - (uint32_t)t * pieces), heads = min(kReadHeads, c.Hkv - hg);
  if (t >= p.N) return;
  const int len = paged_length(c, b, SITE_QUANT_READ), first = p.starts ? p.starts[b] : 0;
  const int64_t slot = (int64_t)first + t;
  int page = -1, at = 0;
  if (first < 0) set_err(c.err, ERR_BAD_ARG, SITE_QUANT_READ);
  if (slot >= 0 && slot < len) {
    const int index = (int)slot / c.page_size;
    page = paged_page(c, c.table, b * c.table_stride, index, SITE_QUANT_READ);
    at = (int)slot - index * c.page_size;
  }
  uint32_t w[2][kReadHeads][BITS / 4] = {};
  __nv_bfloat16 s[2][kReadHeads];
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h) {
    s[0][h] = s[1][h] = __float2bfloat16_rn(0.f);
    if (page >= 0 && h < heads) {
      const int64_t r = (int64_t)(hg + h) * c.page_size + at;
      const uint8_t *k = (const uint8_t*)c.k + page * c.k_stride + r * p.m.row + piece * BITS;
      const uint8_t *v = (const uint8_t*)c.v + page * c.v_stride + r * p.m.row + piece * BITS;
      const __nv_bfloat16* sc = (const __nv_bfloat16*)p.m.scales + page * p.m.s_stride + r * 2 * p.m.groups + piece / 4;
      if constexpr (BITS == 4) {
        w[0][h][0] = *reinterpret_cast<const uint32_t*>(k);
        w[1][h][0] = *reinterpret_cast<const uint32_t*>(v);
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(k), y = *reinterpret_cast<const uint2*>(v);
        w[0][h][0] = x.x; w[0][h][1] = x.y; w[1][h][0] = y.x; w[1][h][1] = y.y;
      }
      s[0][h] = sc[0];
      s[1][h] = sc[p.m.groups];
    }
  }
  const int64_t out = (((int64_t)b * c.Hkv + hg) * p.N + t) * c.Dh + piece * 8, step = (int64_t)p.N * c.Dh;
#pragma unroll
  for (int h = 0; h < kReadHeads; ++h) {
    if (h >= heads) break;
    Eight<T> x;
    quant_open<BITS>(w[0][h], s[0][h], x);
    if (page < 0) x = Eight<T>{};
    x.store((T*)p.k + out + h * step);
    quant_open<BITS>(w[1][h], s[1][h], x);
    if (page < 0) x = Eight<T>{};
    x.store((T*)p.v + out + h * step);
  }
}

}  // namespace one
