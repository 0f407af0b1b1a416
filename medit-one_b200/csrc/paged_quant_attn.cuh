// Attention of one new token per sequence over a paged cache held in 4 or 8 bits (paged_quant.cuh), in
// the frame of paged_attn.cuh: the engine below takes the place of PaBf16 and PaF32.
//
//   s_t = scale log2(e) sum_g ks[t, g] (q_g . c_g)        c = u - z, the stored byte or half less its offset z
//   o_g = sum_t (2^(s_t - m) vs[t, g]) c_g
//
// The scales of a group of 32 dims factor out of its products, so the matrix instructions take the codes
// themselves. HBM bounds the long cases in principle (72 bytes per slot and kv head of 64 dims at 4 bits);
// per byte read there are four times the products of a bf16 cache, so what counts is instructions per code:
//  - a code lies in the low bits of an fp16 whose exponent is 0 (or 1), and that fp16 is u 2^-24, exactly:
//    one AND opens two codes, and no conversion follows. Halves of bytes at bits 4-7 read as u 2^-20; q,
//    or the output's scaling, takes up the difference.
//  - keys: sum q u starts from -z sum q (per query and group, computed once), so u needs no subtraction.
//    That costs three bits of the fp32 sum at most (u reaches 2 z, c reaches z).
//  - values: u - z by one packed addition (exact), since a sum over many slots of p z would drown o.
//  - ldmatrix brings a 16-byte piece of eight rows to the lanes as the B operands need it: keys straight,
//    values transposed, where a 16-bit element is four (two) codes of one slot.
// fp16 takes q scaled by a power of two to [2^14, 2^15) per row, and 2^(s - m) vs 2^15 / ref with ref a
// power of two above all the value scales so far, which rises like the running maximum. A bf16 q is exact
// in it down to 2^-38 of the row's largest; the weights are rounded to 11 bits (2^-11 each, against the
// output's 2^-8). In fp32, q and the weights are two fp16 parts (22 bits), in rows r and r + 8.
#pragma once

#include "paged_attn.cuh"
#include "paged_quant.cuh"

namespace one {

ONE_DEVINL void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0,
                              float c1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %11, %11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
ONE_DEVINL void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool TRANS>
ONE_DEVINL void ldmatrix_x4(uint32_t (&w)[4], uint32_t at) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
template <bool TRANS>
ONE_DEVINL void ldmatrix_x2(uint32_t& a, uint32_t& b, uint32_t at) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at) : "memory");
}
ONE_DEVINL uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
ONE_DEVINL float f16_lo(uint32_t u) {
  float f;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, l;}" : "=f"(f) : "r"(u));
  return f;
}
ONE_DEVINL float f16_hi(uint32_t u) {
  float f;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.f32.f16 %0, h;}" : "=f"(f) : "r"(u));
  return f;
}
ONE_DEVINL uint32_t f16x2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The first `bytes` of 16, 8 or 4 bytes, the rest as zeros
template <int N>
ONE_DEVINL void cp_async_some(uint32_t s, const void* g, int bytes) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(g), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(s), "l"(g), "n"(N), "r"(bytes) : "memory");
}

// PQ_8, PQ_16: bf16, up to 8 or 16 query heads. PQ_PAIR: fp32, up to 8, in two parts.
enum PqKind { PQ_8, PQ_16, PQ_PAIR };

template <int DH_, int BITS_, PqKind KIND>
struct PaQuant {
  using T = std::conditional_t<KIND == PQ_PAIR, float, __nv_bfloat16>;
  using Cell = uint8_t;
  static constexpr bool kQuant = true;
  static constexpr int DH = DH_, BITS = BITS_, ROWS = KIND == PQ_16 ? 16 : 8;
  static constexpr bool SECOND = KIND != PQ_8;           // rows r + 8 are used
  static constexpr int RW = KIND == PQ_16 ? 2 : 1;       // query rows of a lane
  static constexpr int G = DH / kQuantGroup;             // groups of a row
  static constexpr int RB = DH * BITS / 8, CH = RB / 16; // bytes and pieces of a row
  static constexpr int SR = 4 * G;                       // bytes of a slot's scales
  static constexpr int PG = CH / G;                      // pieces of a group: 1 or 2
  static constexpr int NT = DH / 8;                      // value tiles
  static constexpr int EP = BITS == 4 ? 4 : 2;           // codes in 16 bits
  static constexpr float kZero = BITS == 4 ? 8.f : 128.f;
  static constexpr int kGroup = 16 * (2 * RB + SR);      // bytes of 16 slots
  static constexpr int kValues = 16 * RB, kScales = 32 * RB;
  static constexpr int kGroups = DH * BITS <= 128 ? 4 : DH * BITS <= 256 ? 2 : 1;  // 16-slot groups per warp and step
  static constexpr int TILE = 16 * kGroups * kPaWarps;
  static constexpr int kStages = 4, kStagesFew = kStages;
  static constexpr int kExtra = 0;
  ONE_DEVINL static float weight(float x) { return KIND == PQ_PAIR ? exp2f(x) : ex2_approx(x); }

  uint32_t qa[G][2][SECOND ? 4 : 2];  // A operands of a group's two products: a0, a2, then a1, a3
  float off[G][SECOND ? 2 : 1];       // -z sum q, rows r and r + 8
  float fac[RW];                      // from sums to scores
  float o[NT][4];
  float m[RW], l[RW];
  float ref, mult;                    // above all the value scales so far; 2^15 / ref

  // Where piece ch of row `row` lies: eight rows' pieces ch are on different banks, and a 128-byte line of
  // memory stays one.
  ONE_DEVINL static int at(int row, int ch) {
    const int x = CH == 2 || CH == 6 ? row >> 2 & 1 : CH == 4 ? row >> 1 & 3 : CH == 8 ? row & 7 : 0;
    return row * RB + (ch ^ x) * 16;
  }
  // The copies of 16 rows that follow one another in memory; k, v, s from this lane's 16 bytes on. live:
  // of so many rows, the rest as zeros.
  template <bool ALL>
  ONE_DEVINL static void copy(uint32_t to, const uint8_t* k, const uint8_t* v, const uint8_t* s, int live) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < (16 * CH + 31) / 32; ++n) {
      const int e = n * 32 + lane, row = e / CH, ch = e % CH;
      if (16 * CH % 32 == 0 || e < 16 * CH) {
        const uint32_t x = to + at(row, ch);
        cp_async_some<16>(x, k + n * 512, ALL || row < live ? 16 : 0);
        cp_async_some<16>(x + kValues, v + n * 512, ALL || row < live ? 16 : 0);
      }
    }
    if (lane < 4 * G) cp_async_some<16>(to + kScales + lane * 16, s, ALL ? 16 : min(16, max(0, live * SR - lane * 16)));
  }
  // Rows anywhere: lane t (16 + t) holds slot t's page and row in the head, or -1; pieces of 16 bytes or of 8.
  ONE_DEVINL static void copy_any(uint32_t to, const PagedAttn& p, const uint8_t* k, const uint8_t* v, const uint8_t* s, int page,
                                  int row) {
    const int lane = threadIdx.x & 31;
    auto rows = [&](auto unit) {
      constexpr int U = decltype(unit)::value, PER = RB / U;
#pragma unroll
      for (int n = 0; n < (16 * PER + 31) / 32; ++n) {
        const int e = n * 32 + lane, r = e / PER, ch = e % PER;
        const int pg = __shfl_sync(0xffffffffu, page, r & 15), rw = __shfl_sync(0xffffffffu, row, r & 15);
        if (16 * PER % 32 == 0 || e < 16 * PER) {
          const bool there = pg >= 0 && ch * U < p.row;
          const int64_t in = (int64_t)rw * p.row + ch * U;
          const uint32_t x = to + at(r, ch * U / 16) + ch * U % 16;
          cp_async_some<U>(x, there ? k + pg * p.c.k_stride + in : k, there ? U : 0);
          cp_async_some<U>(x + kValues, there ? v + pg * p.c.v_stride + in : v, there ? U : 0);
        }
      }
    };
    if (p.vec16) rows(Int<16>()); else rows(Int<8>());
#pragma unroll
    for (int n = 0; n < (16 * G + 31) / 32; ++n) {
      const int e = n * 32 + lane, r = e / G, w = e % G;
      const int pg = __shfl_sync(0xffffffffu, page, r & 15), rw = __shfl_sync(0xffffffffu, row, r & 15);
      if (16 * G % 32 == 0 || e < 16 * G)
        cp_async_some<4>(to + kScales + e * 4, pg >= 0 ? s + pg * p.s_stride + (int64_t)rw * SR + w * 4 : s, pg >= 0 ? 4 : 0);
    }
  }

  ONE_DEVINL void begin(const PagedAttn& p, uint8_t*, const T* q, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      // this lane's 8 dims of each group, in memory's order: 8 c .., or 4 c .. and 16 + 4 c ..
      float x[G][8], top = 0.f;
      const bool in = r + 8 * w < rows;
      const T* y = q + (int64_t)(r + 8 * w) * p.q_hs;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int d0 = g * 32 + (BITS == 4 ? 8 * c : 4 * c);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int d = d0 + (BITS == 4 ? 4 : 16) * hh;
          const bool there = in && d < p.c.Dh;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[g][4 * hh + i] = 0.f;
          if (there) {
            if (p.q_vec) {
              if constexpr (KIND == PQ_PAIR) {
                const float4 u = *reinterpret_cast<const float4*>(y + d);
                x[g][4 * hh] = u.x; x[g][4 * hh + 1] = u.y; x[g][4 * hh + 2] = u.z; x[g][4 * hh + 3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(y + d);
                x[g][4 * hh] = bf2_lo(u.x); x[g][4 * hh + 1] = bf2_hi(u.x); x[g][4 * hh + 2] = bf2_lo(u.y); x[g][4 * hh + 3] = bf2_hi(u.y);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) x[g][4 * hh + i] = ld<T>(y + d + i);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[g][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = (int)(__float_as_uint(top) >> 23);                  // 0 .. 255
      const float up = __uint_as_float((uint32_t)min(254, 268 - e) << 23);  // 2^14 over the power of two of top
      // acc = sum q up u 2^-24; halves that read as u 2^-20 have q up 2^-4
      fac[w] = p.scale_log2 * 1024.f * __uint_as_float((uint32_t)max(14, e) << 23);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const float f = BITS == 4 && k ? up * 0.0625f : up, back = BITS == 4 && k ? 16.f : 1.f;
            // dims of this register in memory's order
            const int i0 = BITS == 4 ? k + 2 * a : 4 * k + a, i1 = BITS == 4 ? i0 + 4 : i0 + 2;
            const float y0 = x[g][i0] * f, y1 = x[g][i1] * f;
            const uint32_t hi = pack_f16x2(y0, y1);
            sum[0] += (f16_lo(hi) + f16_hi(hi)) * back;
            if (KIND == PQ_16 && w == 1) {
              qa[g][k][(SECOND ? 2 : 0) + a] = hi;
            } else {
              qa[g][k][a] = hi;
            }
            if constexpr (KIND == PQ_PAIR) {
              const uint32_t lo = pack_f16x2(y0 - f16_lo(hi), y1 - f16_hi(hi));
              sum[1] += (f16_lo(lo) + f16_hi(lo)) * back;
              qa[g][k][2 + a] = lo;
            }
          }
#pragma unroll
        for (int j = 0; j < (KIND == PQ_PAIR ? 2 : 1); ++j) {
          sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
          sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
          off[g][SECOND ? w + j : 0] = sum[j] * (-kZero * 5.9604644775390625e-8f);
        }
      }
      m[w] = -INFINITY;
      l[w] = 0.f;
    }
    ref = 0.f;
    mult = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }

  // A slot pair's scales: element i of slot h (K_0 .., V_0 ..)
  struct Scales {
    uint32_t w[2 * G];
    ONE_DEVINL float operator()(int h, int i) const {
      const uint32_t x = w[h * G + i / 2];
      return i & 1 ? bf2_hi(x) : bf2_lo(x);
    }
    ONE_DEVINL void load(uint32_t at) {
      if constexpr (G % 2 == 0) {
#pragma unroll
        for (int k = 0; k < 2 * G; k += 4)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[k]), "=r"(w[k + 1]), "=r"(w[k + 2]), "=r"(w[k + 3]) : "r"(at + k * 4) : "memory");
      } else {
#pragma unroll
        for (int k = 0; k < 2 * G; k += 2)
          asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[k]), "=r"(w[k + 1]) : "r"(at + k * 4) : "memory");
      }
    }
  };
  // [piece][slots 0-7, 8-15] of a group's 16 rows
  template <bool TRANS>
  ONE_DEVINL static void pieces(uint32_t (&w)[CH][2], uint32_t base) {
    const int lane = threadIdx.x & 31, row = 8 * (lane >> 3 & 1) + (lane & 7), up = lane >> 4;
#pragma unroll
    for (int i = 0; i + 1 < CH; i += 2) {
      uint32_t x[4];
      ldmatrix_x4<TRANS>(x, base + at(row, i + up));
      w[i][0] = x[0]; w[i][1] = x[1]; w[i + 1][0] = x[2]; w[i + 1][1] = x[3];
    }
    if constexpr (CH % 2) ldmatrix_x2<TRANS>(w[CH - 1][0], w[CH - 1][1], base + at(row, CH - 1));
  }
  // Two codes of a word as fp16: those at half (4 bits) or byte (8 bits) e of each of its 16-bit elements
  ONE_DEVINL static uint32_t open(uint32_t w, int e) {
    if (BITS == 4) return (e & 2 ? w >> 8 : w) & (e & 1 ? 0x00f000f0u : 0x000f000fu);
    return (e ? w >> 8 : w) & 0x00ff00ffu;
  }

  ONE_DEVINL void consume(const PagedAttn& p, const uint8_t* stage, const uint32_t (&live)[kGroups], float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const uint32_t base = smem_u32(stage);
    float pr[kGroups][RW][4];
    float vmax = 0.f;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      float s[RW][4];
#pragma unroll
      for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = s[w][2] = s[w][3] = 0.f;
      if (live[i]) {
        uint32_t kw[CH][2];
        pieces<false>(kw, base + i * kGroup);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Scales sc;
          sc.load(base + i * kGroup + kScales + (8 * j + 2 * c) * SR);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float a[4];
            const uint32_t w0 = kw[g * PG][j], w1 = kw[g * PG + PG - 1][j];
            // 4 bits: halves 0, 2 then 1, 3 of the word; 8 bits: bytes 0, 1 of the first word, then of the second
            mma_f16_16816(a, qa[g][0][0], SECOND ? qa[g][0][SECOND ? 2 : 0] : 0, qa[g][0][1], SECOND ? qa[g][0][SECOND ? 3 : 0] : 0,
                          open(w0, 0), open(w0, BITS == 4 ? 2 : 1), off[g][0], SECOND ? off[g][SECOND ? 1 : 0] : 0.f);
            mma_f16_16816(a, qa[g][1][0], SECOND ? qa[g][1][SECOND ? 2 : 0] : 0, qa[g][1][1], SECOND ? qa[g][1][SECOND ? 3 : 0] : 0,
                          open(w1, BITS == 4 ? 1 : 0), open(w1, BITS == 4 ? 3 : 1));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float ks = sc(h, g);
              if constexpr (KIND == PQ_PAIR) {
                s[0][2 * j + h] += ks * (a[h] + a[2 + h]);
              } else {
#pragma unroll
                for (int w = 0; w < RW; ++w) s[w][2 * j + h] += ks * a[2 * w + h];
              }
              vmax = fmaxf(vmax, sc(h, G + g));
            }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int t = 0; t < 4; ++t) pr[i][w][t] = s[w][t] * fac[w];
      if (live[i] != 0xffffu) {
        const uint32_t mine = live[i] >> (2 * c);
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (!(mine >> (8 * (t >> 1) + (t & 1)) & 1)) pr[i][w][t] = -INFINITY;
      }
      if (scores) {
#pragma unroll
        for (int w = 0; w < RW; ++w)
          if (r + 8 * w < rows) {
            float* to = scores + (r + 8 * w) * p.score_ld + 16 * i + 2 * c;
            *reinterpret_cast<float2*>(to) = make_float2(pr[i][w][0], pr[i][w][1]);
            *reinterpret_cast<float2*>(to + 8) = make_float2(pr[i][w][2], pr[i][w][3]);
          }
      }
    }
    float mx[RW];
    bool rises = vmax > ref;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      mx[w] = pr[0][w][0];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        mx[w] = fmax3(mx[w], pr[i][w][0], pr[i][w][1]);
        mx[w] = fmax3(mx[w], pr[i][w][2], pr[i][w][3]);
      }
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
      rises |= mx[w] > m[w];
    }
    if (__any_sync(0xffffffffu, rises)) {
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
      vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));
      float f = 1.f;
      if (vmax > ref) {  // the same in all lanes; 2^-100 < ref <= 2^127
        const uint32_t e = min(max(__float_as_uint(vmax) >> 23, 27u) + 1, 254u);
        const float now = __uint_as_float(e << 23);
        f = ref == 0.f ? 0.f : ref * __uint_as_float((254 - min(e, 253u)) << 23) * (e == 254u ? 0.5f : 1.f);
        ref = now;
        mult = __uint_as_float((269 - e) << 23);
      }
      float a[2];
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        const float mn = fmaxf(m[w], mx[w]);
        a[w] = weight(m[w] - (mn == -INFINITY ? 0.f : mn));
        m[w] = mn;
        l[w] *= a[w];
        a[w] *= f;
      }
      if (RW == 1) a[1] = a[0];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] *= a[0]; o[i][1] *= a[0];
        if (SECOND) { o[i][2] *= a[1]; o[i][3] *= a[1]; }
      }
    }
    float ms[RW];
#pragma unroll
    for (int w = 0; w < RW; ++w) ms[w] = m[w] == -INFINITY ? 0.f : m[w];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      if (!live[i]) continue;
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        float (&x)[4] = pr[i][w];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = weight(x[t] - ms[w]);
        l[w] += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] *= mult;
      }
      uint32_t vw[CH][2];
      pieces<true>(vw, base + i * kGroup + kValues);
      Scales sc[2];
      sc[0].load(base + i * kGroup + kScales + 2 * c * SR);
      sc[1].load(base + i * kGroup + kScales + (8 + 2 * c) * SR);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t hi[2], second[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float v0 = sc[j](0, G + g), v1 = sc[j](1, G + g);
          const float y0 = pr[i][0][2 * j] * v0, y1 = pr[i][0][2 * j + 1] * v1;
          hi[j] = pack_f16x2(y0, y1);
          if constexpr (KIND == PQ_PAIR) second[j] = pack_f16x2(y0 - f16_lo(hi[j]), y1 - f16_hi(hi[j]));
          if constexpr (KIND == PQ_16) second[j] = pack_f16x2(pr[i][RW - 1][2 * j] * v0, pr[i][RW - 1][2 * j + 1] * v1);
        }
#pragma unroll
        for (int k = 0; k < PG; ++k)
#pragma unroll
          for (int e = 0; e < EP; ++e) {
            const uint32_t z = BITS == 8 || (e & 1) ? 0x80808080u : 0x80088008u;  // -z 2^-24 (bytes), -z 2^-20, -z 2^-24
            mma_f16_16816(o[(g * PG + k) * EP + e], hi[0], second[0], hi[1], second[1],
                          f16x2_add(open(vw[g * PG + k][0], e), z), f16x2_add(open(vw[g * PG + k][1], e), z));
          }
      }
    }
  }

  // This warp's (m, l) [ROWS][2] and o [rows][DH] into shared memory.
  ONE_DEVINL void leave(float* ml, float* so, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      float t = l[w];
      t += __shfl_xor_sync(0xffffffffu, t, 1);
      t += __shfl_xor_sync(0xffffffffu, t, 2);
      if (c == 0) {
        ml[2 * (r + 8 * w)] = m[w];
        ml[2 * (r + 8 * w) + 1] = t;
      }
      if (r + 8 * w >= rows) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int e = i % EP, d0 = i / EP * 8 * EP + e;  // column n is dim d0 + EP n
        const float f = BITS == 4 && (e & 1) ? 32.f : 512.f;  // 2^24 or 2^20, over mult's 2^15
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = KIND == PQ_PAIR ? o[i][h] + o[i][2 + h] : o[i][2 * w + h];
          so[(r + 8 * w) * DH + d0 + EP * (2 * c + h)] = x * f * ref;
        }
      }
    }
  }
};

}  // namespace one
