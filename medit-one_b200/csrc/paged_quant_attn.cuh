// Attention of one new token per sequence over a paged cache held in 4 or 8 bits (paged_quant.cuh), in
// the frame of paged_attn.cuh: the engine below takes the place of PaBf16 and PaF32.
//
//   s_t = scale log2(e) sum_g ks[t, g] (q_g . c_g)        c = u - z, the stored byte or half less its offset z
//   o_g = sum_t (2^(s_t - m) vs[t, g]) c_g
//
// The scales of a group of 32 dims factor out of its products, so the matrix instructions take the codes
// themselves. HBM bounds the long cases in principle (72 bytes per slot and kv head of 64 dims at 4 bits);
// per byte read there are four times the products of a bf16 cache, so what counts is instructions per code:
//  - keys, in fp16: the bits of 1024 above the code (16 times it, of halves of bytes at bits 4-7) and one packed
//    addition or fma, which takes 1024 and z off (and 16 out), exactly. (A code as it lies is an fp16 u 2^-24 whose
//    exponent is 0: one AND opens two, and the offset goes off their sum. But an instruction aligns its terms by
//    their operands' exponents, up to 2^10 above such numbers, and where large dims of q meet codes of 0 their
//    offsets cancel: the scores of dims 2^8 below those were off by ten times an fp32 sum's bound, of dims 2^16
//    below by thousands of times, at 38.8 us instead of 39.0 and 44.3 instead of 45.8 in the cases below.)
//  - q scaled by a power of two per row and group, its largest to [2^14, 2^15): a bf16 q is exact in it down to
//    2^-31 of its group's largest; in fp32, q is two fp16 parts (22 bits), in neighbouring columns, the second with
//    2^11 more: 18 bits are left at 2^-30. (Keys in bf16, as the values are, would take any q as it is: 40.4 us
//    instead of 39.1 at 64 x 4096 ragged, in 8 bits, which bf16 opens in two steps, 54 instead of 48.)
//  - values, in bf16: the bits of 128 or 16 above the code and one packed addition of -(128 + z) or -(16 + z),
//    both exact (a sum over many slots of p z would drown o).
//  - weights times their scales, in bf16 parts, which together have 16 bits (fp32: all 24): a part has its own
//    exponent, so that each output is as good as its own terms, whatever the scales of other slots and
//    groups are. (fp16 with an exponent in common, of the largest scale so far, lost values 2^-28 of it,
//    and took 36 us where this takes 39.)
//  - the codes are the instructions' 16 rows: S^T = K Q^T has slots as rows, O^T = V^T P^T dims, and the
//    queries are the 8 columns. ldmatrix brings 16-byte pieces of eight slots to the lanes as both need
//    them: keys straight, values transposed, where a 16-bit element is four (two) codes of one slot.
//    movmatrix turns the weights from rows to columns in between.
// Measured: 64 ragged sequences up to 4096 slots, 12 heads x 64, 4 bits: 39 us, 46 % of the measured copy rate (dense
// bf16: 73); 8 up to 32768, 8 heads x 128 of 4 queries: 46 us, 54 %; one of 1048576, 12 x 64: 202 us, 69 %.
#pragma once

#include "paged_attn.cuh"
#include "paged_quant.cuh"

namespace one {

ONE_DEVINL void mma_bf16_acc(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
ONE_DEVINL void mma_f16_acc(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Lane (r, c) holds elements 2 c, 2 c + 1 of row r of an 8 x 8 matrix; the same of the transposed one
ONE_DEVINL uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
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
ONE_DEVINL uint32_t f16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// (a & mask) | bits in one instruction (two, where the compiler was left to it: 64 x 4096 ragged 41.5 us, 38.9 so; fp32
// 50.3, 44.4)
ONE_DEVINL uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
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

// PQ_4, PQ_8, PQ_16: bf16, up to so many query heads. PQ_PAIR4, PQ_PAIR8: fp32 in two parts, up to 4 or 8.
// PQ_4 and the pairs have a query's parts in the columns 2 c and 2 c + 1, so that a lane has the scores of one
// head rather than of two (PQ_4: q has one part, its weights two).
enum PqKind { PQ_4, PQ_8, PQ_16, PQ_PAIR4, PQ_PAIR8 };

// Tiles of a list that a segment's begin and end count as. Us at 0, 2, 3, 5 of them: 64 x 4096 ragged x 12 x 64 55.0,
// 41.6, 41.5, 43.5; in 8 bits 69, 50.0, 51.6, 53.5; 64 x 1024 21.8, 19.1, 20.2, 20.9 (before codes opened with one
// instruction less each, as below).
constexpr int kQuantUnits = 2;

template <int DH_, int BITS_, PqKind KIND>
struct PaQuant {
  static constexpr bool PAIR = KIND == PQ_PAIR4 || KIND == PQ_PAIR8;
  using T = std::conditional_t<PAIR, float, __nv_bfloat16>;
  using Cell = uint8_t;
  static constexpr bool kQuant = true;
  static constexpr int kSite = SITE_QUANT_ATTN;
  static constexpr int DH = DH_, BITS = BITS_, ROWS = KIND == PQ_16 ? 16 : KIND == PQ_4 || KIND == PQ_PAIR4 ? 4 : 8;
  static constexpr int NL = KIND == PQ_16 || KIND == PQ_PAIR8 ? 2 : 1;  // tiles of 8 columns
  static constexpr bool ODD = KIND == PQ_8 || KIND == PQ_16;  // odd columns are queries of their own
  static constexpr int NP = KIND == PQ_4 ? 1 : 2;        // instructions that a weight's parts take: 2, or 3 of fp32
  static constexpr int QL = ODD ? 2 : 1, NQ = NL * QL;   // queries of a lane, per tile and in all
  static constexpr int G = DH / kQuantGroup;             // groups of a row
  static constexpr int RB = DH * BITS / 8, CH = RB / 16; // bytes and pieces of a row
  static constexpr int SR = 4 * G;                       // bytes of a slot's scales
  static constexpr int PG = CH / G;                      // pieces of a group: 1 or 2
  static constexpr int NT = DH / 16;                     // value tiles
  static constexpr int kGroup = 16 * (2 * RB + SR);      // bytes of 16 slots
  static constexpr int kValues = 16 * RB, kScales = 32 * RB;
  // 16-slot groups per warp and step, CTAs on an SM at most: long steps for independent work between the
  // instructions of a warp, as far as registers go. Us at 1, 2, 4 groups: 64 x 4096 ragged x 12 x 64, 4 bits 56, 45,
  // 42; in 8 bits 63, 53, 50; 8 x 32768 x 8 x 4 x 128 65, 51, 49; of 16 queries 105, 93, 174.
  static constexpr int kGroups = RB <= 64 && (NL == 1 || DH <= 64) ? 4 : 2;
  static constexpr int TILE = 16 * kGroups * kPaWarps;
  static constexpr int kStages = 2, kStagesFew = kStages;
  static constexpr int kQueries = ROWS * DH * (int)sizeof(T);  // bytes of a segment's queries
  static constexpr int kExtra = 0, kMaxPerSm = DH <= 32 ? (NL == 1 ? 4 : 3) : DH <= 64 && NL == 1 ? 3 : 2;
  static constexpr int kSegmentUnits = kQuantUnits;
  ONE_DEVINL static float weight(float x) { return PAIR ? exp2f(x) : ex2_approx(x); }

  uint32_t qb[NL][G][2][2];  // B operands of a group's two products
  float fac[NQ][G];          // from a group's sums to scores, positive
  float o[NL][NT][4];
  float m[NQ], l[NQ];
  uint32_t mine;             // where this lane's row of the first pieces lies

  // Where piece ch of row `row` lies: eight rows' pieces ch are on different banks, and a 128-byte line of
  // memory stays one.
  ONE_DEVINL static int at(int row, int ch) {
    const int x = CH == 2 || CH == 6 ? row >> 2 & 1 : CH == 4 ? row >> 1 & 3 : CH == 8 ? row & 7 : 0;
    return row * RB + (ch ^ x) * 16;
  }
  // at(row, 2 i + up) from at(row, up), for even i
  ONE_DEVINL static uint32_t step(uint32_t first, int i) { return (CH & (CH - 1)) == 0 ? first ^ (16 * i) : first + 16 * i; }
  // The copies of 16 rows that follow one another in memory; k, v, s from this lane's 16 bytes on. ALL: but
  // for the scales. live: of so many rows, the rest as zeros.
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
    if (!ALL && lane < 4 * G) cp_async_some<16>(to + kScales + lane * 16, s, min(16, max(0, live * SR - lane * 16)));
  }
  // The same of kGroups whole groups; lane from + g holds the places of group g in the pools, in 16 bytes
  ONE_DEVINL static void copy_step(uint32_t to, const uint8_t* k, const uint8_t* v, const uint8_t* s, uint32_t k_at, uint32_t v_at,
                                   uint32_t s_at, int from) {
    const int lane = threadIdx.x & 31;
    if constexpr (16 * CH % 32 == 0) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const uint8_t* kp = k + (uint64_t)__shfl_sync(0xffffffffu, k_at, from + g) * 16;
        const uint8_t* vp = v + (uint64_t)__shfl_sync(0xffffffffu, v_at, from + g) * 16;
#pragma unroll
        for (int n = 0; n < CH / 2; ++n) {
          const int e = n * 32 + lane;
          const uint32_t x = to + g * kGroup + at(e / CH, e % CH);
          cp_async_some<16>(x, kp + n * 512, 16);
          cp_async_some<16>(x + kValues, vp + n * 512, 16);
        }
      }
    } else {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const uint8_t* kp = k + (uint64_t)__shfl_sync(0xffffffffu, k_at, from + g) * 16;
        const uint8_t* vp = v + (uint64_t)__shfl_sync(0xffffffffu, v_at, from + g) * 16;
        copy<true>(to + g * kGroup, kp, vp, nullptr, 16);
      }
    }
    // scales: 4 G pieces per group, of all groups together
#pragma unroll
    for (int n = 0; n < (kGroups * 4 * G + 31) / 32; ++n) {
      const int e = n * 32 + lane, g = min(e / (4 * G), kGroups - 1), piece = e - g * (4 * G);
      // s is this lane's 16 bytes on; the piece's instead
      const uint8_t* sp = s + (uint64_t)__shfl_sync(0xffffffffu, s_at, from + g) * 16 + (piece - lane) * 16;
      if (kGroups * 4 * G % 32 == 0 || e < kGroups * 4 * G) cp_async_some<16>(to + g * kGroup + kScales + piece * 16, sp, 16);
    }
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

  // The queries of a segment, 16 bytes per copy, into [ROWS][DH]; only where q_vec and Dh is DH
  ONE_DEVINL static void copy_q(uint32_t to, const PagedAttn& p, const T* q, int rows) {
    constexpr int PER = DH * (int)sizeof(T) / 16;
    for (int e = threadIdx.x & 31; e < rows * PER; e += 32)
      cp_async_some<16>(to + e * 16, q + (e / PER) * p.q_hs + e % PER * (16 / (int)sizeof(T)), 16);
  }
  // q: rows `stride` apart, of whole vectors where vec
  ONE_DEVINL void begin(const PagedAttn& p, const T* q, int64_t stride, bool vec, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    mine = at(8 * (lane >> 3 & 1) + (lane & 7), CH == 1 ? 0 : lane >> 4);
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      // column r: query 8 n + r, or part r % 2 of query 4 n + r / 2 (PQ_4: the second part is 0). This lane's 8
      // dims of each group in memory's order: 8 c .., or 4 c .. and 16 + 4 c ..
      const int row = ODD ? 8 * n + r : 4 * n + (r >> 1);
      float x[G][8];
      const T* y = q + row * stride;
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int d = g * 32 + (BITS == 4 ? 8 * c + 4 * hh : 4 * c + 16 * hh);
          float* z = x[g] + 4 * hh;
          z[0] = z[1] = z[2] = z[3] = 0.f;
          if (row < rows && d < p.c.Dh) {
            if (vec) {
              if constexpr (PAIR) {
                const float4 u = *reinterpret_cast<const float4*>(y + d);
                z[0] = u.x; z[1] = u.y; z[2] = u.z; z[3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(y + d);
                z[0] = bf2_lo(u.x); z[1] = bf2_hi(u.x); z[2] = bf2_lo(u.y); z[3] = bf2_hi(u.y);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) z[i] = ld<T>(y + d + i);
            }
          }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[g][i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int)(__float_as_uint(top) >> 23);                      // 0 .. 255
        // 2^14 over the power of two of top, with the scale's sign
        const float up = copysignf(__uint_as_float((uint32_t)min(254, 268 - e) << 23), p.scale_log2);
        const float back = fabsf(p.scale_log2) * __uint_as_float((uint32_t)max(14, e) << 23) * 0x1p-14f;
        // lane (r, c) has columns 2 c and 2 c + 1 of the sums
#pragma unroll
        for (int h = 0; h < QL; ++h) fac[n * QL + h][g] = __shfl_sync(0xffffffffu, back, (2 * c + h) * 4);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const int i0 = BITS == 4 ? k + 2 * a : 4 * k + a, i1 = BITS == 4 ? i0 + 4 : i0 + 2;
            const float y0 = x[g][i0] * up, y1 = x[g][i1] * up;
            uint32_t w = pack_f16x2(y0, y1);
            if (!ODD && (r & 1)) {  // 2^11 times what the first part leaves: nothing of an infinity
              const float h0 = f16_lo(w), h1 = f16_hi(w);
              w = PAIR ? pack_f16x2(y0 == h0 ? 0.f : (y0 - h0) * 2048.f, y1 == h1 ? 0.f : (y1 - h1) * 2048.f) : 0;
            }
            qb[n][g][k][a] = w;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < NL; ++n)
#pragma unroll
      for (int i = 0; i < NT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }

  // A slot's scales, K_0 .., V_0 .., two of bf16 to a word. The upper one is an fp32 once the lower one's bits are
  // cleared (not by a product with 0, which leaves a NaN one).
  struct Scales {
    uint32_t w[G];
    ONE_DEVINL float get(int i) const { return i & 1 ? bf2_hi(w[i / 2]) : bf2_lo(w[i / 2]); }
    ONE_DEVINL void load(uint32_t at) {
      if constexpr (G == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
      else if constexpr (G == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
      else {
#pragma unroll
        for (int k = 0; k < G; ++k) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[k]) : "r"(at + 4 * k) : "memory");
      }
    }
  };
  // [piece][slots 0-7, 8-15] of a group's 16 rows
  template <bool TRANS>
  ONE_DEVINL void pieces(uint32_t (&w)[CH][2], uint32_t base) const {
#pragma unroll
    for (int i = 0; i + 1 < CH; i += 2) {
      uint32_t x[4];
      ldmatrix_x4<TRANS>(x, base + step(mine, i));
      w[i][0] = x[0]; w[i][1] = x[1]; w[i + 1][0] = x[2]; w[i + 1][1] = x[3];
    }
    if constexpr (CH % 2) ldmatrix_x2<TRANS>(w[CH - 1][0], w[CH - 1][1], base + step(mine, CH - 1));
  }
  // Two codes of a word, those at half (4 bits) or byte (8 bits) e of each of its 16-bit elements, in fp16
  ONE_DEVINL static uint32_t open_key(uint32_t w, int e) {
    if (BITS == 8) return f16x2_add(and_or(e ? w >> 8 : w, 0x00ff00ffu, 0x64006400u), 0xe480e480u);        // 1024 + u - 1152
    const uint32_t x = e & 2 ? w >> 8 : w;
    if (e & 1) return f16x2_fma(and_or(x, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);  // (1024 + 16 u) / 16 - 72
    return f16x2_add(and_or(x, 0x000f000fu, 0x64006400u), 0xe408e408u);                          // 1024 + u - 1032
  }
  // The same in bf16
  ONE_DEVINL static uint32_t open_value(uint32_t w, int e) {
    if (BITS == 4) {
      if (e & 1) return bf2_add(and_or(e & 2 ? w >> 9 : w >> 1, 0x00780078u, 0x41804180u), 0xc1c0c1c0u);  // 16 + u - 24
      return bf2_add(and_or(e & 2 ? w >> 8 : w, 0x000f000fu, 0x43004300u), 0xc308c308u);             // 128 + u - 136
    }
    const uint32_t x = e ? w >> 8 : w;  // of the 8 bits 7 fit: 128 + u % 128 - (u < 128 ? 256 : 128)
    return bf2_add(and_or(x, 0x007f007fu, 0x43004300u), (x & 0x00800080u) ^ 0xc380c380u);
  }
  // Weights as bf16 parts whose sum is the weight to 16 bits (PAIR: all 24), as B operands before their turn:
  // the two columns of y0 and y1, or of the parts of y0
  ONE_DEVINL static void parts(float y0, float y1, uint32_t (&w)[NP]) {
    const uint32_t u0 = __float_as_uint(y0), u1 = __float_as_uint(y1);
    const float r0 = y0 - bf2_hi(u0), r1 = y1 - bf2_hi(u1);  // exact
    if constexpr (ODD) {
      w[0] = __byte_perm(u0, u1, 0x7632);
      w[1] = pack_bf16x2(r0, r1);
    } else if constexpr (PAIR) {
      w[0] = __byte_perm(u0, __float_as_uint(r0), 0x7632);
      w[1] = __float_as_uint(r0 - bf2_hi(__float_as_uint(r0))) >> 16;
    } else {
      w[0] = pack_bf16x2(bf2_hi(u0), r0);
    }
  }

  // kGroups x 16 slots, all of them copied; live(i): a bit per slot of group i, full: all are set. scores:
  // row 0's scores of these slots, or null.
  template <typename F>
  ONE_DEVINL void consume(const PagedAttn& p, uint32_t base, bool full, F&& live, float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const uint32_t scale_at = base + kScales + r * SR;
    float pr[kGroups][NQ][2];  // slots r and r + 8
    Scales sc[kGroups][2];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      uint32_t kw[CH][2];
      pieces<false>(kw, base + i * kGroup);
      sc[i][0].load(scale_at + i * kGroup);
      sc[i][1].load(scale_at + i * kGroup + 8 * SR);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t *w0 = kw[g * PG], *w1 = kw[g * PG + PG - 1];
        // 4 bits: halves 0, 2 then 1, 3 of the words; 8 bits: bytes 0, 1 of the first piece, then of the second
        constexpr int e1 = BITS == 4 ? 2 : 1, e2 = BITS == 4 ? 1 : 0, e3 = BITS == 4 ? 3 : 1;
        const uint32_t x[2][4] = {{open_key(w0[0], 0), open_key(w0[1], 0), open_key(w0[0], e1), open_key(w0[1], e1)},
                                  {open_key(w1[0], e2), open_key(w1[1], e2), open_key(w1[0], e3), open_key(w1[1], e3)}};
        const float ks[2] = {sc[i][0].get(g), sc[i][1].get(g)};
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          float a[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16_acc(a, x[0], qb[n][g][0]);
          mma_f16_acc(a, x[1], qb[n][g][1]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < QL; ++k) {
              const float y = PAIR ? a[2 * h] + a[2 * h + 1] * 0x1p-11f : a[2 * h + k];
              const float f = ks[h] * fac[n * QL + k][g];
              float& s = pr[i][n * QL + k][h];
              s = g ? s + f * y : f * y;
            }
        }
      }
    }
    if (!full) {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const uint32_t bits = live(i) >> r;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < NQ; ++t)
            if (!(bits >> (8 * h) & 1)) pr[i][t][h] = -INFINITY;
      }
    }
    if (scores) {
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        const int row = ODD ? 8 * (t >> 1) + 2 * c + (t & 1) : 4 * t + c;
        if (row < rows) {
          float* to = scores + row * p.score_ld + r;
#pragma unroll
          for (int i = 0; i < kGroups; ++i) {
            to[16 * i] = pr[i][t][0];
            to[16 * i + 8] = pr[i][t][1];
          }
        }
      }
    }
    float mx[NQ];
    bool rises = false;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      mx[t] = fmaxf(pr[0][t][0], pr[0][t][1]);
#pragma unroll
      for (int i = 1; i < kGroups; ++i) mx[t] = fmax3(mx[t], pr[i][t][0], pr[i][t][1]);
      rises |= mx[t] > m[t];
    }
    // m stands in all the lanes of a column, so that it rises for none of them alone
    if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int t = 0; t < NQ; ++t) mx[t] = fmaxf(mx[t], __shfl_xor_sync(0xffffffffu, mx[t], d));
      float a[NQ];
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        const float mn = fmaxf(m[t], mx[t]);
        a[t] = weight(m[t] - (mn == -INFINITY ? 0.f : mn));
        m[t] = mn;
        l[t] *= a[t];
      }
#pragma unroll
      for (int n = 0; n < NL; ++n)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[n][i][k] *= a[ODD ? 2 * n + (k & 1) : n];
    }
    float ms[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) ms[t] = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        float(&x)[2] = pr[i][t];
        x[0] = weight(x[0] - ms[t]);
        x[1] = weight(x[1] - ms[t]);
        l[t] += x[0] + x[1];
      }
      uint32_t vw[CH][2];
      pieces<true>(vw, base + i * kGroup + kValues);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t b[NL][NP][2];  // the weights, times the values' scales
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v = sc[i][h].get(G + g);
#pragma unroll
          for (int n = 0; n < NL; ++n) {
            uint32_t w[NP];
            parts(pr[i][n * QL][h] * v, pr[i][n * QL + QL - 1][h] * v, w);
#pragma unroll
            for (int k = 0; k < NP; ++k) b[n][k][h] = movmatrix_trans(w[k]);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // rows r and r + 8: halves 2 k and 2 k + 1 (4 bits), bytes 0 and 1 of piece k (8 bits)
          const uint32_t* w = vw[BITS == 4 ? g : 2 * g + k];
          const int e = BITS == 4 ? 2 * k : 0;
          const uint32_t x[4] = {open_value(w[0], e), open_value(w[0], e + 1), open_value(w[1], e), open_value(w[1], e + 1)};
#pragma unroll
          for (int n = 0; n < NL; ++n)
#pragma unroll
            for (int part = 0; part < NP; ++part) mma_bf16_acc(o[n][2 * g + k], x, b[n][part]);
        }
      }
    }
  }

  // This warp's (m, l) [ROWS][2] and o [rows][DH] into shared memory.
  ONE_DEVINL void leave(float* ml, float* so, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const int n = t / QL, h = t % QL, row = ODD ? 8 * n + 2 * c + h : 4 * n + c;
      float x = l[t];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      if (r == 0) {
        ml[2 * row] = m[t];
        ml[2 * row + 1] = x;
      }
      if (row >= rows) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // rows r and r + 8 of the tile
          const int d = BITS == 4 ? i / 2 * 32 + 4 * r + i % 2 * 2 + k : i * 16 + 2 * r + k;
          so[row * DH + d] = ODD ? o[n][i][2 * k + h] : o[n][i][2 * k] + o[n][i][2 * k + 1];
        }
    }
  }
};

}  // namespace one
