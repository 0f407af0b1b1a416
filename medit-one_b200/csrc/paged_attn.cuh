// Attention of one new token per sequence over a paged cache, split over the cache's length.
//
//   s_t = q . k_t * scale * log2(e)    m = max_t s_t    l = sum_t 2^(s_t - m)
//   o   = sum_t 2^(s_t - m) v_t / l    mass_t += 2^(s_t - m) / l, summed over a kv head's queries
//
// One pass over K and V with the running maximum and sum; parts of a sequence join by their (m, l, o).
// HBM bounds it: every K and V row is read once per query-head tile (up to 16 query heads in bf16, 4 in
// fp32), at 1 flop per byte and query head. Measured, of the measured copy rate: 64 ragged sequences up to
// 4096 slots, 12 heads x 64, bf16: 75 us, 84 %; 8 up to 32768, 8 heads x 128 of 4 queries: 98 us, 90 %, of
// 32 queries, two tiles: 184 us. Small batches are bound by a chain: lengths -> page numbers -> rows ->
// softmax -> join, 5 us for one sequence of 200 slots, one call after the other.
//
// Partition. Few or short segments (a segment: one sequence's tiles of 64 slots or more for one query-head
// tile) have a cluster of CTAs each, and one launch. Otherwise the work is the list of all segments' tiles
// in order; a grid that fills the GPU takes equal shares of that list, whatever the lengths, so a ragged
// batch and a few long sequences keep all SMs busy. A share is a run of pieces of segments. A piece that
// is its whole segment is finished on the spot; the others leave (m, l, o) in the workspace, and
// paged_join_kernel joins them in a fixed order (no atomics: equal inputs give equal bits).
//
// Inside a CTA, each of four warps owns a quarter of a tile (groups of 16 slots) and a ring of stages
// in shared memory that its own cp.async fill in the order of the matrix fragments: the ring needs no
// barrier between warps, bytes in flight do not cost registers, and it runs across segment boundaries.
#pragma once

#include <utility>

#include "paged.cuh"

namespace one {

constexpr int kPaWarps = 4;
constexpr size_t kSmPerSm = 228 * 1024;    // shared memory of an SM, 1 KB of it per CTA reserved
constexpr int kMaxSms = 160;            // SMs that share a list, at most
constexpr int kPaPerSm = 3;             // CTAs of these kernels on an SM, at most

struct PagedAttn {
  PagedCache c;
  const void* q;
  int64_t q_bs, q_hs;
  int G, hv_per_kv;       // query heads per kv head; query-head tiles per kv head
  int q_vec;              // q rows may be read 16 bytes at a time
  uint32_t div_m;         // t / page_size = t * div_m >> div_s for t < 2^31
  int div_s;
  float scale_log2;
  float* mass;
  int64_t mass_width;
  void* out;              // [B][Hq][Dh]
  float* part_ml;         // [2 * ranges][rows][2]
  float* part_o;          // [2 * ranges][rows][DH]
  float* row_ml;          // [B * Hq][2], of segments in one piece
  float* scores;          // [B * Hq][score_ld], log2 domain
  int64_t score_ld;
  int2* parts;            // [B * Hkv * hv_per_kv]: first CTA of a segment; last << 1 | (its first part is slot 1)
  int ranges;             // CTAs that share the list
  int cluster;            // CTAs per segment, where there is no list
};

template <int TILE>
ONE_DEVINL int pa_tiles(const PagedCache& c, int b) {
  return (paged_length(c, b, SITE_PAGED_ATTN) + TILE - 1) / TILE;
}

// Tiles in the list (the host keeps them, rounded up to shares, below 2^31). Every warp computes them for itself.
template <int TILE>
ONE_DEVINL int pa_total(const PagedAttn& p) {
  int n = 0;
  for (int b = threadIdx.x & 31; b < p.c.B; b += 32) n += pa_tiles<TILE>(p.c, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * p.c.Hkv * p.hv_per_kv;
}

// A place in the list: tile `tile` of query-head tile gi of kv head kv of sequence b; the heads' tiles
// of a sequence follow one another, ng query-head tiles per kv head.
template <int TILE>
struct PaCursor {
  int b, kv, gi, tile, tiles, len;
  ONE_DEVINL void load(const PagedCache& c) {
    len = b < c.B ? paged_length(c, b, SITE_PAGED_ATTN) : 0;
    tiles = (len + TILE - 1) / TILE;
  }
  ONE_DEVINL void seek(const PagedCache& c, int ng, int w) {
    const int HV = c.Hkv * ng, lane = threadIdx.x & 31;
    for (int base = 0; base < c.B; base += 32) {
      const int n = base + lane < c.B ? pa_tiles<TILE>(c, base + lane) : 0;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, w < HV * incl);
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = base + src;
        w -= HV * __shfl_sync(0xffffffffu, incl - n, src);
        load(c);
        const int hv = w / tiles;
        tile = w - hv * tiles;
        kv = hv / ng;
        gi = hv - kv * ng;
        return;
      }
      w -= HV * __shfl_sync(0xffffffffu, incl, 31);
    }
    b = c.B;
    kv = gi = tile = tiles = len = 0;
  }
  // Returns whether this is another segment.
  ONE_DEVINL bool next(const PagedCache& c, int ng) {
    if (++tile < tiles) return false;
    tile = 0;
    if (++gi < ng) return true;
    gi = 0;
    if (++kv < c.Hkv) return true;
    kv = 0;
    do {
      ++b;
      load(c);
    } while (tiles == 0 && b < c.B);
    return true;
  }
};

// cp.async that writes zeros when there is nothing to read
ONE_DEVINL void cp_async16_or_zero(void* smem, const void* gmem, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(there ? 16 : 0) : "memory");
}
// 16 bytes from g + GO to shared address s + SO; the offsets are part of the instruction
template <int SO, int GO>
ONE_DEVINL void cp_async16_at(uint32_t s, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(s), "l"(g), "n"(SO), "n"(GO) : "memory");
}
// f(0), f(1), .. as compile-time constants
template <typename F, int... I>
ONE_DEVINL void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
ONE_DEVINL void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}
ONE_DEVINL void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The copies of a group's 16 rows, in pieces of 16 bytes, CH of them per row. Consecutive lanes take
// consecutive pieces, and D::at(row, piece), where a piece goes, keeps a 128-byte line of a row in one
// 128-byte line of shared memory with its pieces permuted, which spreads the fragments' reads over
// the banks. (Pieces that go to lines of their own are asked for one by one, and each 32-byte sector
// twice: that read 1.5 times the bytes into the SMs and took 96 us where this took 80, at 64 x 4096
// ragged tokens.) D::at is linear over exclusive or, so the unrolled loop splits it into a lane's
// constant and a compile-time one.
template <typename D, int CH>
struct PaCopy {
  static constexpr int N = 16 * CH / 32;
  // 16 whole rows that follow one another in memory, from this lane's first piece on
  ONE_DEVINL static void full(uint32_t to, const uint8_t* from) {
    const int lane = threadIdx.x & 31;
    if constexpr (32 % CH == 0) {
      const uint32_t mine = D::at(lane / CH, lane % CH);
      static_for<N>([&](auto n) {
        constexpr int k = decltype(n)::value, at = D::at(k * 32 / CH, 0);
        cp_async16_at<(at & ~127), k * 512>(to + (mine ^ (at & 127)), from);
      });
    } else {
      static_for<N>([&](auto n) {
        constexpr int k = decltype(n)::value;
        const int e = k * 32 + lane;
        cp_async16_at<0, k * 512>(to + D::at(e / CH, e % CH), from);
      });
    }
  }
  // the first `live` of such rows, the rest as zeros
  ONE_DEVINL static void some(uint8_t* to, const uint8_t* from, int live) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = k * 32 + lane, row = e / CH, ch = e % CH;
      cp_async16_or_zero(to + D::at(row, ch), from + k * 512, row < live);
    }
  }
  // rows anywhere: lane first + t holds the byte offset of row t, or -1
  ONE_DEVINL static void any(uint8_t* to, const uint8_t* base, int64_t off, int first, int pieces) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = k * 32 + lane, row = e / CH, ch = e % CH;
      const int64_t at = __shfl_sync(0xffffffffu, off, first + row);
      const bool there = at >= 0 && ch < pieces;
      cp_async16_or_zero(to + D::at(row, ch), base + (there ? at + ch * 16 : 0), there);
    }
  }
};

// ------------------------------------------------------------------ bf16: matrix instructions
// m16n8k16 with the query heads as the 16 rows. Sums over the head dim and over slots do not depend
// on the order of their terms, so the fragments are assigned to make every shared-memory access a
// lane's own 16 bytes (r = lane / 4, c = lane % 4):
//   S = Q K^T  the lane's B operand for key column r is pieces c + 4 i of a key row, as they lie in
//              memory; Q is read the same way. Column r of key tile j is slot 4 (r / 2) + 2 j + r % 2,
//   O += P V   so that the lane's four scores are slots 4 c .. 4 c + 3, and its B operand pairs
//              those four value rows: piece r (+ 8 i) of each, interleaved in registers. Column r of
//              value tile j is dim 8 r + j. The last 32 dims of DH = 32 and 96 go by half pieces:
//              dim 4 r + j.
// P enters as a bf16 high part plus the bf16 rounding of the remainder (16 significant bits; bf16
// alone would double the output's rounding error). Up to 8 query heads take rows 0-7 and the low
// parts ride in rows 8-15 of the same instruction; 9 to 16 heads (WIDE) take a second instruction.
template <int DH_, bool WIDE>
struct PaBf16 {
  using T = __nv_bfloat16;
  static constexpr int DH = DH_, ROWS = WIDE ? 16 : 8;
  static constexpr int KC = DH / 32;                   // 16-byte chunks of a key row per lane
  static constexpr int VC = DH / 64, VH = DH % 64 / 32;  // 16-byte and 8-byte pieces of a value row per lane
  static constexpr int NT = DH / 8;                    // value tiles
  static constexpr int kGroups = DH <= 64 ? 128 / DH : 1;  // 16-slot groups per warp and step
  static constexpr int TILE = 16 * kGroups * kPaWarps;
  static constexpr int kGroup = 64 * DH;               // bytes of a group's keys and values
  static constexpr int kStages = 2, kStagesFew = 3;    // where CTAs fill the SMs; where they are few
  static constexpr int kExtra = 0;                     // further shared bytes per warp
  ONE_DEVINL static float weight(float x) { return ex2_approx(x); }  // 2^x as consume computes it
  uint32_t qa[WIDE ? 2 : 1][KC][4];
  float o[NT][4];
  float m[2], l[2];  // rows r and r + 8

  static constexpr int CH = DH / 8;                    // pieces of a row
  // piece ch of row `row`: by lines of 64 dims, then the last 32 dims
  struct KTo {
    __host__ __device__ static constexpr int at(int row, int ch) {
      return ch < 8 * VC ? (ch >> 3) * 2048 + row * 128 + ((ch & 7) ^ (row & 1) << 2) * 16 : VC * 2048 + row * 64 + (ch - 8 * VC) * 16;
    }
  };
  struct VTo {
    __host__ __device__ static constexpr int at(int row, int ch) {
      return ch < 8 * VC ? (ch >> 3) * 2048 + row * 128 + ((ch & 7) ^ row >> 2 << 1) * 16
                         : VC * 2048 + ((row & 3) * 4 + (row >> 2)) * 64 + ((ch - 8 * VC) ^ row >> 3 << 1) * 16;
    }
  };
  static constexpr int kValues = 32 * DH;  // where a group's values start
  // 16 slots anywhere: lane t holds the element offset of slot t's key, lane 16 + t that of its value,
  // or -1.
  using Keys = PaCopy<KTo, CH>;
  using Values = PaCopy<VTo, CH>;
  ONE_DEVINL static void issue_any(uint8_t* stage, const T* keys, const T* values, int64_t off, int Dh) {
    const int64_t at = off < 0 ? -1 : off * (int)sizeof(T);
    Keys::any(stage, (const uint8_t*)keys, at, 0, Dh / 8);
    Values::any(stage + kValues, (const uint8_t*)values, at, 16, Dh / 8);
  }

  ONE_DEVINL void begin(const PagedAttn& p, uint8_t*, const T* q, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int w = 0; w < (WIDE ? 2 : 1); ++w)
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const int d = (c + 4 * i) * 8;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r + 8 * w < rows && d < p.c.Dh) {
          const T* x = q + (r + 8 * w) * p.q_hs + d;
          if (p.q_vec) {
            u = *reinterpret_cast<const uint4*>(x);
          } else {
            const uint16_t* y = reinterpret_cast<const uint16_t*>(x);
            u = make_uint4(y[0] | y[1] << 16, y[2] | y[3] << 16, y[4] | y[5] << 16, y[6] | y[7] << 16);
          }
        }
        qa[w][i][0] = u.x; qa[w][i][1] = u.y; qa[w][i][2] = u.z; qa[w][i][3] = u.w;
      }
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }

  // kGroups x 16 slots; live: a bit per slot of each group. scores: row 0's scores of these slots, or
  // null.
  ONE_DEVINL void consume(const PagedAttn& p, const uint8_t* stage, const uint32_t (&live)[kGroups], float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    constexpr int RW = WIDE ? 2 : 1;
    float pr[kGroups][RW][4];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if (live[g]) {
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 k = *reinterpret_cast<const uint4*>(stage + g * kGroup + KTo::at(4 * (r >> 1) + 2 * j + (r & 1), c + 4 * i));
            mma_bf16_16816(s[j], qa[0][i][0], WIDE ? qa[WIDE][i][0] : 0, qa[0][i][1], WIDE ? qa[WIDE][i][1] : 0, k.x, k.y);
            mma_bf16_16816(s[j], qa[0][i][2], WIDE ? qa[WIDE][i][2] : 0, qa[0][i][3], WIDE ? qa[WIDE][i][3] : 0, k.z, k.w);
          }
      }
#pragma unroll
      for (int w = 0; w < RW; ++w)
#pragma unroll
        for (int t = 0; t < 4; ++t) pr[g][w][t] = s[t >> 1][2 * w + (t & 1)] * p.scale_log2;
      if (live[g] != 0xffffu) {
        const uint32_t mine = live[g] >> (4 * c);
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (!(mine >> t & 1)) pr[g][w][t] = -INFINITY;
      }
      if (scores) {
#pragma unroll
        for (int w = 0; w < RW; ++w)
          if (r + 8 * w < rows)
            *reinterpret_cast<float4*>(scores + (r + 8 * w) * p.score_ld + 16 * g + 4 * c) =
                make_float4(pr[g][w][0], pr[g][w][1], pr[g][w][2], pr[g][w][3]);
      }
    }
    float mx[RW];
    bool rises = false;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      mx[w] = pr[0][w][0];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        mx[w] = fmax3(mx[w], pr[g][w][0], pr[g][w][1]);
        mx[w] = fmax3(mx[w], pr[g][w][2], pr[g][w][3]);
      }
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
      rises |= mx[w] > m[w];
    }
    if (__any_sync(0xffffffffu, rises)) {
      float a[2];
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        const float mn = fmaxf(m[w], mx[w]);
        a[w] = ex2_approx(m[w] - (mn == -INFINITY ? 0.f : mn));
        m[w] = mn;
        l[w] *= a[w];
      }
      if (!WIDE) a[1] = a[0];  // the low parts
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] *= a[0]; o[i][1] *= a[0]; o[i][2] *= a[1]; o[i][3] *= a[1];
      }
    }
    float ms[RW];
#pragma unroll
    for (int w = 0; w < RW; ++w) ms[w] = m[w] == -INFINITY ? 0.f : m[w];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (!live[g]) continue;
      uint32_t hi[RW][2], lo[RW][2];
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        float (&x)[4] = pr[g][w];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = ex2_approx(x[t] - ms[w]);
        l[w] += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          hi[w][h] = pack_bf16x2(x[2 * h], x[2 * h + 1]);
          lo[w][h] = pack_bf16x2(x[2 * h] - bf2_lo(hi[w][h]), x[2 * h + 1] - bf2_hi(hi[w][h]));
        }
      }
      const uint8_t* vs = stage + g * kGroup + 32 * DH;
      auto pv = [&](int tile, uint32_t b0, uint32_t b1) {
        if (WIDE) {
          mma_bf16_16816(o[tile], hi[0][0], hi[RW - 1][0], hi[0][1], hi[RW - 1][1], b0, b1);
          mma_bf16_16816(o[tile], lo[0][0], lo[RW - 1][0], lo[0][1], lo[RW - 1][1], b0, b1);
        } else {
          mma_bf16_16816(o[tile], hi[0][0], lo[0][0], hi[0][1], lo[0][1], b0, b1);
        }
      };
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        uint4 v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const uint4*>(vs + VTo::at(4 * c + t, r + 8 * i));
        const uint32_t x[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                  {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pv(8 * i + 2 * e, __byte_perm(x[0][e], x[1][e], 0x5410), __byte_perm(x[2][e], x[3][e], 0x5410));
          pv(8 * i + 2 * e + 1, __byte_perm(x[0][e], x[1][e], 0x7632), __byte_perm(x[2][e], x[3][e], 0x7632));
        }
      }
      if (VH) {
        uint2 v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const uint2*>(vs + VTo::at(4 * c + t, 8 * VC + (r >> 1)) + (r & 1) * 8);
        const uint32_t x[4][2] = {{v[0].x, v[0].y}, {v[1].x, v[1].y}, {v[2].x, v[2].y}, {v[3].x, v[3].y}};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pv(8 * VC + 2 * e, __byte_perm(x[0][e], x[1][e], 0x5410), __byte_perm(x[2][e], x[3][e], 0x5410));
          pv(8 * VC + 2 * e + 1, __byte_perm(x[0][e], x[1][e], 0x7632), __byte_perm(x[2][e], x[3][e], 0x7632));
        }
      }
    }
  }

  // This warp's (m, l) [ROWS][2] and o [rows][DH] into shared memory.
  ONE_DEVINL void leave(float* ml, float* so, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int w = 0; w < (WIDE ? 2 : 1); ++w) {
      float t = l[w];
      t += __shfl_xor_sync(0xffffffffu, t, 1);
      t += __shfl_xor_sync(0xffffffffu, t, 2);
      if (c == 0) {
        ml[2 * (r + 8 * w)] = m[w];
        ml[2 * (r + 8 * w) + 1] = t;
      }
      if (r + 8 * w >= rows) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x = WIDE ? o[i][2 * w + h] : o[i][h] + o[i][2 + h];
          const int col = 2 * c + h;
          const int d = i < 8 * VC ? (i / 8) * 64 + col * 8 + i % 8 : VC * 64 + col * 4 + (i - 8 * VC);
          so[(r + 8 * w) * DH + d] = x;
        }
    }
  }
};

// ------------------------------------------------------------------ fp32: FMA units
// ROWS query heads, 1 or 4. Scores: lane (r, c) takes slots r and r + 8 and every fourth 16-byte piece
// of their keys, for all heads; the sums over c are exchanged so that lane c ends with head c (one
// head: every lane with its score). Weighted sum: the weights pass through shared memory, a lane owns
// the dims lane + 32 i.
template <int DH_, int ROWS_>
struct PaF32 {
  using T = float;
  static constexpr int DH = DH_, ROWS = ROWS_;
  static constexpr int KC = DH / 16, VC = DH / 32, CH = DH / 4;
  static constexpr int kGroups = 1, TILE = 16 * kPaWarps;
  static constexpr int kGroup = 128 * DH;
  static constexpr int kValues = 64 * DH;
  static constexpr int kStages = DH == 32 ? 4 : DH == 96 ? 2 : 3, kStagesFew = kStages;
  static constexpr int kExtra = ROWS * DH * 4 + 16 * ROWS * 4;  // q [ROWS][DH], weights [16][ROWS]
  ONE_DEVINL static float weight(float x) { return exp2f(x); }   // 2^x as consume computes it
  float o[ROWS][VC];
  float m, l;  // of head c
  float *qs, *ps;

  struct KTo {
    __host__ __device__ static constexpr int at(int row, int ch) {
      return (ch >> 3) * 2048 + row * 128 + ((ch & 7) ^ (row & 1) << 2) * 16;
    }
  };
  struct VTo {
    __host__ __device__ static constexpr int at(int row, int ch) { return (row * CH + ch) * 16; }
  };
  using Keys = PaCopy<KTo, CH>;
  using Values = PaCopy<VTo, CH>;
  ONE_DEVINL static void issue_any(uint8_t* stage, const T* keys, const T* values, int64_t off, int Dh) {
    const int64_t at = off < 0 ? -1 : off * (int)sizeof(T);
    Keys::any(stage, (const uint8_t*)keys, at, 0, Dh / 4);
    Values::any(stage + kValues, (const uint8_t*)values, at, 16, Dh / 4);
  }

  ONE_DEVINL void begin(const PagedAttn& p, uint8_t* extra, const T* q, int rows) {
    const int lane = threadIdx.x & 31;
    qs = reinterpret_cast<float*>(extra);
    ps = qs + ROWS * DH;
    __syncwarp();
    for (int i = lane; i < ROWS * DH; i += 32) {
      const int g = i / DH, d = i % DH;
      qs[i] = g < rows && d < p.c.Dh ? q[g * p.q_hs + d] : 0.f;
    }
    __syncwarp();
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int g = 0; g < ROWS; ++g)
#pragma unroll
      for (int i = 0; i < VC; ++i) o[g][i] = 0.f;
  }

  ONE_DEVINL void consume(const PagedAttn& p, const uint8_t* stage, const uint32_t (&lives)[1], float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const uint32_t live = lives[0];
    if (!live) {  // nothing was copied; here for the scores alone
      if (c < rows) scores[c * p.score_ld + r] = scores[c * p.score_ld + r + 8] = -INFINITY;
      return;
    }
    float s[2][ROWS];
#pragma unroll
    for (int g = 0; g < ROWS; ++g) s[0][g] = s[1][g] = 0.f;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(stage + KTo::at(r, c + 4 * i));
      const float4 b = *reinterpret_cast<const float4*>(stage + KTo::at(r + 8, c + 4 * i));
#pragma unroll
      for (int g = 0; g < ROWS; ++g) {
        const float4 q = *reinterpret_cast<const float4*>(qs + g * DH + (c + 4 * i) * 4);
        s[0][g] += q.x * a.x + q.y * a.y + q.z * a.z + q.w * a.w;
        s[1][g] += q.x * b.x + q.y * b.y + q.z * b.z + q.w * b.w;
      }
    }
    float x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (ROWS == 4) {  // lane c keeps head c
        const float k0 = c & 2 ? s[j][2] : s[j][0], k1 = c & 2 ? s[j][3] : s[j][1];
        const float g0 = c & 2 ? s[j][0] : s[j][2], g1 = c & 2 ? s[j][1] : s[j][3];
        const float y0 = k0 + __shfl_xor_sync(0xffffffffu, g0, 2), y1 = k1 + __shfl_xor_sync(0xffffffffu, g1, 2);
        x[j] = (c & 1 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, c & 1 ? y0 : y1, 1);
      } else {
        x[j] = s[j][0] + __shfl_xor_sync(0xffffffffu, s[j][0], 2);
        x[j] += __shfl_xor_sync(0xffffffffu, x[j], 1);
      }
      x[j] = live >> (r + 8 * j) & 1 ? x[j] * p.scale_log2 : -INFINITY;
      if (scores && c < rows) scores[c * p.score_ld + r + 8 * j] = x[j];
    }
    float mx = fmaxf(x[0], x[1]);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if (__any_sync(0xffffffffu, mx > m)) {
      const float mn = fmaxf(m, mx);
      const float a = exp2f(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= a;
#pragma unroll
      for (int g = 0; g < ROWS; ++g) {
        const float ag = ROWS == 1 ? a : __shfl_sync(0xffffffffu, a, g);
#pragma unroll
        for (int i = 0; i < VC; ++i) o[g][i] *= ag;
      }
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[j] = exp2f(x[j] - ms);
      l += x[j];
      if (c < ROWS) ps[(r + 8 * j) * ROWS + c] = x[j];
    }
    __syncwarp();
    const float* vs = reinterpret_cast<const float*>(stage + kValues);
#pragma unroll
    for (int t0 = 0; t0 < 16; t0 += 4) {
      float w[4][ROWS];
#pragma unroll
      for (int t = 0; t < 4 * ROWS; t += 4) *reinterpret_cast<float4*>(&w[0][0] + t) = *reinterpret_cast<const float4*>(ps + t0 * ROWS + t);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          const float v = vs[(t0 + t) * DH + lane + 32 * i];
#pragma unroll
          for (int g = 0; g < ROWS; ++g) o[g][i] += w[t][g] * v;
        }
    }
    __syncwarp();
  }

  ONE_DEVINL void leave(float* ml, float* so, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    float t = l;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (r == 0 && c < ROWS) {
      ml[2 * c] = m;
      ml[2 * c + 1] = t;
    }
#pragma unroll
    for (int g = 0; g < ROWS; ++g)
#pragma unroll
      for (int i = 0; i < VC; ++i)
        if (g < rows) so[g * DH + lane + 32 * i] = o[g][i];
  }
};

ONE_DEVINL void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
ONE_DEVINL uint32_t cluster_at(const void* mine, int rank) {
  uint32_t far;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(smem_u32(mine)), "r"(rank));
  return far;
}
// what CTA `rank` of the cluster has where this one has `mine`
ONE_DEVINL float2 cluster_ld2(const float* mine, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_at(mine, rank)) : "memory");
  return v;
}
ONE_DEVINL float4 cluster_ld4(const float* mine, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_at(mine, rank))
               : "memory");
  return v;
}

// What a CTA takes: a share of the list; a segment, or its share of a cluster's; the same with a deeper ring.
enum PaMode { PA_LIST, PA_SEGMENT, PA_DEEP };

template <typename E, PaMode MODE>
struct PaSmem {
  static constexpr bool SPLIT = MODE == PA_LIST;
  static constexpr int kStage = E::kGroup * E::kGroups;                  // bytes per warp
  static constexpr int kStages = MODE == PA_DEEP ? E::kStagesFew : E::kStages;
  static constexpr int kWarp = kStage * kStages;
  static constexpr int kML = kPaWarps * kWarp;                           // [2][warps][ROWS][2]
  static constexpr int kFin = kML + 2 * kPaWarps * E::ROWS * 8;          // [ROWS][2]: m, 1 / l
  static constexpr int kExtra = kFin + (E::ROWS * 8 + 15) / 16 * 16;
  static constexpr int kSum = kExtra + kPaWarps * E::kExtra;
  // of a cluster: this CTA's sums [ROWS][DH]; of a list: the warps' sums [1 or 2][warps][rows][DH] where they fit
  static constexpr int kApart = 2 * kPaWarps * E::ROWS * E::DH * 4 < 9216 ? 2 * kPaWarps * E::ROWS * E::DH * 4 : 9216;
  static constexpr int kTotal = kSum + (SPLIT ? kApart : E::ROWS * E::DH * 4);
  static constexpr int kPerSm = kSmPerSm / (kTotal + 1024) < 3 ? kSmPerSm / (kTotal + 1024) : 3;
  // a warp's sums fit the stage that it consumed last
  static_assert(kStage >= E::ROWS * E::DH * 4, "stage");
};

// PA_LIST: CTA i takes the i-th share of the list. Otherwise a cluster of p.cluster CTAs (1 to 8) takes
// each segment, in equal shares, and joins them through its shared memory: one launch, for small batches.
// RUN: pages hold a multiple of 16 slots and Dh is E::DH, so that a group lies in one page and its copies
// need two addresses.
template <typename E, bool RUN, PaMode MODE>
__global__ void __launch_bounds__(kPaWarps * 32, PaSmem<E, MODE>::kPerSm) paged_attn_kernel(const __grid_constant__ PagedAttn p) {
  extern __shared__ __align__(16) uint8_t smem[];
  using S = PaSmem<E, MODE>;
  constexpr bool SPLIT = S::SPLIT;
  using T = typename E::T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int TILE = E::TILE, GR = E::kGroups;
  uint8_t* ring = smem + warp * S::kWarp;
  float* fin = reinterpret_cast<float*>(smem + S::kFin);
  uint8_t* extra = smem + S::kExtra + warp * E::kExtra;
  const PagedCache& c = p.c;
  const int ng = p.hv_per_kv;
  pdl_wait();
  pdl_launch_dependents();
  PaCursor<TILE> cur;
  int left, share = 0;  // tiles to do; a full share
  if (SPLIT) {
    const int total = pa_total<TILE>(p);
    share = max(1, (total + p.ranges - 1) / p.ranges);
    const long long w0 = (long long)share * blockIdx.x;
    if (w0 >= total) return;
    left = min(share, total - (int)w0);
    cur.seek(c, ng, (int)w0);
  } else {
    const int seg = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster, HV = c.Hkv * ng;
    cur.b = seg / HV;
    cur.kv = (seg - cur.b * HV) / ng;
    cur.gi = seg % ng;
    cur.load(c);
    cur.tile = (int)((int64_t)cur.tiles * rank / p.cluster);
    left = (int)((int64_t)cur.tiles * (rank + 1) / p.cluster) - cur.tile;
  }
  // ---- the copying side: page numbers are asked for one tile ahead of the copies. RUN: one per group;
  //      otherwise lane t and lane 16 + t look slot t up.
  PaCursor<TILE> src = cur;
  int to_copy = left, pg[GR], row[GR];  // page and first element in its head of each group
  uint32_t live[S::kStages][GR];        // slots in use of the tiles in the ring, the oldest first
#pragma unroll
  for (int k = 0; k < S::kStages; ++k)
#pragma unroll
    for (int g = 0; g < GR; ++g) live[k][g] = 0;
  const int mine = warp * (16 * GR) + (RUN ? 0 : lane & 15);
  const int* table;          // of the segment being copied:
  const T *keys, *values;    // its block table, and its head in page 0 (RUN: this lane's first piece)
  auto segment = [&] {
    const int64_t head = (int64_t)src.kv * c.page_size * c.Dh + (RUN ? lane * (int)(16 / sizeof(T)) : 0);
    table = c.table + src.b * c.table_stride;
    keys = (const T*)c.k + head;
    values = (const T*)c.v + head;
  };
  int ahead = src.len - src.tile * TILE - mine;  // slots from this warp's first one to the end
  auto ask = [&] {
    const int t0 = src.len - ahead;
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      pg[g] = -1;
      if (ahead > 16 * g) {
        const int t = t0 + 16 * g, index = (int)(((uint64_t)(uint32_t)t * p.div_m) >> p.div_s);
        row[g] = (t - index * c.page_size) * c.Dh;
        pg[g] = table[index];
      }
    }
  };
  const int ks = (int)c.k_stride, vs = (int)c.v_stride;
  uint32_t put = 0, get = 0;  // byte offsets of stages
  auto copy = [&] {
#pragma unroll
    for (int k = 0; k + 1 < S::kStages; ++k)
#pragma unroll
      for (int g = 0; g < GR; ++g) live[k][g] = live[k + 1][g];
    if (to_copy > 0) {
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        uint8_t* to = ring + put + g * E::kGroup;
        uint32_t& alive = live[S::kStages - 1][g];
        const bool good = (uint32_t)pg[g] < (uint32_t)c.num_pages;
        if (!good && ahead > 16 * g) set_err(c.err, ERR_BAD_ARG, SITE_PAGED_ATTN);
        if (RUN) {
          alive = 0;
          if (good) {
            const uint8_t* kp = (const uint8_t*)(keys + ((int64_t)pg[g] * ks + row[g]));
            const uint8_t* vp = (const uint8_t*)(values + ((int64_t)pg[g] * vs + row[g]));
            if (ahead >= 16 * g + 16) {
              alive = 0xffffu;
              E::Keys::full(smem_u32(to), kp);
              E::Values::full(smem_u32(to) + E::kValues, vp);
            } else {
              const int n = ahead - 16 * g;
              alive = (1u << n) - 1;
              E::Keys::some(to, kp, n);
              E::Values::some(to + E::kValues, vp, n);
            }
          }
        } else {
          const int64_t off = !good ? -1 : lane < 16 ? (int64_t)pg[g] * ks + row[g] : (int64_t)pg[g] * vs + row[g];
          alive = __ballot_sync(0xffffffffu, good) & 0xffffu;
          if (alive) E::issue_any(to, keys, values, off, c.Dh);
        }
      }
      if (--to_copy > 0) {
        ahead -= TILE;
        if (src.next(c, ng)) {
          segment();
          ahead = src.len - src.tile * TILE - mine;
        }
        ask();
      }
    }
    cp_async_commit();
    put = put + S::kStage == S::kWarp ? 0 : put + S::kStage;
  };
  segment();
  if (to_copy == 0) ahead = 0;
  ask();
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) copy();
  // ---- the computing side, piece by piece. At a piece's end the warps' sums go through shared memory. In
  //      a list, where there is room for a piece's sums, the copies go on meanwhile, and where there is room
  //      for two pieces' one barrier per piece is enough; otherwise the sums go where each warp consumed
  //      last, the stage filled next. (64 ragged sequences of up to 4096 slots: 78.6 us with the copies
  //      held up at each end, 74.9 as here; up to 1024: 36.8, 30.8.)
  E eng;
  bool begun_inside = false, copied = false;  // the piece does not start this CTA's share; its first tile is on its way
  const int most = min(E::ROWS, p.G);
  const bool apart = SPLIT && kPaWarps * most * E::DH * 4 <= S::kApart;
  const bool twice = SPLIT && 2 * kPaWarps * most * E::DH * 4 <= S::kApart;
  int parity = 0;
  do {
    const int kv = cur.kv, g0 = cur.gi * E::ROWS, rows = min(E::ROWS, p.G - g0);
    const int64_t hq0 = ((int64_t)cur.b * c.Hkv + kv) * p.G + g0;  // output row of this query-head tile
    const int first = cur.tile, last = min(cur.tiles, cur.tile + left);
    if (SPLIT && (cur.b >= c.B || last <= first)) break;  // lengths that changed during the call
    eng.begin(p, extra, (const T*)p.q + cur.b * p.q_bs + ((int64_t)kv * p.G + g0) * p.q_hs, rows);
    for (int tile = first; tile < last; ++tile) {
      if (!copied) copy();
      copied = false;
      cp_async_wait<S::kStages - 1>();
      uint32_t any = 0;
#pragma unroll
      for (int g = 0; g < GR; ++g) any |= live[0][g];
      __syncwarp();
      if (any || p.scores)
        eng.consume(p, ring + get, live[0], p.scores ? p.scores + hq0 * p.score_ld + tile * TILE + warp * (16 * GR) : nullptr, rows);
      __syncwarp();
      get = get + S::kStage == S::kWarp ? 0 : get + S::kStage;
      if (apart && tile + 1 == last) {
        copy();
        copied = true;
      }
    }
    float* so = reinterpret_cast<float*>(smem + (apart ? S::kSum : put));
    const int so_warp = apart ? most * E::DH : S::kWarp / 4;
    if (apart) so += parity * kPaWarps * so_warp;
    float* ml = reinterpret_cast<float*>(smem + S::kML) + parity * kPaWarps * E::ROWS * 2;
    eng.leave(ml + warp * E::ROWS * 2, so + warp * so_warp, rows);
    __syncthreads();
    const bool whole = first == 0 && last == cur.tiles;
    if (SPLIT && first == 0 && threadIdx.x == 0) {  // which CTAs hold this segment: tiles from `left` on go to later ones
      const int more = (cur.tiles - left + share - 1) / share;
      p.parts[(cur.b * c.Hkv + cur.kv) * ng + cur.gi] =
          make_int2((int)blockIdx.x, ((int)blockIdx.x + max(0, more)) << 1 | (int)begun_inside);
    }
    const int64_t part = 2ll * blockIdx.x + begun_inside;
    float* sum = reinterpret_cast<float*>(smem + S::kSum);
    for (int i = threadIdx.x; i < rows * (E::DH / 4); i += blockDim.x) {
      const int g = i / (E::DH / 4), d = i % (E::DH / 4) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < kPaWarps; ++k) M = fmaxf(M, ml[(k * E::ROWS + g) * 2]);
      const float Ms = M == -INFINITY ? 0.f : M;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kPaWarps; ++k) {
        const float f = exp2f(ml[(k * E::ROWS + g) * 2] - Ms);
        L += f * ml[(k * E::ROWS + g) * 2 + 1];
        const float4 x = *reinterpret_cast<const float4*>(so + k * so_warp + g * E::DH + d);
        a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
      }
      if (!SPLIT && p.cluster > 1) {
        *reinterpret_cast<float4*>(sum + g * E::DH + d) = a;
        if (d == 0) {
          fin[2 * g] = M;
          fin[2 * g + 1] = L;
        }
      } else if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (d < c.Dh) {
          T* y = (T*)p.out + (hq0 + g) * c.Dh + d;
          st<T>(y, a.x * inv); st<T>(y + 1, a.y * inv); st<T>(y + 2, a.z * inv); st<T>(y + 3, a.w * inv);
        }
        if (d == 0 && p.mass) {
          float* x = SPLIT ? p.row_ml + 2 * (hq0 + g) : fin + 2 * g;
          x[0] = Ms;
          x[1] = inv;
        }
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part * E::ROWS + g) * E::DH + d) = a;
        if (d == 0) {
          p.part_ml[(part * E::ROWS + g) * 2] = M;
          p.part_ml[(part * E::ROWS + g) * 2 + 1] = L;
        }
      }
    }
    if (twice) parity ^= 1;
    else __syncthreads();
    const float* joint = fin;  // m, 1 / l of the whole segment
    if (!SPLIT && p.cluster > 1) {
      cluster_sync();
      // thread t joins pieces of the rows; with mass, thread g the row g as well
      const int cs = p.cluster, rank = blockIdx.x % cs;
      auto row = [&](int g, float (&f)[8], float& inv) -> float {  // each CTA's weight over the joint l; returns m
        float2 x[8];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k >= cs) break;
          x[k] = cluster_ld2(fin + 2 * g, k);
          M = fmaxf(M, x[k].x);
        }
        if (M == -INFINITY) M = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k >= cs) break;
          f[k] = exp2f(x[k].x - M);
          L += f[k] * x[k].y;
        }
        inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] *= inv;
        return M;
      };
      for (int i = rank * kPaWarps * 32 + threadIdx.x; i < rows * (E::DH / 4); i += cs * kPaWarps * 32) {
        const int g = i / (E::DH / 4), d = i % (E::DH / 4) * 4;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        float inv;
        row(g, f, inv);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k >= cs) break;
          const float4 x = cluster_ld4(sum + g * E::DH + d, k);
          a.x += f[k] * x.x; a.y += f[k] * x.y; a.z += f[k] * x.z; a.w += f[k] * x.w;
        }
        if (d < c.Dh) {
          T* y = (T*)p.out + (hq0 + g) * c.Dh + d;
          st<T>(y, a.x); st<T>(y + 1, a.y); st<T>(y + 2, a.z); st<T>(y + 3, a.w);
        }
      }
      if (p.mass) {
        if (threadIdx.x < rows) {
          float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, inv;
          ml[2 * threadIdx.x] = row(threadIdx.x, f, inv);
          ml[2 * threadIdx.x + 1] = inv;
        }
        __syncthreads();
        joint = ml;
      }
    }
    if (!SPLIT && p.mass) {  // one query-head tile per kv head: this CTA wrote all the scores of its slots
      float* mass = p.mass + ((int64_t)cur.b * c.Hkv + kv) * p.mass_width;
      for (int t = first * TILE + threadIdx.x; t < min(last * TILE, cur.len); t += blockDim.x) {
        float a = 0.f;
        for (int g = 0; g < rows; ++g) a += E::weight(p.scores[(hq0 + g) * p.score_ld + t] - joint[2 * g]) * joint[2 * g + 1];
        mass[t] += a;
      }
    }
    if (!SPLIT && p.cluster > 1) cluster_sync();  // nobody leaves while its sums are read
    begun_inside = true;
    left -= last - first;
    cur.tile = last - 1;
    if (left > 0) cur.next(c, ng);
  } while (left > 0);
}

// Joins what paged_attn_kernel left of a split list: one output row per block, then, with mass, one
// block per 1024 slots of a (sequence, kv head), which adds the weights of all its query heads. Chains
// of three round trips to L2: which parts, their (m, l), their sums.
constexpr int kJoinThreads = 256;
constexpr int kJoinSlots = 4 * kJoinThreads;
constexpr int kJoinAhead = 4;

template <typename E>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttn p, int mass_blocks) {
  using T = typename E::T;
  constexpr int ROWS = E::ROWS, DH = E::DH;
  __shared__ float4 red[kJoinThreads];
  __shared__ float weight[kMaxSms * kPaPerSm];  // 2^(m - M) of each part
  __shared__ float fin[2][128];                 // M and 1 / l of a kv head's query heads
  const PagedCache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hq = c.Hkv * p.G, ng = p.hv_per_kv;
  pdl_wait();
  // slot of part i of the CTAs that hold a segment
  auto slot = [](int2 seg, int i) -> int64_t { return 2ll * i + (i == seg.x ? seg.y & 1 : 0); };
  // joint m and 1 / l of row g of a segment's parts, by one warp; w: the parts' weights
  auto joint = [&](int2 seg, int g, float& M, float& inv, float* w) {
    const int first = seg.x, last = seg.y >> 1;
    float mm = -INFINITY;
    for (int i = first + lane; i <= last; i += 32) mm = fmaxf(mm, p.part_ml[(slot(seg, i) * ROWS + g) * 2]);
    M = warp_max(mm);
    if (M == -INFINITY) M = 0.f;
    float L = 0.f;
    for (int i = first + lane; i <= last; i += 32) {
      const float2 x = *reinterpret_cast<const float2*>(p.part_ml + (slot(seg, i) * ROWS + g) * 2);
      const float f = exp2f(x.x - M);
      if (w) w[i - first] = f;
      L += x.y * f;
    }
    L = warp_sum(L);
    inv = L == 0.f ? 0.f : 1.f / L;
  };
  if ((int)blockIdx.x < c.B * hq) {
    const int b = blockIdx.x / hq, j = blockIdx.x % hq, kv = j / p.G, g = j % p.G, row = g % ROWS;
    const int2 seg = p.parts[(b * c.Hkv + kv) * ng + g / ROWS];
    T* out = (T*)p.out + (int64_t)blockIdx.x * c.Dh;
    if (paged_length(c, b, SITE_PAGED_ATTN) == 0) {  // no CTA holds it
      for (int d = tid; d < c.Dh; d += kJoinThreads) st<T>(out + d, 0.f);
      return;
    }
    const int first = seg.x, last = seg.y >> 1;
    if (first == last || first < 0 || last < first || last >= p.ranges) return;  // whole; lengths changed during the call
    constexpr int C4 = DH / 4, NG = kJoinThreads / C4;  // float4 columns; parts summed side by side
    const int col = tid % C4, grp = tid / C4;
    auto part = [&](int i) { return *reinterpret_cast<const float4*>(p.part_o + (slot(seg, i) * ROWS + row) * DH + col * 4); };
    float4 x[kJoinAhead];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k)
      if (grp < NG && first + grp + k * NG <= last) x[k] = part(first + grp + k * NG);
    float M, inv;
    if (warp == 0) {
      joint(seg, row, M, inv, weight);
      if (lane == 0) fin[0][0] = inv;
    }
    __syncthreads();
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = grp; grp < NG && first + i0 <= last; i0 += kJoinAhead * NG) {
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) {
        const int i = i0 + k * NG;
        if (first + i > last) break;
        const float f = weight[i];
        a.x += f * x[k].x; a.y += f * x[k].y; a.z += f * x[k].z; a.w += f * x[k].w;
        if (first + i + kJoinAhead * NG <= last) x[k] = part(first + i + kJoinAhead * NG);
      }
    }
    red[tid] = a;
    __syncthreads();
    if (tid < C4 && tid * 4 < c.Dh) {
      for (int k = 1; k < NG; ++k) {
        const float4 y = red[k * C4 + tid];
        a.x += y.x; a.y += y.y; a.z += y.z; a.w += y.w;
      }
      inv = fin[0][0];
      T* y = out + tid * 4;
      st<T>(y, a.x * inv); st<T>(y + 1, a.y * inv); st<T>(y + 2, a.z * inv); st<T>(y + 3, a.w * inv);
    }
    return;
  }
  // ---- mass: four slots per thread; rows of scores are padded, so that they may be read past the length
  const int at = blockIdx.x - c.B * hq, bh = at / mass_blocks, t = at % mass_blocks * kJoinSlots + tid * 4, b = bh / c.Hkv;
  const int len = paged_length(c, b, SITE_PAGED_ATTN);
  if (at % mass_blocks * kJoinSlots >= len) return;
  const int64_t row0 = (int64_t)bh * p.G;
  float add[4] = {0.f, 0.f, 0.f, 0.f};
  for (int gb = 0; gb < p.G; gb += 128) {
    const int gn = min(128, p.G - gb);
    if (gb) __syncthreads();
    for (int g = gb + warp; g < gb + gn; g += kJoinThreads / 32) {
      const int2 seg = p.parts[bh * ng + g / ROWS];
      float M, inv;
      if (seg.x == seg.y >> 1 || seg.x < 0 || seg.y < 0 || seg.y >> 1 >= p.ranges) {
        M = p.row_ml[2 * (row0 + g)];
        inv = p.row_ml[2 * (row0 + g) + 1];
      } else {
        joint(seg, g % ROWS, M, inv, nullptr);
      }
      if (lane == 0) {
        fin[0][g - gb] = M;
        fin[1][g - gb] = inv;
      }
    }
    __syncthreads();
    if (t < len) {
#pragma unroll 4
      for (int g = 0; g < gn; ++g) {
        const float4 s = *reinterpret_cast<const float4*>(p.scores + (row0 + gb + g) * p.score_ld + t);
        const float M = fin[0][g], inv = fin[1][g];
        add[0] += E::weight(s.x - M) * inv;
        add[1] += E::weight(s.y - M) * inv;
        add[2] += E::weight(s.z - M) * inv;
        add[3] += E::weight(s.w - M) * inv;
      }
    }
  }
  float* mass = p.mass + (int64_t)bh * p.mass_width + t;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t + k < len) mass[k] += add[k];
}

}  // namespace one
