// Attention of one new token per sequence over a paged cache, split over the cache's length.
//
//   s_t = q . k_t * scale * log2(e)    m = max_t s_t    l = sum_t 2^(s_t - m)
//   o   = sum_t 2^(s_t - m) v_t / l    mass_t += 2^(s_t - m) / l, summed over a kv head's queries
//
// One pass over K and V with the running maximum and sum; parts of a sequence join by their (m, l, o).
// HBM bounds it: every K and V row is read once, at 1 flop per byte and query head of a group.
//
// Partition. The work is the list of 64-slot tiles of every (sequence, query-head tile) in order; a
// grid that fills the GPU takes equal shares of that list, whatever the lengths, so a ragged batch
// and a single long sequence keep all SMs busy. A share is a run of pieces of segments (a segment:
// one sequence's tiles for one query-head tile). A piece that is its whole segment is finished on the
// spot; the others leave (m, l, o) in the workspace, and paged_join_kernel joins them in a fixed
// order (no atomics: equal inputs give equal bits).
//
// Inside a CTA, each of four warps owns 16 slots of a tile and a ring of stages in shared memory
// that cp.async fills with the lane's own matrix fragments: no lane reads what another one
// copied, so the ring needs no barrier, and bytes in flight do not cost registers. The ring runs
// across segment boundaries.
#pragma once

#include "paged.cuh"

namespace one {

constexpr int kPaWarps = 4;
constexpr int kPaTile = 16 * kPaWarps;  // slots per tile
constexpr size_t kSmPerSm = 228 * 1024;    // shared memory of an SM, 1 KB of it per CTA reserved
constexpr int kPaPerSm = 4;             // CTAs of these kernels on an SM, at most

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
  int ranges;             // CTAs that share the list
};

ONE_DEVINL int pa_tiles(const PagedCache& c, int b) { return (paged_length(c, b, SITE_PAGED_ATTN) + kPaTile - 1) / kPaTile; }

// The list's length and a position in it. Every warp computes them for itself.
ONE_DEVINL long long pa_total(const PagedAttn& p) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < p.c.B; b += 32) n += pa_tiles(p.c, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * p.c.Hkv * p.hv_per_kv;
}
// Tiles (of one query-head tile) of the sequences before `upto`.
ONE_DEVINL long long pa_before(const PagedAttn& p, int upto) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < upto; b += 32) n += pa_tiles(p.c, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}
ONE_DEVINL long long pa_chunk(const PagedAttn& p, long long total) { return max(1ll, (total + p.ranges - 1) / p.ranges); }

// A place in the list: tile `tile` of query-head tile hv of sequence b.
struct PaCursor {
  int b, hv, tile, tiles, len;
  ONE_DEVINL void load(const PagedCache& c) {
    len = b < c.B ? paged_length(c, b, SITE_PAGED_ATTN) : 0;
    tiles = (len + kPaTile - 1) / kPaTile;
  }
  ONE_DEVINL void seek(const PagedCache& c, int HV, long long w) {
    const int lane = threadIdx.x & 31;
    long long run = 0;
    for (int base = 0; base < c.B; base += 32) {
      const int n = base + lane < c.B ? pa_tiles(c, base + lane) : 0;
      long long incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, w < (long long)HV * (run + incl));
      if (hit) {
        const int src = __ffs(hit) - 1;
        b = base + src;
        const long long first = (long long)HV * (run + __shfl_sync(0xffffffffu, incl - n, src));
        load(c);
        hv = (int)((w - first) / tiles);
        tile = (int)((w - first) % tiles);
        return;
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    b = c.B;
    hv = tile = tiles = len = 0;
  }
  ONE_DEVINL void next(const PagedCache& c, int HV) {
    if (++tile < tiles) return;
    tile = 0;
    if (++hv < HV) return;
    hv = 0;
    do {
      ++b;
      load(c);
    } while (tiles == 0 && b < c.B);
  }
};

// cp.async that writes zeros when there is nothing to read
ONE_DEVINL void cp_async16_or_zero(void* smem, const void* gmem, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(there ? 16 : 0) : "memory");
}
ONE_DEVINL void cp_async8_or_zero(void* smem, const void* gmem, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(there ? 8 : 0) : "memory");
}
ONE_DEVINL void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ------------------------------------------------------------------ bf16: matrix instructions
// m16n8k16 with the query heads as the 16 rows. Sums over the head dim and over slots do not depend
// on the order of their terms, so the fragments are assigned to make every copy a lane's own 16
// bytes (r = lane / 4, c = lane % 4):
//   S = Q K^T  the lane's B operand for key column r is chunk c + 4 i of a key row, as it lies in
//              memory; Q is read the same way. Column r of key tile j is slot 4 (r / 2) + 2 j + r % 2,
//   O += P V   so that the lane's four scores are slots 4 c .. 4 c + 3, and its B operand pairs
//              those four value rows: chunk r (+ 8 i) of each, interleaved in registers. Column r of
//              value tile j is dim 8 r + j.
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
  static constexpr int kStage = 64 * DH;               // bytes per warp
  static constexpr int kStages = DH == 32 ? 6 : DH == 64 ? (WIDE ? 3 : 4) : DH == 96 ? (WIDE ? 3 : 4) : (WIDE ? 2 : 3);
  static constexpr int kExtra = 0;                     // further shared bytes per warp
  uint32_t qa[WIDE ? 2 : 1][KC][4];
  float o[NT][4];
  float m[2], l[2];  // rows r and r + 8

  ONE_DEVINL static void issue(const PagedAttn& p, uint8_t* stage, int64_t off, int chunks) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const T* kb = (const T*)p.c.k;
    const T* vb = (const T*)p.c.v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = __shfl_sync(0xffffffffu, off, 4 * (r >> 1) + 2 * j + (r & 1));
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const bool there = at >= 0 && c + 4 * i < chunks;
        cp_async16_or_zero(stage + ((j * KC + i) * 32 + lane) * 16, kb + (there ? at + (c + 4 * i) * 8 : 0), there);
      }
    }
    uint8_t* vs = stage + 32 * DH;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t at = __shfl_sync(0xffffffffu, off, 16 + 4 * c + t);
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const bool there = at >= 0 && r + 8 * i < chunks;
        cp_async16_or_zero(vs + ((t * VC + i) * 32 + lane) * 16, vb + (there ? at + (r + 8 * i) * 8 : 0), there);
      }
      if (VH) {
        const bool there = at >= 0 && 8 * VC + r / 2 < chunks;
        cp_async8_or_zero(vs + VC * 2048 + (t * 32 + lane) * 8, vb + (there ? at + VC * 64 + r * 4 : 0), there);
      }
    }
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

  // 16 slots; `live`: a bit per slot. scores: row 0's scores of these slots, or null.
  ONE_DEVINL void consume(const PagedAttn& p, const uint8_t* stage, uint32_t live, float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint4 k = *reinterpret_cast<const uint4*>(stage + ((j * KC + i) * 32 + lane) * 16);
        mma_bf16_16816(s[j], qa[0][i][0], WIDE ? qa[WIDE][i][0] : 0, qa[0][i][1], WIDE ? qa[WIDE][i][1] : 0, k.x, k.y);
        mma_bf16_16816(s[j], qa[0][i][2], WIDE ? qa[WIDE][i][2] : 0, qa[0][i][3], WIDE ? qa[WIDE][i][3] : 0, k.z, k.w);
      }
    }
    constexpr int RW = WIDE ? 2 : 1;
    float mx[2], pr[RW][4];
    const uint32_t mine = live >> (4 * c);
#pragma unroll
    for (int w = 0; w < RW; ++w) {
#pragma unroll
      for (int t = 0; t < 4; ++t) pr[w][t] = mine >> t & 1 ? s[t >> 1][2 * w + (t & 1)] * p.scale_log2 : -INFINITY;
      if (scores && r + 8 * w < rows)
        *reinterpret_cast<float4*>(scores + (r + 8 * w) * p.score_ld + 4 * c) = make_float4(pr[w][0], pr[w][1], pr[w][2], pr[w][3]);
      mx[w] = fmaxf(fmaxf(pr[w][0], pr[w][1]), fmaxf(pr[w][2], pr[w][3]));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 1));
      mx[w] = fmaxf(mx[w], __shfl_xor_sync(0xffffffffu, mx[w], 2));
    }
    bool rises = mx[0] > m[0];
    if (WIDE) rises |= mx[RW - 1] > m[1];
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
    uint32_t hi[RW][2], lo[RW][2];
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      const float ms = m[w] == -INFINITY ? 0.f : m[w];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        pr[w][t] = ex2_approx(pr[w][t] - ms);
        l[w] += pr[w][t];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        hi[w][h] = pack_bf16x2(pr[w][2 * h], pr[w][2 * h + 1]);
        lo[w][h] = pack_bf16x2(pr[w][2 * h] - bf2_lo(hi[w][h]), pr[w][2 * h + 1] - bf2_hi(hi[w][h]));
      }
    }
    const uint8_t* vs = stage + 32 * DH;
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
      for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const uint4*>(vs + ((t * VC + i) * 32 + lane) * 16);
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
      for (int t = 0; t < 4; ++t) v[t] = *reinterpret_cast<const uint2*>(vs + VC * 2048 + (t * 32 + lane) * 8);
      const uint32_t x[4][2] = {{v[0].x, v[0].y}, {v[1].x, v[1].y}, {v[2].x, v[2].y}, {v[3].x, v[3].y}};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pv(8 * VC + 2 * e, __byte_perm(x[0][e], x[1][e], 0x5410), __byte_perm(x[2][e], x[3][e], 0x5410));
        pv(8 * VC + 2 * e + 1, __byte_perm(x[0][e], x[1][e], 0x7632), __byte_perm(x[2][e], x[3][e], 0x7632));
      }
    }
  }

  // This warp's (m, l) [ROWS][2] and o [ROWS][DH] into shared memory.
  ONE_DEVINL void leave(float* ml, float* so) {
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
// Four query heads. Scores: lane (r, c) takes slots r and r + 8 and every fourth 16-byte chunk of
// their keys, for all four heads; the sums over c are exchanged so that lane c ends with head c.
// Weighted sum: the weights pass through shared memory, a lane owns the dims lane + 32 i.
template <int DH_>
struct PaF32 {
  using T = float;
  static constexpr int DH = DH_, ROWS = 4;
  static constexpr int KC = DH / 16, VC = DH / 32;
  static constexpr int kStage = 128 * DH;
  static constexpr int kStages = DH == 32 ? 4 : DH == 96 ? 2 : 3;
  static constexpr int kExtra = 4 * DH * 4 + 16 * 16;  // q [4][DH], weights [16][4]
  float o[4][VC];
  float m, l;  // of head c
  float *qs, *ps;

  ONE_DEVINL static void issue(const PagedAttn& p, uint8_t* stage, int64_t off, int chunks) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const T* kb = (const T*)p.c.k;
    const T* vb = (const T*)p.c.v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = __shfl_sync(0xffffffffu, off, r + 8 * j);
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const bool there = at >= 0 && c + 4 * i < 2 * chunks;
        cp_async16_or_zero(stage + ((j * KC + i) * 32 + lane) * 16, kb + (there ? at + (c + 4 * i) * 4 : 0), there);
      }
    }
#pragma unroll
    for (int i = 0; i < DH / 8; ++i) {
      const int e = lane + 32 * i, t = e / (DH / 4), ch = e % (DH / 4);
      const int64_t at = __shfl_sync(0xffffffffu, off, 16 + t);
      const bool there = at >= 0 && ch < 2 * chunks;
      cp_async16_or_zero(stage + 64 * DH + e * 16, vb + (there ? at + ch * 4 : 0), there);
    }
  }

  ONE_DEVINL void begin(const PagedAttn& p, uint8_t* extra, const T* q, int rows) {
    const int lane = threadIdx.x & 31;
    qs = reinterpret_cast<float*>(extra);
    ps = qs + 4 * DH;
    __syncwarp();
    for (int i = lane; i < 4 * DH; i += 32) {
      const int g = i / DH, d = i % DH;
      qs[i] = g < rows && d < p.c.Dh ? q[g * p.q_hs + d] : 0.f;
    }
    __syncwarp();
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < VC; ++i) o[g][i] = 0.f;
  }

  ONE_DEVINL void consume(const PagedAttn& p, const uint8_t* stage, uint32_t live, float* scores, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(stage + (i * 32 + lane) * 16);
      const float4 b = *reinterpret_cast<const float4*>(stage + ((KC + i) * 32 + lane) * 16);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 q = *reinterpret_cast<const float4*>(qs + g * DH + (c + 4 * i) * 4);
        s[0][g] += q.x * a.x + q.y * a.y + q.z * a.z + q.w * a.w;
        s[1][g] += q.x * b.x + q.y * b.y + q.z * b.z + q.w * b.w;
      }
    }
    float x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // lane c keeps head c
      const float k0 = c & 2 ? s[j][2] : s[j][0], k1 = c & 2 ? s[j][3] : s[j][1];
      const float g0 = c & 2 ? s[j][0] : s[j][2], g1 = c & 2 ? s[j][1] : s[j][3];
      const float y0 = k0 + __shfl_xor_sync(0xffffffffu, g0, 2), y1 = k1 + __shfl_xor_sync(0xffffffffu, g1, 2);
      x[j] = (c & 1 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, c & 1 ? y0 : y1, 1);
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
      for (int g = 0; g < 4; ++g) {
        const float ag = __shfl_sync(0xffffffffu, a, g);
#pragma unroll
        for (int i = 0; i < VC; ++i) o[g][i] *= ag;
      }
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[j] = exp2f(x[j] - ms);
      l += x[j];
      ps[(r + 8 * j) * 4 + c] = x[j];
    }
    __syncwarp();
    const float* vs = reinterpret_cast<const float*>(stage + 64 * DH);
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const float4 w = *reinterpret_cast<const float4*>(ps + 4 * t);
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const float v = vs[t * DH + lane + 32 * i];
        o[0][i] += w.x * v;
        o[1][i] += w.y * v;
        o[2][i] += w.z * v;
        o[3][i] += w.w * v;
      }
    }
    __syncwarp();
  }

  ONE_DEVINL void leave(float* ml, float* so) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    float t = l;
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (r == 0) {
      ml[2 * c] = m;
      ml[2 * c + 1] = t;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < VC; ++i) so[g * DH + lane + 32 * i] = o[g][i];
  }
};

template <typename E>
struct PaSmem {
  static constexpr int kRing = kPaWarps * E::kStage * E::kStages;
  static constexpr int kO = kRing;                                       // [warps][ROWS][DH] floats
  static constexpr int kML = kO + kPaWarps * E::ROWS * E::DH * 4;        // [warps][ROWS][2]
  static constexpr int kFin = kML + kPaWarps * E::ROWS * 8;              // [ROWS][2]: m, 1 / l
  static constexpr int kLive = kFin + E::ROWS * 8;                       // [warps][stages] live masks
  static constexpr int kExtra = kLive + kPaWarps * E::kStages * 4 + 16 - (kPaWarps * E::kStages * 4) % 16;
  static constexpr int kTotal = kExtra + kPaWarps * E::kExtra;
};

// SPLIT: CTA i takes the i-th share of the list. Otherwise CTA (hv, b) takes that segment whole and
// nothing is left to join (short caches: one launch).
template <typename E, bool SPLIT>
__global__ void __launch_bounds__(kPaWarps * 32) paged_attn_kernel(const __grid_constant__ PagedAttn p) {
  extern __shared__ __align__(16) uint8_t smem[];
  using S = PaSmem<E>;
  using T = typename E::T;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * (E::kStage * E::kStages);
  float* so = reinterpret_cast<float*>(smem + S::kO);
  float* ml = reinterpret_cast<float*>(smem + S::kML);
  float* fin = reinterpret_cast<float*>(smem + S::kFin);
  volatile uint32_t* lives = reinterpret_cast<uint32_t*>(smem + S::kLive) + warp * E::kStages;
  uint8_t* extra = smem + S::kExtra + warp * E::kExtra;
  const PagedCache& c = p.c;
  const int chunks = c.Dh / 8, HV = c.Hkv * p.hv_per_kv;
  pdl_wait();
  pdl_launch_dependents();
  PaCursor cur;
  long long w0, w1;
  if (SPLIT) {
    const long long total = pa_total(p), chunk = pa_chunk(p, total);
    w0 = chunk * blockIdx.x;
    w1 = min(w0 + chunk, total);
    if (w0 >= w1) return;
    cur.seek(c, HV, w0);
  } else {
    cur.b = blockIdx.y;
    cur.hv = blockIdx.x;
    cur.tile = 0;
    cur.load(c);
    w0 = 0;
    w1 = cur.tiles;
  }
  // ---- the copying side: page numbers are asked for one tile ahead of the copies
  PaCursor src = cur;
  long long asked = w0;
  int pg = -1;
  auto ask = [&] {
    pg = -1;
    const int t = src.tile * kPaTile + warp * 16 + (lane & 15);
    if (asked < w1 && t < src.len) {
      pg = c.table[src.b * c.table_stride + (int)(((uint64_t)(uint32_t)t * p.div_m) >> p.div_s)];
      if (pg < 0 || pg >= c.num_pages) {
        set_err(c.err, ERR_BAD_ARG, SITE_PAGED_ATTN);
        pg = -1;
      }
    }
  };
  int put = 0, get = 0;
  auto copy = [&] {
    if (asked < w1) {
      const int t = src.tile * kPaTile + warp * 16 + (lane & 15);
      const int slot = t - (int)(((uint64_t)(uint32_t)t * p.div_m) >> p.div_s) * c.page_size;
      const int64_t off =
          pg < 0 ? -1 : pg * (lane < 16 ? c.k_stride : c.v_stride) + ((int64_t)(src.hv / p.hv_per_kv) * c.page_size + slot) * c.Dh;
      const uint32_t live = __ballot_sync(0xffffffffu, off >= 0) & 0xffffu;
      if (lane == 0) lives[put] = live;
      if (live) E::issue(p, ring + put * E::kStage, off, chunks);
      ++asked;
      if (asked < w1) src.next(c, HV);
      ask();
    }
    cp_async_commit();
    put = put + 1 == E::kStages ? 0 : put + 1;
  };
  ask();
#pragma unroll 1
  for (int i = 0; i < E::kStages - 1; ++i) copy();
  // ---- the computing side, piece by piece
  E eng;
  long long w = w0;
  do {
    const int kv = cur.hv / p.hv_per_kv, g0 = (cur.hv % p.hv_per_kv) * E::ROWS, rows = min(E::ROWS, p.G - g0);
    const int64_t hq0 = ((int64_t)cur.b * c.Hkv + kv) * p.G + g0;  // output row of this query-head tile
    const int first = cur.tile, last = (int)min((long long)cur.tiles, cur.tile + (w1 - w));
    if (cur.b >= c.B || (last <= first && cur.tiles > 0)) break;  // lengths that changed during the call
    eng.begin(p, extra, (const T*)p.q + cur.b * p.q_bs + ((int64_t)kv * p.G + g0) * p.q_hs, rows);
    for (int tile = first; tile < last; ++tile) {
      copy();
      cp_async_wait<E::kStages - 1>();
      __syncwarp();
      const uint32_t live = lives[get];
      if (live)
        eng.consume(p, ring + get * E::kStage, live,
                    p.scores ? p.scores + hq0 * p.score_ld + tile * kPaTile + warp * 16 : nullptr, rows);
      else if (p.scores)
        for (int i = lane; i < rows * 16; i += 32)
          p.scores[(hq0 + i / 16) * p.score_ld + tile * kPaTile + warp * 16 + i % 16] = -INFINITY;
      __syncwarp();
      get = get + 1 == E::kStages ? 0 : get + 1;
    }
    eng.leave(ml + warp * E::ROWS * 2, so + warp * E::ROWS * E::DH);
    __syncthreads();
    const bool whole = first == 0 && last == cur.tiles;
    const int64_t part = 2ll * blockIdx.x + (w > w0 ? 1 : 0);
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
        const float4 x = *reinterpret_cast<const float4*>(so + (k * E::ROWS + g) * E::DH + d);
        a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
      }
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (d < c.Dh) {
          T* y = (T*)p.out + (hq0 + g) * c.Dh + d;
          st<T>(y, a.x * inv); st<T>(y + 1, a.y * inv); st<T>(y + 2, a.z * inv); st<T>(y + 3, a.w * inv);
        }
        if (d == 0) {
          fin[2 * g] = Ms;
          fin[2 * g + 1] = inv;
          if (SPLIT && p.mass) {
            p.row_ml[2 * (hq0 + g)] = Ms;
            p.row_ml[2 * (hq0 + g) + 1] = inv;
          }
        }
      } else {
        *reinterpret_cast<float4*>(p.part_o + (part * E::ROWS + g) * E::DH + d) = a;
        if (d == 0) {
          p.part_ml[(part * E::ROWS + g) * 2] = M;
          p.part_ml[(part * E::ROWS + g) * 2 + 1] = L;
        }
      }
    }
    __syncthreads();
    if (!SPLIT && p.mass) {  // one query-head tile per kv head: this CTA wrote all of its scores
      float* mass = p.mass + ((int64_t)cur.b * c.Hkv + kv) * p.mass_width;
      for (int t = threadIdx.x; t < cur.len; t += blockDim.x) {
        float a = 0.f;
        for (int g = 0; g < rows; ++g) a += ex2_approx(p.scores[(hq0 + g) * p.score_ld + t] - fin[2 * g]) * fin[2 * g + 1];
        mass[t] += a;
      }
    }
    w += last - first;
    cur.tile = last - 1;
    if (w < w1) cur.next(c, HV);
  } while (w < w1);
}

// The parts of a segment [s0, s1) of the list, cut every `chunk` tiles.
struct PaParts {
  long long first, last;
  bool inner;  // the first part does not start its CTA's share
  ONE_DEVINL PaParts(long long s0, long long s1, long long chunk)
      : first(s0 / chunk), last((s1 - 1) / chunk), inner(s0 % chunk != 0) {}
  ONE_DEVINL int64_t at(long long i) const { return 2 * i + (i == first && inner ? 1 : 0); }
};

// Joins what paged_attn_kernel<SPLIT> left. Blocks below B * Hq: one output row each. With mass,
// further blocks add the weights: block i takes the i-th share of the tiles of every (sequence, kv
// head), recomputing the joint (m, l) of its rows from the parts.
template <typename E>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedAttn p) {
  using T = typename E::T;
  constexpr int ROWS = E::ROWS, DH = E::DH;
  __shared__ float4 red[128];
  __shared__ float fin[2][128];  // m and 1 / l of a kv head's query heads
  const PagedCache& c = p.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hq = c.Hkv * p.G;
  pdl_wait();
  const long long total = pa_total(p), chunk = pa_chunk(p, total);
  const int HV = c.Hkv * p.hv_per_kv;
  // joint m and 1 / l of row g of the parts, by one warp
  auto joint = [&](const PaParts& parts, int g, float& M, float& inv) {
    float mm = -INFINITY;
    for (long long i = parts.first + lane; i <= parts.last; i += 32) mm = fmaxf(mm, p.part_ml[(parts.at(i) * ROWS + g) * 2]);
    M = warp_max(mm);
    if (M == -INFINITY) M = 0.f;
    float L = 0.f;
    for (long long i = parts.first + lane; i <= parts.last; i += 32) {
      const float* x = p.part_ml + (parts.at(i) * ROWS + g) * 2;
      L += x[1] * exp2f(x[0] - M);
    }
    L = warp_sum(L);
    inv = L == 0.f ? 0.f : 1.f / L;
  };
  if ((long long)blockIdx.x < (long long)c.B * hq) {
    const int b = blockIdx.x / hq, j = blockIdx.x % hq, kv = j / p.G, g = j % p.G;
    const int tiles = pa_tiles(c, b);
    T* out = (T*)p.out + (int64_t)blockIdx.x * c.Dh;
    if (tiles == 0) {
      for (int d = tid; d < c.Dh; d += blockDim.x) st<T>(out + d, 0.f);
      return;
    }
    const int hv = kv * p.hv_per_kv + g / ROWS;
    const long long s0 = HV * pa_before(p, b) + (long long)hv * tiles;
    const PaParts parts(s0, s0 + tiles, chunk);
    if (parts.first == parts.last) return;
    const int row = g % ROWS;
    float M, inv;
    joint(parts, row, M, inv);
    constexpr int C4 = DH / 4, NG = 128 / C4;  // float4 columns; parts summed side by side
    const int col = tid % C4, grp = tid / C4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (grp < NG)
      for (long long i = parts.first + grp; i <= parts.last; i += NG) {
        const int64_t at = parts.at(i) * ROWS + row;
        const float f = exp2f(p.part_ml[2 * at] - M);
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * DH + col * 4);
        a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
      }
    red[tid] = a;
    __syncthreads();
    if (tid < C4 && tid * 4 < c.Dh) {
      for (int k = 1; k < NG; ++k) {
        const float4 x = red[k * C4 + tid];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      }
      T* y = out + tid * 4;
      st<T>(y, a.x * inv); st<T>(y + 1, a.y * inv); st<T>(y + 2, a.z * inv); st<T>(y + 3, a.w * inv);
    }
    return;
  }
  // ---- mass: the tiles of every (sequence, kv head) in the same order, in equal shares
  const long long mtotal = total / p.hv_per_kv, share = max(1ll, (mtotal + p.ranges - 1) / p.ranges);
  long long w = share * (blockIdx.x - (long long)c.B * hq);
  const long long w1 = min(w + share, mtotal);
  if (w >= w1) return;
  PaCursor cur;
  cur.seek(c, c.Hkv, w);
  while (w < w1) {
    const int first = cur.tile, last = (int)min((long long)cur.tiles, cur.tile + (w1 - w));
    if (cur.b >= c.B || last <= first) break;
    const long long before = HV * pa_before(p, cur.b);
    const int t0 = first * kPaTile, t1 = min(last * kPaTile, cur.len);
    float* mass = p.mass + ((int64_t)cur.b * c.Hkv + cur.hv) * p.mass_width;
    const int64_t row0 = ((int64_t)cur.b * c.Hkv + cur.hv) * p.G;
    for (int gb = 0; gb < p.G; gb += 128) {
      const int gn = min(128, p.G - gb);
      __syncthreads();
      for (int g = gb + warp; g < gb + gn; g += 4) {
        const long long s0 = before + (long long)(cur.hv * p.hv_per_kv + g / ROWS) * cur.tiles;
        const PaParts parts(s0, s0 + cur.tiles, chunk);
        float M, inv;
        if (parts.first == parts.last) {
          M = p.row_ml[2 * (row0 + g)];
          inv = p.row_ml[2 * (row0 + g) + 1];
        } else {
          joint(parts, g % ROWS, M, inv);
        }
        if (lane == 0) {
          fin[0][g - gb] = M;
          fin[1][g - gb] = inv;
        }
      }
      __syncthreads();
      for (int t = t0 + tid; t < t1; t += blockDim.x) {
        float a = 0.f;
        for (int g = 0; g < gn; ++g) a += ex2_approx(p.scores[(row0 + gb + g) * p.score_ld + t] - fin[0][g]) * fin[1][g];
        mass[t] += a;
      }
    }
    w += last - first;
    cur.tile = last - 1;
    if (w < w1) cur.next(c, c.Hkv);
  }
}

}  // namespace one
