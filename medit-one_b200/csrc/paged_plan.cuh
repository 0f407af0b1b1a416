// How the attention of one new token over a paged cache is cut: clusters or a list, workspace, launches.
#pragma once

#include "paged_attn.cuh"
#include "serving_host.cuh"

namespace one {
namespace {

constexpr int kMaxTile = 256;  // slots of the largest tile
constexpr int kWhole = 512;    // slots that one CTA takes rather than split them

// CTAs per segment, when segments are not cut from a list: up to 296 in all (two per SM), and no more than
// one per 256 slots of the table.
int paged_cluster(int64_t segments, int64_t slots) {
  int n = 1;
  while (n < 8 && segments * n * 2 <= 296 && slots > 256 * n) n *= 2;
  return n;
}

// Whether the segments are cut from a list. A cluster per segment has one launch and no second pass, but at
// most 8 CTAs for a long sequence, shares as uneven as the lengths, and with weights a second look at the
// scores by the CTAs that hold them alone. The list gains with few segments, uneven lengths and weights,
// clusters with many even segments; 512 slots per CTA lie between. Us per call, by clusters and from a list
// (one after the other in a graph, 64 dims, bf16 unless said):
//   12 heads of one sequence (8 CTAs each): 1000 slots 6.4, 6.6; 2500 8.3, 7.5; 4000 9.3, 7.8; 8000 13.8, 9.9
//   16 x 4 heads x 3 queries (4 CTAs each): 1600 slots 9.7, 10.1; 2500 13.4, 14.4; 3500 16.2, 17.3
//     with weights: 1200 11.3, 11.5; 1600 13.4, 11.7; 2500 20.4, 17.4; fp32 1200 16.3, 18.0; 2500 25.7, 24.6
//   16 x 12 heads (1 CTA each), ragged up to 500: 7.2, 9.4; 700 9.2, 9.6; 1024 11.8, 10.3; 2048 23.5, 16.4
//   64 x 12 heads, ragged up to 700: 20.4, 22.6; 1024 27.3, 27.9; 2048 46.6, 45.4; 4096 86.7, 73.0; all of
//     700: 28.0, 31.7
bool paged_split(int64_t segments, int64_t slots) {
  const int64_t n = paged_cluster(segments, slots);
  return slots > kWhole * n;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Query heads that one pass over a kv head's cache serves.
int paged_rows(int dtype, int G) { return dtype == ONE_DTYPE_F32 ? (G > 1 ? 4 : 1) : G > 8 ? 16 : 8; }

struct PagedWs {
  size_t part_ml, part_o, row_ml, segs, scores, total;
  int64_t score_ld;
  PagedWs(int b, int hq, int rows, int dh_pad, int64_t slots, bool mass) {
    const size_t parts = 2 * (size_t)kMaxSms * kPaPerSm * rows;
    part_ml = 0;
    part_o = align256(parts * 8);
    row_ml = part_o + align256(parts * dh_pad * 4);
    segs = row_ml + align256(mass ? (size_t)b * hq * 8 : 0);
    scores = segs + align256((size_t)b * hq * 8);
    score_ld = (slots + kMaxTile - 1) / kMaxTile * kMaxTile;
    total = scores + (mass ? (size_t)b * hq * score_ld * 4 : 0);
  }
};

int pad_dh(int dh) { return dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : 128; }

template <typename E, bool RUN, PaMode MODE>
int attend(PagedAttn& p, int cluster, cudaStream_t st) {
  constexpr bool SPLIT = MODE == PA_LIST;
  static std::atomic<bool> done[kMaxDevices];
  int rc = allow_smem(paged_attn_kernel<E, RUN, MODE>, PaSmem<E, MODE>::kTotal, done);
  if (rc) return rc;
  const int64_t heads = (int64_t)p.c.B * p.c.Hkv, slots = (int64_t)p.c.max_pages * p.c.page_size;
  p.ranges = std::min(num_sms(), kMaxSms) * PaSmem<E, MODE>::kPerSm;
  p.cluster = SPLIT ? 1 : cluster;
  rc = launched(launch_cluster(p.cluster, paged_attn_kernel<E, RUN, MODE>, dim3((unsigned)(SPLIT ? p.ranges : heads * p.hv_per_kv * cluster)),
                               dim3(kPaWarps * 32), PaSmem<E, MODE>::kTotal, st, p),
                "paged attention");
  if (rc || !SPLIT) return rc;
  const int mass_blocks = p.mass ? (int)((slots + kJoinSlots - 1) / kJoinSlots) : 0;
  return launched(launch(paged_join_kernel<E>, dim3((unsigned)(heads * (p.G + mass_blocks))), dim3(kJoinThreads), 0, st, p,
                         mass_blocks),
                  "paged attention join");
}

// A deeper ring costs the third CTA of an SM: taken where two per SM hold the grid at once, and clusters
// of 4 and 8 are not placed as densely as that (36 of 8 are not, 32 are). bf16, slots as given, us per call
// one after the other in a graph, with the deeper ring and without: 16 x 8 heads x 128, 1000 (256 CTAs in
// pairs) 15.7, 17.3; 37 x 8 x 128, 500 (296 single) 16.0, 17.2; 24 x 12 x 64, 500 (288) 10.3, 11.0; 26 x 12
// x 64, 500 (312) 16.0, 11.6; 8 x 4 x 64, 4000 (32 clusters of 8) 11.6, 12.6; 9 x 4 x 64, 4000 (36) 21.4,
// 13.4; 64 x 12 x 64, 128 (768) 10.1, 8.0; 149 x 16 x 64, 32 (2384) 24.7, 18.3.
bool paged_deep(int64_t segments, int cluster) { return segments * cluster <= (cluster > 2 ? 256 : 296); }

template <typename E, bool RUN>
int attend(PagedAttn& p, bool split, cudaStream_t st) {
  const int64_t segments = (int64_t)p.c.B * p.c.Hkv * p.hv_per_kv;
  const int cluster = paged_cluster(segments, (int64_t)p.c.max_pages * p.c.page_size);
  if (split) return attend<E, RUN, PA_LIST>(p, cluster, st);
  if constexpr (E::kStagesFew > E::kStages)
    if (paged_deep(segments, cluster)) return attend<E, RUN, PA_DEEP>(p, cluster, st);
  return attend<E, RUN, PA_SEGMENT>(p, cluster, st);
}

template <typename E>
int attend(PagedAttn& p, bool split, cudaStream_t st) {
  const bool run = p.c.page_size % 16 == 0 && p.c.Dh == E::DH;
  return run ? attend<E, true>(p, split, st) : attend<E, false>(p, split, st);
}

}  // namespace
}  // namespace one
