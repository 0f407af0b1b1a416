// Host side of the operators over a paged cache: checks, the cut of the attention into clusters or a list, its
// workspace, launches.
#pragma once

#include "paged_attn.cuh"
#include "serving_host.cuh"

namespace one {
namespace {

// What the operators over a paged cache of either kind ask of its table and sizes; head_dim in units of `dims`.
template <typename S>
int check_table(PagedCache& c, const S* x, int dims) {
  if (!x || !x->k_pages || !x->v_pages || !x->block_table || !x->lengths)
    return fail(ONE_ERR_INVALID, "paged cache: null argument");
  if (x->num_pages < 1 || x->page_size < 1 || x->max_pages < 1 || x->b < 1 || x->hkv < 1 || x->dh < 1)
    return fail(ONE_ERR_INVALID, "paged cache: sizes must be positive");
  if (x->dh > 128 || x->dh % dims) return fail(ONE_ERR_UNSUPPORTED, "paged cache: head_dim a multiple of %d, at most 128", dims);
  if (x->b > 65535 || x->hkv > 65535) return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 65535 sequences and heads");
  if ((int64_t)x->max_pages * x->page_size > 0x3fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 2^30 - 1 slots per sequence");
  if (x->table_stride < x->max_pages) return fail(ONE_ERR_INVALID, "paged cache: block table rows overlap");
  if (x->mass && x->mass_width < (int64_t)x->max_pages * x->page_size)
    return fail(ONE_ERR_INVALID, "paged cache: mass rows are shorter than the block table's slots");
  c.table = x->block_table; c.table_stride = x->table_stride; c.lengths = x->lengths;
  c.num_pages = x->num_pages; c.page_size = x->page_size; c.max_pages = x->max_pages; c.B = x->b; c.Hkv = x->hkv; c.Dh = x->dh;
  return ONE_OK;
}

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
// All of these are of a dense cache. One in 4 or 8 bits goes by the same rule, for which it has not been measured.
bool paged_split(int64_t segments, int64_t slots) {
  const int64_t n = paged_cluster(segments, slots);
  return slots > kWhole * n;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// t / page_size for t < 2^31 as a product and a shift.
void paged_divisor(PagedAttn& p, int page_size) {
  while ((1 << p.div_s) < page_size) ++p.div_s;
  p.div_m = (uint32_t)((1ull << (31 + p.div_s)) / page_size + 1);
  p.div_s += 31;
}

// Query heads that one pass over a kv head's cache serves.
int paged_rows(int dtype, int G) { return dtype == ONE_DTYPE_F32 ? (G > 1 ? 4 : 1) : G > 8 ? 16 : 8; }

struct PagedWs {
  size_t part_ml, part_o, row_ml, segs, scores, total;
  int64_t score_ld;
  PagedWs(int b, int hq, int rows, int dh_pad, int64_t slots, bool mass, int per_sm) {
    const size_t parts = 2 * (size_t)kMaxSms * per_sm * rows;
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

// What the attention over a cache of either kind, in p.c, asks of its arguments, and its plan; `rows` query
// heads per pass, at most per_sm shares of a list per SM, `units` as E::kSegmentUnits, tiles of least_tile slots or more. need: workspace bytes.
template <typename S>
int plan_attention(PagedAttn& p, bool& split, const S* cache, const void* q, int64_t q_bs, int64_t q_hs, int hq, int rows, int per_sm, int units, int least_tile,
                   float scale, void* out, void* workspace, size_t workspace_bytes, size_t need) {
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh, page_size = cache->page_size;
  float* mass = cache->mass;
  const int64_t slots = (int64_t)cache->max_pages * page_size;
  // tiles and a segment's further units, and the list's length rounded up to equal shares, in 31 bits
  if ((int64_t)b * hq > 0x3fffffff || (int64_t)b * hq * (slots / least_tile + 1 + units) > 0x7fffffff - kMaxSms * per_sm)
    return fail(ONE_ERR_UNSUPPORTED, "paged attention: too many rows");
  if (need && (!workspace || workspace_bytes < need)) return fail(ONE_ERR_INVALID, "workspace too small");
  p.q = q; p.q_bs = q_bs; p.q_hs = q_hs; p.G = hq / hkv;
  p.hv_per_kv = (p.G + rows - 1) / rows;
  p.q_vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_bs % 8 == 0 && q_hs % 8 == 0;
  paged_divisor(p, page_size);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mass = mass; p.mass_width = cache->mass_width; p.out = out;
  const PagedWs w(b, hq, rows, pad_dh(dh), slots, mass != nullptr, per_sm);
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  p.part_ml = reinterpret_cast<float*>(ws + w.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.row_ml = reinterpret_cast<float*>(ws + w.row_ml);
  p.parts = reinterpret_cast<int2*>(ws + w.segs);
  p.scores = mass ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  p.score_ld = w.score_ld;
  split = paged_split((int64_t)b * hkv * p.hv_per_kv, slots) || (mass && p.hv_per_kv > 1);
  return ONE_OK;
}

size_t attention_bytes(int b, int hq, int hkv, int dh, int rows, int page_size, int max_pages, bool with_mass, int per_sm) {
  if (b < 1 || hq < 1 || hkv < 1 || dh < 1 || page_size < 1 || max_pages < 1) return 0;
  const int64_t slots = (int64_t)max_pages * page_size;
  const int tiles = (hq / hkv + rows - 1) / rows;
  if (!with_mass && !paged_split((int64_t)b * hkv * tiles, slots)) return 0;
  return PagedWs(b, hq, rows, pad_dh(dh), slots, with_mass, per_sm).total + 256;
}

template <typename E, bool RUN, PaMode MODE>
int attend(PagedAttn& p, int cluster, cudaStream_t st) {
  constexpr bool SPLIT = MODE == PA_LIST;
  static std::atomic<bool> done[kMaxDevices];
  int rc = allow_smem(paged_attn_kernel<E, RUN, MODE>, PaSmem<E, MODE>::kTotal, done);
  if (rc) return rc;
  const int64_t heads = (int64_t)p.c.B * p.c.Hkv, slots = (int64_t)p.c.max_pages * p.c.page_size;
  const int ctas = std::min(num_sms(), kMaxSms) * PaSmem<E, MODE>::kPerSm;
  p.ranges = ctas * (PaSmem<E, MODE>::kLone ? kPaWarps : 1);
  p.cluster = SPLIT ? 1 : cluster;
  rc = launched(launch_cluster(p.cluster, paged_attn_kernel<E, RUN, MODE>, dim3((unsigned)(SPLIT ? ctas : heads * p.hv_per_kv * cluster)),
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
  const bool run = p.c.page_size % 16 == 0 && p.c.Dh == E::DH && (!E::kQuant || p.run);
  return run ? attend<E, true>(p, split, st) : attend<E, false>(p, split, st);
}

// Eviction over a cache of either kind, in p.c: `pieces` units of U per row.
template <typename U, typename S>
int evict(PagedEvictParams& p, const S* cache, int pieces, const int32_t* dst_table, int64_t dst_stride, int32_t dst_max_pages,
          int32_t budget, int32_t recent, int32_t sink, float* mass_out, int64_t mass_out_width, int32_t* kept, cudaStream_t st) {
  if (!dst_table || !mass_out || !kept) return fail(ONE_ERR_INVALID, "paged evict: null argument");
  const int b = cache->b, hkv = cache->hkv, page_size = cache->page_size;
  if (budget < 1 || recent < 0 || sink < 0 || (int64_t)recent + sink > budget)
    return fail(ONE_ERR_INVALID, "paged evict: 1 <= budget, 0 <= recent, sink and recent + sink <= budget");
  if (dst_max_pages < 1 || dst_stride < dst_max_pages || (int64_t)dst_max_pages * page_size < budget)
    return fail(ONE_ERR_INVALID, "paged evict: the destination pages hold fewer slots than the budget");
  if (mass_out_width < budget) return fail(ONE_ERR_INVALID, "paged evict: mass rows are too short");
  if (mass_out_width > 0x3fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged evict: too many rows");
  p.dst = dst_table; p.dst_stride = dst_stride; p.mass = cache->mass; p.mass_width = cache->mass_width;
  p.budget = budget; p.recent = recent; p.sink = sink; p.mass_out = mass_out; p.out_width = mass_out_width; p.kept = kept;
  const int64_t slots = (int64_t)cache->max_pages * page_size, heads = (int64_t)b * hkv;
  const int64_t parts = (budget + 255) / 256, per_bh = (mass_out_width + kMovePlaces - 1) / kMovePlaces;
  // where the CTAs fit the SMs at once: two per SM, one of those that hold 64 keys per thread (192 CTAs of
  // those, 48 heads of 30000 slots to 1000: 49 us in one launch, 29 in two; device times)
  const bool one_launch = heads * parts <= (slots > 16384 && slots <= 32768 ? 1 : 2) * num_sms();
  if (heads * std::max(parts, per_bh) > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged evict: too many rows");
  auto select = [&](auto keys) {
    constexpr int KPT = decltype(keys)::value;
    return one_launch ? launch(paged_evict_kernel<KPT, true, U>, dim3((unsigned)(heads * parts)), dim3(kEvictThreads), 0, st, p,
                               (int)parts, pieces)
                      : launch(paged_evict_kernel<KPT, false, U>, dim3((unsigned)heads), dim3(kEvictThreads), 0, st, p, 1, pieces);
  };
  const int rc = launched(slots <= 1024    ? select(Int<2>())
                          : slots <= 2048  ? select(Int<4>())
                          : slots <= 4096  ? select(Int<8>())
                          : slots <= 8192  ? select(Int<16>())
                          : slots <= 16384 ? select(Int<32>())
                          : slots <= 32768 ? select(Int<64>())
                                           : select(Int<0>()),
                          "paged evict");
  if (rc || one_launch) return rc;
  return launched(launch(paged_move_kernel<U>, dim3((unsigned)(per_bh * heads)), dim3(kMoveThreads), 0, st, p, (int)per_bh, pieces),
                  "paged move");
}

}  // namespace
}  // namespace one
