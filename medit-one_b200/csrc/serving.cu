// extern "C" operators of one serving step over a paged key-value cache and of the logits
// processor (one_b200.h, "serving ops").
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <utility>

#include "../../include/one_b200.h"
#include "common.cuh"
#include "logits.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"

using namespace one;

// Hidden helpers of engine.cu: the calling thread's error message and the standalone ops' device
// error record on the current device.
extern "C" __attribute__((visibility("hidden"))) int one_set_error(int code, const char* msg);
extern "C" __attribute__((visibility("hidden"))) void* one_ops_err_record();

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return one_set_error(code, buf);
}

bool use_pdl() {
  static const bool pdl = [] {
    const char* v = getenv("ONE_B200_NO_PDL");
    return !(v && v[0] == '1');
  }();
  return pdl;
}

// Launches with programmatic stream serialization, as clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(unsigned cluster, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                           cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (use_pdl()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  return launch_cluster(1, kernel, grid, block, smem, st, std::forward<Args>(args)...);
}

// cudaFuncAttributeMaxDynamicSharedMemorySize of a kernel, once per device.
constexpr int kMaxDevices = 64;
template <typename K>
int allow_smem(K* kernel, int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return ONE_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(ONE_ERR_CUDA, "shared memory of a kernel: %s", cudaGetErrorString(e));
  if (dev < kMaxDevices) done[dev].store(true, std::memory_order_release);
  return ONE_OK;
}

// SMs of the current device.
int num_sms() {
  static std::atomic<int> sms[kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < kMaxDevices && (n = sms[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
  if (dev < kMaxDevices) sms[dev].store(n, std::memory_order_relaxed);
  return n;
}

int elem_bytes(int dtype) { return dtype == ONE_DTYPE_F32 ? 4 : 2; }

// What every operator over a cache asks of it.
int check_cache(PagedCache& c, const one_paged_cache* x) {
  if (!x || !x->k_pages || !x->v_pages || !x->block_table || !x->lengths)
    return fail(ONE_ERR_INVALID, "paged cache: null argument");
  if (x->dtype != ONE_DTYPE_BF16 && x->dtype != ONE_DTYPE_F32) return fail(ONE_ERR_INVALID, "paged cache: dtype");
  if (x->num_pages < 1 || x->page_size < 1 || x->max_pages < 1 || x->b < 1 || x->hkv < 1 || x->dh < 1)
    return fail(ONE_ERR_INVALID, "paged cache: sizes must be positive");
  if (x->dh > 128 || x->dh % 8) return fail(ONE_ERR_UNSUPPORTED, "paged cache: head_dim a multiple of 8, at most 128");
  if (x->b > 65535 || x->hkv > 65535) return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 65535 sequences and heads");
  if ((int64_t)x->max_pages * x->page_size > 0x3fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 2^30 - 1 slots per sequence");
  if (x->table_stride < x->max_pages) return fail(ONE_ERR_INVALID, "paged cache: block table rows overlap");
  const int64_t page = (int64_t)x->hkv * x->page_size * x->dh, es = elem_bytes(x->dtype);
  const int64_t ks = x->k_page_stride, vs = x->v_page_stride;
  if (ks > 0x7fffffff || vs > 0x7fffffff || page > 0x7fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: pages of at most 2^31 - 1 elements");
  if (ks < page || vs < page) return fail(ONE_ERR_INVALID, "paged cache: pages overlap");
  if (((reinterpret_cast<uintptr_t>(x->k_pages) | reinterpret_cast<uintptr_t>(x->v_pages)) & 15) || ks * es % 16 || vs * es % 16)
    return fail(ONE_ERR_INVALID, "paged cache: pages must start on 16-byte boundaries");
  if (x->mass && x->mass_width < (int64_t)x->max_pages * x->page_size)
    return fail(ONE_ERR_INVALID, "paged cache: mass rows are shorter than the block table's slots");
  c.k = x->k_pages; c.v = x->v_pages; c.k_stride = ks; c.v_stride = vs;
  c.table = x->block_table; c.table_stride = x->table_stride; c.lengths = x->lengths;
  c.num_pages = x->num_pages; c.page_size = x->page_size; c.max_pages = x->max_pages; c.B = x->b; c.Hkv = x->hkv; c.Dh = x->dh;
  c.err = reinterpret_cast<DevErr*>(one_ops_err_record());
  return ONE_OK;
}

int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? ONE_OK : fail(ONE_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace

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

extern "C" size_t one_paged_attention_workspace_bytes(int32_t b, int32_t hq, int32_t hkv, int32_t dh, int32_t page_size,
                                                      int32_t max_pages, int32_t dtype, int32_t with_mass) {
  if (b < 1 || hq < 1 || hkv < 1 || dh < 1 || page_size < 1 || max_pages < 1) return 0;
  const int64_t slots = (int64_t)max_pages * page_size;
  const int rows = paged_rows(dtype, hq / hkv), tiles = (hq / hkv + rows - 1) / rows;
  if (!with_mass && !paged_split((int64_t)b * hkv * tiles, slots)) return 0;
  return PagedWs(b, hq, rows, pad_dh(dh), slots, with_mass != 0).total + 256;
}

extern "C" int one_paged_attention(const one_paged_cache* cache, const void* q, int64_t q_batch_stride,
                                   int64_t q_head_stride, int32_t hq, float scale, void* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!q || !out) return fail(ONE_ERR_INVALID, "paged attention: null argument");
  PagedAttn p = {};
  int rc = check_cache(p.c, cache);
  if (rc) return rc;
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh, dtype = cache->dtype, page_size = cache->page_size;
  float* mass = cache->mass;
  if (hq < 1 || hq % hkv) return fail(ONE_ERR_INVALID, "paged attention: the query heads must be a multiple of the kv heads");
  const int64_t slots = (int64_t)cache->max_pages * page_size;
  // tiles, and the list's length rounded up to equal shares, in 31 bits
  if ((int64_t)b * hq > 0x3fffffff || (int64_t)b * hq * (slots / 64 + 1) > 0x7fffffff - kMaxSms * kPaPerSm)
    return fail(ONE_ERR_UNSUPPORTED, "paged attention: too many rows");
  const size_t need = one_paged_attention_workspace_bytes(b, hq, hkv, dh, page_size, cache->max_pages, dtype, mass != nullptr);
  if (need && (!workspace || workspace_bytes < need)) return fail(ONE_ERR_INVALID, "workspace too small");
  p.q = q; p.q_bs = q_batch_stride; p.q_hs = q_head_stride; p.G = hq / hkv;
  const int rows = paged_rows(dtype, p.G);
  p.hv_per_kv = (p.G + rows - 1) / rows;
  p.q_vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && q_batch_stride % 8 == 0 && q_head_stride % 8 == 0;
  while ((1 << p.div_s) < page_size) ++p.div_s;
  p.div_m = (uint32_t)((1ull << (31 + p.div_s)) / page_size + 1);
  p.div_s += 31;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mass = mass; p.mass_width = cache->mass_width; p.out = out;
  const PagedWs w(b, hq, rows, pad_dh(dh), slots, mass != nullptr);
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  p.part_ml = reinterpret_cast<float*>(ws + w.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.row_ml = reinterpret_cast<float*>(ws + w.row_ml);
  p.parts = reinterpret_cast<int2*>(ws + w.segs);
  p.scores = mass ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  p.score_ld = w.score_ld;
  const bool split = paged_split((int64_t)b * hkv * p.hv_per_kv, slots) || (mass && p.hv_per_kv > 1);
  cudaStream_t st = (cudaStream_t)stream;
  const int d = pad_dh(dh);
  if (dtype == ONE_DTYPE_F32) {
    if (rows == 1) {
      switch (d) {
        case 32: return attend<PaF32<32, 1>>(p, split, st);
        case 64: return attend<PaF32<64, 1>>(p, split, st);
        case 96: return attend<PaF32<96, 1>>(p, split, st);
        default: return attend<PaF32<128, 1>>(p, split, st);
      }
    }
    switch (d) {
      case 32: return attend<PaF32<32, 4>>(p, split, st);
      case 64: return attend<PaF32<64, 4>>(p, split, st);
      case 96: return attend<PaF32<96, 4>>(p, split, st);
      default: return attend<PaF32<128, 4>>(p, split, st);
    }
  }
  if (rows == 16) {
    switch (d) {
      case 32: return attend<PaBf16<32, true>>(p, split, st);
      case 64: return attend<PaBf16<64, true>>(p, split, st);
      case 96: return attend<PaBf16<96, true>>(p, split, st);
      default: return attend<PaBf16<128, true>>(p, split, st);
    }
  }
  switch (d) {
    case 32: return attend<PaBf16<32, false>>(p, split, st);
    case 64: return attend<PaBf16<64, false>>(p, split, st);
    case 96: return attend<PaBf16<96, false>>(p, split, st);
    default: return attend<PaBf16<128, false>>(p, split, st);
  }
}

extern "C" int one_paged_append(const one_paged_cache* cache, const one_paged_tokens* tokens, void* stream) {
  if (!tokens || !tokens->k || !tokens->v || !tokens->q != !tokens->q_out || !tokens->cos != !tokens->sin)
    return fail(ONE_ERR_INVALID, "paged append: null argument");
  PagedAppendParams p = {};
  int rc = check_cache(p.c, cache);
  if (rc) return rc;
  const one_paged_tokens& x = *tokens;
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh, dtype = cache->dtype, n = x.n, hq = x.hq;
  if (n < 1 || (x.q && hq < 1)) return fail(ONE_ERR_INVALID, "paged append: sizes must be positive");
  if (x.cos && x.cos_batch != 1 && x.cos_batch != b) return fail(ONE_ERR_INVALID, "cos_batch must be 1 or b");
  const void *k = x.k, *v = x.v, *q = x.q, *cosv = x.cos, *sinv = x.sin;
  p.k = k; p.v = v; p.q = q;
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = x.k_strides[i];
    p.vs[i] = x.v_strides[i];
    p.qs[i] = x.q_strides[i];
  }
  p.cosv = cosv; p.sinv = sinv; p.cos_bs = x.cos_batch == 1 ? 0 : (int64_t)n * dh; p.counts = x.counts;
  p.mass = cache->mass; p.mass_width = cache->mass_width; p.q_out = x.q_out; p.N = n; p.Hq = hq;
  // 16-byte pieces need aligned rows of whole pieces, a power of two of them or two halves; anything else
  // goes element by element
  const int64_t unit = 16 / elem_bytes(dtype);
  auto aligned = [&](const void* at, const int64_t* s) {
    return (reinterpret_cast<uintptr_t>(at) & 15) == 0 && s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0;
  };
  const int pieces = dh % unit == 0 ? dh / (int)unit : 0;
  const bool vec = pieces >= 2 && pieces % 2 == 0 && aligned(k, p.ks) && aligned(v, p.vs) && (!q || aligned(q, p.qs)) &&
                   ((reinterpret_cast<uintptr_t>(x.q_out) | reinterpret_cast<uintptr_t>(cosv) | reinterpret_cast<uintptr_t>(sinv)) & 15) == 0;
  const bool pair = (pieces & (pieces - 1)) != 0;
  const int64_t rows = 2 * (int64_t)hkv + (q ? hq : 0);
  auto groups = [](int64_t heads) { return (heads + kAppendRows - 1) / kAppendRows; };
  const int64_t threads = vec ? n * (2 * groups(hkv) + groups(q ? hq : 0)) * (pair ? pieces / 2 : pieces) : n * rows * 32;
  if (threads > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged append: too many rows");
  const dim3 grid((unsigned)((threads + 255) / 256), b);
  cudaStream_t st = (cudaStream_t)stream;
  auto append = [&](auto t, auto c) {
    using T = decltype(t);
    using C = decltype(c);
    return !vec   ? launch(paged_append_any_kernel<T, C>, grid, dim3(256), 0, st, p)
           : pair ? launch(paged_append_kernel<T, C, true>, grid, dim3(256), 0, st, p)
                  : launch(paged_append_kernel<T, C, false>, grid, dim3(256), 0, st, p);
  };
  return launched(dtype == ONE_DTYPE_F32   ? append(float(0), float(0))
                  : x.cos && x.tables_fp32 ? append(__nv_bfloat16(), float(0))
                                           : append(__nv_bfloat16(), __nv_bfloat16()),
                  "paged append");
}

extern "C" int one_paged_evict(const one_paged_cache* cache, const int32_t* dst_table, int64_t dst_stride,
                               int32_t dst_max_pages, int32_t budget, int32_t recent, int32_t sink, float* mass_out,
                               int64_t mass_out_width, int32_t* kept, void* stream) {
  PagedEvictParams p = {};
  if (!dst_table || !mass_out || !kept || !cache || !cache->mass) return fail(ONE_ERR_INVALID, "paged evict: null argument");
  int rc = check_cache(p.c, cache);
  if (rc) return rc;
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh, dtype = cache->dtype, page_size = cache->page_size;
  if (budget < 1 || recent < 0 || sink < 0 || (int64_t)recent + sink > budget)
    return fail(ONE_ERR_INVALID, "paged evict: 1 <= budget, 0 <= recent, sink and recent + sink <= budget");
  if (dst_max_pages < 1 || dst_stride < dst_max_pages || (int64_t)dst_max_pages * page_size < budget)
    return fail(ONE_ERR_INVALID, "paged evict: the destination pages hold fewer slots than the budget");
  if (mass_out_width < budget) return fail(ONE_ERR_INVALID, "paged evict: mass rows are too short");
  if (mass_out_width > 0x3fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged evict: too many rows");
  p.dst = dst_table; p.dst_stride = dst_stride; p.mass = cache->mass; p.mass_width = cache->mass_width;
  p.budget = budget; p.recent = recent; p.sink = sink; p.mass_out = mass_out; p.out_width = mass_out_width; p.kept = kept;
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t slots = (int64_t)cache->max_pages * page_size, heads = (int64_t)b * hkv;
  const int64_t parts = (budget + 255) / 256, per_bh = (mass_out_width + kMovePlaces - 1) / kMovePlaces;
  // where the CTAs fit the SMs at once: two per SM, one of those that hold 64 keys per thread (192 CTAs of
  // those, 48 heads of 30000 slots to 1000: 49 us in one launch, 29 in two; device times)
  const bool one_launch = heads * parts <= (slots > 16384 && slots <= 32768 ? 1 : 2) * num_sms();
  if (heads * std::max(parts, per_bh) > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged evict: too many rows");
  const int pieces = dh * elem_bytes(dtype) / 16;
  auto evict = [&](auto keys) {
    constexpr int KPT = decltype(keys)::value;
    return one_launch ? launch(paged_evict_kernel<KPT, true>, dim3((unsigned)(heads * parts)), dim3(kEvictThreads), 0, st, p,
                               (int)parts, pieces)
                      : launch(paged_evict_kernel<KPT, false>, dim3((unsigned)heads), dim3(kEvictThreads), 0, st, p, 1, pieces);
  };
  rc = launched(slots <= 1024    ? evict(Int<2>())
                : slots <= 2048  ? evict(Int<4>())
                : slots <= 4096  ? evict(Int<8>())
                : slots <= 8192  ? evict(Int<16>())
                : slots <= 16384 ? evict(Int<32>())
                : slots <= 32768 ? evict(Int<64>())
                                 : evict(Int<0>()),
                "paged evict");
  if (rc || one_launch) return rc;
  return launched(launch(paged_move_kernel, dim3((unsigned)(per_bh * heads)), dim3(kMoveThreads), 0, st, p, (int)per_bh, pieces),
                  "paged move");
}

extern "C" int one_process_logits(const one_logits_rules* rules, const void* logits, int64_t ld, int32_t batch,
                                  int32_t vocab, int32_t dtype, float* out, int64_t out_ld, int32_t* best, void* stream) {
  if (!rules || !logits || !out || (!rules->history && rules->history_len))
    return fail(ONE_ERR_INVALID, "process logits: null argument");
  const one_logits_rules& x = *rules;
  int hist_len = x.history_len;
  if (batch < 1 || vocab < 1 || ld < vocab || out_ld < vocab || hist_len < 0 || (hist_len && x.history_ld < hist_len))
    return fail(ONE_ERR_INVALID, "process logits: bad sizes");
  if (vocab > 0x3fffffff) return fail(ONE_ERR_UNSUPPORTED, "process logits: at most 2^30 - 1 tokens");
  if (dtype != ONE_DTYPE_BF16 && dtype != ONE_DTYPE_F32) return fail(ONE_ERR_INVALID, "dtype");
  if (hist_len && x.history_bytes != 4 && x.history_bytes != 8)
    return fail(ONE_ERR_INVALID, "process logits: int32 or int64 history");
  if (!(x.repetition_all > 0.0f)) return fail(ONE_ERR_INVALID, "process logits: the repetition penalty must be positive");
  if ((x.bias && x.bias_ld && x.bias_ld < vocab) || (x.token_mask && x.mask_ld && x.mask_ld < (vocab + 31) / 32))
    return fail(ONE_ERR_INVALID, "process logits: bias or mask rows overlap");
  // a history that no penalty uses is not read
  if (!x.repetition && !x.presence && !x.frequency && x.repetition_all == 1.0f && x.presence_all == 0.0f && x.frequency_all == 0.0f)
    hist_len = 0;
  LogitsParams p = {};
  p.logits = logits; p.ld = ld; p.B = batch; p.V = vocab; p.history = x.history; p.hist_ld = x.history_ld; p.T = hist_len;
  p.starts = x.output_starts; p.rep = x.repetition; p.pres = x.presence; p.freq = x.frequency;
  p.rep1 = x.repetition_all; p.pres1 = x.presence_all; p.freq1 = x.frequency_all;
  p.bias = x.bias; p.bias_ld = x.bias_ld; p.mask = reinterpret_cast<const uint32_t*>(x.token_mask); p.mask_ld = x.mask_ld;
  p.out = out; p.out_ld = out_ld; p.best = best;
  cudaStream_t st = (cudaStream_t)stream;
  // CTAs per row (at most a portable cluster) until there are two per SM, each with a few tokens per thread;
  // no more, since every CTA reads the row's whole history (256 rows of 32000 tokens, 2176 ids: 18.8 us
  // with 1 CTA per row, 24.9 with 2; 148 rows, 500 ids: 14.1 and 10.6; calls back to back).
  int ctas = 1;
  while (ctas < 8 && (int64_t)batch * ctas <= num_sms() && vocab > ctas * kLogitsThreads * 8) ctas *= 2;
  const int slice = ((vocab + ctas - 1) / ctas + 31) / 32 * 32;
  if ((int64_t)batch * ctas > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "process logits: too many rows");
  const bool wide = hist_len > 32767;  // a count may not fit 15 bits
  const size_t smem = hist_len ? std::min<size_t>((size_t)slice * (wide ? 4 : 2), kLogitsBytes) + 32 : 0;
  const bool full = (int64_t)batch * ctas > 2 * num_sms();
  static std::atomic<bool> done[16][kMaxDevices];
  auto run = [&](auto t, auto i, auto w, auto per_sm) -> int {
    using T = decltype(t);
    using I = decltype(i);
    constexpr int WIDE = decltype(w)::value, PER_SM = decltype(per_sm)::value;
    auto* kernel = logits_kernel<T, I, WIDE != 0, PER_SM>;
    const int rc = allow_smem(kernel, kLogitsBytes + 32, done[(sizeof(T) == 4) * 8 + (sizeof(I) == 8) * 4 + WIDE * 2 + (PER_SM == 3)]);
    if (rc) return rc;
    return launched(launch_cluster(ctas, kernel, dim3((unsigned)batch * ctas), dim3(kLogitsThreads), smem, st, p, slice, ctas),
                    "process logits");
  };
  auto by_rows = [&](auto t, auto i, auto w) { return full ? run(t, i, w, Int<3>()) : run(t, i, w, Int<2>()); };
  auto by_counts = [&](auto t, auto i) { return wide ? by_rows(t, i, Int<1>()) : by_rows(t, i, Int<0>()); };
  if (dtype == ONE_DTYPE_BF16)
    return x.history_bytes == 8 ? by_counts(__nv_bfloat16(), int64_t(0)) : by_counts(__nv_bfloat16(), int32_t(0));
  return x.history_bytes == 8 ? by_counts(float(0), int64_t(0)) : by_counts(float(0), int32_t(0));
}
