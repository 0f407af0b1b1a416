// extern "C" operators of one serving step over a paged key-value cache and of the logits
// processor (one_b200.h, "serving ops").
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <utility>

#include "../../include/one_b200.h"
#include "common.cuh"
#include "logits.cuh"
#include "paged.cuh"

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

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  static const bool pdl = [] {
    const char* v = getenv("ONE_B200_NO_PDL");
    return !(v && v[0] == '1');
  }();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

int elem_bytes(int dtype) { return dtype == ONE_DTYPE_F32 ? 4 : 2; }

// What every operator over a cache asks of it.
int check_cache(PagedCache& c, void* k_pages, void* v_pages, int64_t ks, int64_t vs, int num_pages, int page_size,
                const int32_t* table, int64_t table_stride, int max_pages, const int32_t* lengths, int b, int hkv,
                int dh, int dtype) {
  if (!k_pages || !v_pages || !table || !lengths) return fail(ONE_ERR_INVALID, "paged cache: null argument");
  if (dtype != ONE_DTYPE_BF16 && dtype != ONE_DTYPE_F32) return fail(ONE_ERR_INVALID, "paged cache: dtype");
  if (num_pages < 1 || page_size < 1 || max_pages < 1 || b < 1 || hkv < 1 || dh < 1)
    return fail(ONE_ERR_INVALID, "paged cache: sizes must be positive");
  if (dh > 128 || dh % 8) return fail(ONE_ERR_UNSUPPORTED, "paged cache: head_dim a multiple of 8, at most 128");
  if (b > 65535 || hkv > 65535) return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 65535 sequences and heads");
  if ((int64_t)max_pages * page_size > 0x3fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: at most 2^30 - 1 slots per sequence");
  if (table_stride < max_pages) return fail(ONE_ERR_INVALID, "paged cache: block table rows overlap");
  const int64_t page = (int64_t)hkv * page_size * dh, es = elem_bytes(dtype);
  if (ks < page || vs < page) return fail(ONE_ERR_INVALID, "paged cache: pages overlap");
  if (((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) || ks * es % 16 || vs * es % 16)
    return fail(ONE_ERR_INVALID, "paged cache: pages must start on 16-byte boundaries");
  c.k = k_pages; c.v = v_pages; c.k_stride = ks; c.v_stride = vs;
  c.table = table; c.table_stride = table_stride; c.lengths = lengths;
  c.num_pages = num_pages; c.page_size = page_size; c.max_pages = max_pages; c.B = b; c.Hkv = hkv; c.Dh = dh;
  c.err = reinterpret_cast<DevErr*>(one_ops_err_record());
  return ONE_OK;
}

int launched(cudaError_t e, const char* what) {
  return e == cudaSuccess ? ONE_OK : fail(ONE_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" size_t one_paged_attention_workspace_bytes(int32_t b, int32_t hq, int32_t hkv, int32_t dh, int32_t page_size,
                                                      int32_t max_pages, int32_t dtype, int32_t with_mass) {
  return 1024;
}

extern "C" int one_paged_attention(const void* q, int64_t q_batch_stride, int64_t q_head_stride, const void* k_pages,
                                   const void* v_pages, int64_t k_page_stride, int64_t v_page_stride, int32_t num_pages,
                                   int32_t page_size, const int32_t* block_table, int64_t table_stride, int32_t max_pages,
                                   const int32_t* lengths, int32_t b, int32_t hq, int32_t hkv, int32_t dh, float scale,
                                   int32_t dtype, float* mass, int64_t mass_width, void* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!q || !out || !workspace) return fail(ONE_ERR_INVALID, "paged attention: null argument");
  PagedAttnParams p = {};
  int rc = check_cache(p.c, const_cast<void*>(k_pages), const_cast<void*>(v_pages), k_page_stride, v_page_stride, num_pages,
                       page_size, block_table, table_stride, max_pages, lengths, b, hkv, dh, dtype);
  if (rc) return rc;
  if (hq < 1 || hq % hkv) return fail(ONE_ERR_INVALID, "paged attention: the query heads must be a multiple of the kv heads");
  if (mass && mass_width < (int64_t)max_pages * page_size)
    return fail(ONE_ERR_INVALID, "paged attention: mass rows are shorter than the block table's slots");
  if (workspace_bytes < one_paged_attention_workspace_bytes(b, hq, hkv, dh, page_size, max_pages, dtype, mass != nullptr))
    return fail(ONE_ERR_INVALID, "workspace too small");
  p.q = q; p.q_bs = q_batch_stride; p.q_hs = q_head_stride; p.G = hq / hkv;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mass = mass; p.mass_width = mass_width; p.out = out;
  const dim3 grid(hkv, b);
  return launched(dtype == ONE_DTYPE_BF16
                      ? launch(paged_attn_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, p)
                      : launch(paged_attn_simple_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, p),
                  "paged attention");
}

extern "C" int one_paged_append(const void* k, int64_t k_batch_stride, int64_t k_head_stride, int64_t k_token_stride,
                                const void* v, int64_t v_batch_stride, int64_t v_head_stride, int64_t v_token_stride,
                                const void* q, int64_t q_batch_stride, int64_t q_head_stride, int64_t q_token_stride,
                                const void* cosv, const void* sinv, int32_t cos_batch, const int32_t* counts, void* k_pages, void* v_pages,
                                int64_t k_page_stride, int64_t v_page_stride, int32_t num_pages, int32_t page_size,
                                const int32_t* block_table, int64_t table_stride, int32_t max_pages,
                                const int32_t* lengths, int32_t b, int32_t n, int32_t hq, int32_t hkv, int32_t dh,
                                int32_t dtype, float* mass, int64_t mass_width, void* q_out, void* stream) {
  if (!k || !v || !q != !q_out || !cosv != !sinv)
    return fail(ONE_ERR_INVALID, "paged append: null argument");
  PagedAppendParams p = {};
  int rc = check_cache(p.c, k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, block_table, table_stride,
                       max_pages, lengths, b, hkv, dh, dtype);
  if (rc) return rc;
  if (n < 1 || (q && hq < 1)) return fail(ONE_ERR_INVALID, "paged append: sizes must be positive");
  if (cosv && cos_batch != 1 && cos_batch != b) return fail(ONE_ERR_INVALID, "cos_batch must be 1 or b");
  if (mass && mass_width < (int64_t)max_pages * page_size)
    return fail(ONE_ERR_INVALID, "paged append: mass rows are shorter than the block table's slots");
  p.k = k; p.v = v; p.q = q;
  p.ks[0] = k_batch_stride; p.ks[1] = k_head_stride; p.ks[2] = k_token_stride;
  p.vs[0] = v_batch_stride; p.vs[1] = v_head_stride; p.vs[2] = v_token_stride;
  p.qs[0] = q_batch_stride; p.qs[1] = q_head_stride; p.qs[2] = q_token_stride;
  p.cosv = cosv; p.sinv = sinv; p.cos_bs = cos_batch == 1 ? 0 : (int64_t)n * dh; p.counts = counts;
  p.mass = mass; p.mass_width = mass_width; p.q_out = q_out; p.N = n; p.Hq = hq;
  const int64_t blocks = ((int64_t)b * n * (2 * hkv + (q ? hq : 0)) + 7) / 8;
  if (blocks > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged append: too many rows");
  const dim3 grid((unsigned)blocks);
  return launched(dtype == ONE_DTYPE_BF16
                      ? launch(paged_append_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, (cudaStream_t)stream, p)
                      : launch(paged_append_simple_kernel<float>, grid, dim3(256), 0, (cudaStream_t)stream, p),
                  "paged append");
}

extern "C" int one_paged_evict(void* k_pages, void* v_pages, int64_t k_page_stride, int64_t v_page_stride,
                               int32_t num_pages, int32_t page_size, const int32_t* block_table, int64_t table_stride,
                               int32_t max_pages, const int32_t* dst_table, int64_t dst_stride, int32_t dst_max_pages,
                               const int32_t* lengths, const float* mass, int64_t mass_width, int32_t b, int32_t hkv,
                               int32_t dh, int32_t dtype, int32_t budget, int32_t recent, int32_t sink, float* mass_out,
                               int64_t mass_out_width, int32_t* kept, void* stream) {
  PagedEvictParams p = {};
  if (!dst_table || !mass || !mass_out || !kept) return fail(ONE_ERR_INVALID, "paged evict: null argument");
  int rc = check_cache(p.c, k_pages, v_pages, k_page_stride, v_page_stride, num_pages, page_size, block_table, table_stride,
                       max_pages, lengths, b, hkv, dh, dtype);
  if (rc) return rc;
  if (budget < 1 || recent < 0 || sink < 0 || (int64_t)recent + sink > budget)
    return fail(ONE_ERR_INVALID, "paged evict: 1 <= budget, 0 <= recent, sink and recent + sink <= budget");
  if (dst_max_pages < 1 || dst_stride < dst_max_pages || (int64_t)dst_max_pages * page_size < budget)
    return fail(ONE_ERR_INVALID, "paged evict: the destination pages hold fewer slots than the budget");
  if (mass_width < (int64_t)max_pages * page_size || mass_out_width < budget)
    return fail(ONE_ERR_INVALID, "paged evict: mass rows are too short");
  if ((int64_t)b * hkv > 65535 || mass_out_width > 0x3fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged evict: too many rows");
  p.dst = dst_table; p.dst_stride = dst_stride; p.mass = mass; p.mass_width = mass_width;
  p.budget = budget; p.recent = recent; p.sink = sink; p.mass_out = mass_out; p.out_width = mass_out_width; p.kept = kept;
  cudaStream_t st = (cudaStream_t)stream;
  rc = launched(launch(paged_select_simple_kernel, dim3(hkv, b), dim3(256), 0, st, p), "paged select");
  if (rc) return rc;
  const dim3 grid((unsigned)((mass_out_width + 7) / 8), b * hkv);
  return launched(dtype == ONE_DTYPE_BF16 ? launch(paged_move_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p)
                                          : launch(paged_move_simple_kernel<float>, grid, dim3(256), 0, st, p),
                  "paged move");
}

extern "C" int one_process_logits(const void* logits, int64_t ld, int32_t batch, int32_t vocab, int32_t dtype,
                                  const void* history, int64_t hist_ld, int32_t hist_len, int32_t hist_bytes,
                                  const int32_t* output_starts, const float* repetition, float repetition_all,
                                  const float* presence, float presence_all, const float* frequency, float frequency_all,
                                  const float* bias, int64_t bias_ld, const int32_t* token_mask, int64_t mask_ld,
                                  float* out, int64_t out_ld, int32_t* best, void* stream) {
  if (!logits || !out || (!history && hist_len)) return fail(ONE_ERR_INVALID, "process logits: null argument");
  if (batch < 1 || vocab < 1 || ld < vocab || out_ld < vocab || hist_len < 0 || (hist_len && hist_ld < hist_len))
    return fail(ONE_ERR_INVALID, "process logits: bad sizes");
  if (vocab > 0x3fffffff) return fail(ONE_ERR_UNSUPPORTED, "process logits: at most 2^30 - 1 tokens");
  if (dtype != ONE_DTYPE_BF16 && dtype != ONE_DTYPE_F32) return fail(ONE_ERR_INVALID, "dtype");
  if (hist_len && hist_bytes != 4 && hist_bytes != 8) return fail(ONE_ERR_INVALID, "process logits: int32 or int64 history");
  if (!(repetition_all > 0.0f)) return fail(ONE_ERR_INVALID, "process logits: the repetition penalty must be positive");
  if ((bias && bias_ld && bias_ld < vocab) || (token_mask && mask_ld && mask_ld < (vocab + 31) / 32))
    return fail(ONE_ERR_INVALID, "process logits: bias or mask rows overlap");
  LogitsParams p = {};
  p.logits = logits; p.ld = ld; p.B = batch; p.V = vocab; p.history = history; p.hist_ld = hist_ld; p.T = hist_len;
  p.starts = output_starts; p.rep = repetition; p.pres = presence; p.freq = frequency;
  p.rep1 = repetition_all; p.pres1 = presence_all; p.freq1 = frequency_all;
  p.bias = bias; p.bias_ld = bias_ld; p.mask = reinterpret_cast<const uint32_t*>(token_mask); p.mask_ld = mask_ld;
  p.out = out; p.out_ld = out_ld; p.best = best;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(batch), block(512);
  const bool bf = dtype == ONE_DTYPE_BF16, wide = hist_bytes == 8;
  return launched(bf ? wide ? launch(logits_simple_kernel<__nv_bfloat16, int64_t>, grid, block, 0, st, p)
                            : launch(logits_simple_kernel<__nv_bfloat16, int32_t>, grid, block, 0, st, p)
                     : wide ? launch(logits_simple_kernel<float, int64_t>, grid, block, 0, st, p)
                            : launch(logits_simple_kernel<float, int32_t>, grid, block, 0, st, p),
                  "process logits");
}
