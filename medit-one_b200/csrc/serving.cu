// extern "C" operators of one serving step over a paged key-value cache and of the logits
// processor (one_b200.h, "serving ops").
#include "logits.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_plan.cuh"
#include "serving_host.cuh"

using namespace one;

namespace {

// What every operator over a cache asks of it.
int check_cache(PagedCache& c, const one_paged_cache* x) {
  int rc = check_table(c, x, 8);
  if (rc) return rc;
  if (x->dtype != ONE_DTYPE_BF16 && x->dtype != ONE_DTYPE_F32) return fail(ONE_ERR_INVALID, "paged cache: dtype");
  const int64_t page = (int64_t)x->hkv * x->page_size * x->dh, es = elem_bytes(x->dtype);
  const int64_t ks = x->k_page_stride, vs = x->v_page_stride;
  if (ks > 0x7fffffff || vs > 0x7fffffff || page > 0x7fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: pages of at most 2^31 - 1 elements");
  if (ks < page || vs < page) return fail(ONE_ERR_INVALID, "paged cache: pages overlap");
  if (((reinterpret_cast<uintptr_t>(x->k_pages) | reinterpret_cast<uintptr_t>(x->v_pages)) & 15) || ks * es % 16 || vs * es % 16)
    return fail(ONE_ERR_INVALID, "paged cache: pages must start on 16-byte boundaries");
  c.k = x->k_pages; c.v = x->v_pages; c.k_stride = ks; c.v_stride = vs;
  c.err = reinterpret_cast<DevErr*>(one_ops_err_record());
  return ONE_OK;
}

}  // namespace

extern "C" size_t one_paged_attention_workspace_bytes(int32_t b, int32_t hq, int32_t hkv, int32_t dh, int32_t page_size,
                                                      int32_t max_pages, int32_t dtype, int32_t with_mass) {
  if (hq < 1 || hkv < 1) return 0;
  return attention_bytes(b, hq, hkv, dh, paged_rows(dtype, hq / hkv), page_size, max_pages, with_mass != 0, 3);
}

extern "C" int one_paged_attention(const one_paged_cache* cache, const void* q, int64_t q_batch_stride,
                                   int64_t q_head_stride, int32_t hq, float scale, void* out, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!q || !out) return fail(ONE_ERR_INVALID, "paged attention: null argument");
  PagedAttn p = {};
  int rc = check_cache(p.c, cache);
  if (rc) return rc;
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh, dtype = cache->dtype;
  if (hq < 1 || hq % hkv) return fail(ONE_ERR_INVALID, "paged attention: the query heads must be a multiple of the kv heads");
  const size_t need = one_paged_attention_workspace_bytes(b, hq, hkv, dh, cache->page_size, cache->max_pages, dtype, cache->mass != nullptr);
  const int rows = paged_rows(dtype, hq / hkv);
  bool split;
  rc = plan_attention(p, split, cache, q, q_batch_stride, q_head_stride, hq, rows, 3, 0, 64, scale, out, workspace, workspace_bytes, need);
  if (rc) return rc;
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
  if (!cache || !cache->mass) return fail(ONE_ERR_INVALID, "paged evict: null argument");
  const int rc = check_cache(p.c, cache);
  return rc ? rc
            : evict<uint4>(p, cache, cache->dh * elem_bytes(cache->dtype) / 16, dst_table, dst_stride, dst_max_pages, budget,
                           recent, sink, mass_out, mass_out_width, kept, (cudaStream_t)stream);
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
