// extern "C" operators of one serving step over a paged key-value cache held in 4 or 8 bits (one_b200.h).
#include "paged_plan.cuh"
#include "paged_quant.cuh"
#include "paged_quant_attn.cuh"
#include "serving_host.cuh"

using namespace one;

namespace {

int check_quant(PagedQuant& m, const one_paged_quant_cache* x) {
  int rc = check_table(m.c, x, 16);
  if (rc) return rc;
  if (!x->scales) return fail(ONE_ERR_INVALID, "paged cache: null argument");
  if (x->bits != 4 && x->bits != 8) return fail(ONE_ERR_INVALID, "paged cache: 4 or 8 bits");
  m.row = x->dh * x->bits / 8;
  m.groups = (x->dh + kQuantGroup - 1) / kQuantGroup;
  const int64_t rows = (int64_t)x->hkv * x->page_size, ks = x->k_page_stride, vs = x->v_page_stride, ss = x->scale_page_stride;
  if (std::max({ks, vs, ss, rows * x->dh}) > 0x7fffffff)
    return fail(ONE_ERR_UNSUPPORTED, "paged cache: pages of at most 2^31 - 1 elements");
  if (ks < rows * m.row || vs < rows * m.row || ss < rows * 2 * m.groups) return fail(ONE_ERR_INVALID, "paged cache: pages overlap");
  if (((reinterpret_cast<uintptr_t>(x->k_pages) | reinterpret_cast<uintptr_t>(x->v_pages) | ks | vs) & 7) ||
      ((reinterpret_cast<uintptr_t>(x->scales) | 2 * ss) & 3))
    return fail(ONE_ERR_INVALID, "paged cache: codes must start on 8-byte boundaries, scales on 4-byte ones");
  m.c.k = x->k_pages; m.c.v = x->v_pages; m.c.k_stride = ks; m.c.v_stride = vs;
  m.scales = x->scales; m.s_stride = ss;
  m.c.err = reinterpret_cast<DevErr*>(one_ops_err_record());
  return ONE_OK;
}

int check_dtype(int dtype) {
  return dtype == ONE_DTYPE_BF16 || dtype == ONE_DTYPE_F32 ? ONE_OK : fail(ONE_ERR_INVALID, "paged cache: dtype");
}

}  // namespace

extern "C" int one_paged_quant_append(const one_paged_quant_cache* cache, const one_paged_tokens* tokens, int32_t dtype,
                                      void* stream) {
  if (!tokens || !tokens->k || !tokens->v || !tokens->q != !tokens->q_out || !tokens->cos != !tokens->sin)
    return fail(ONE_ERR_INVALID, "paged append: null argument");
  PagedQuant m = {};
  int rc = check_quant(m, cache);
  if (!rc) rc = check_dtype(dtype);
  if (rc) return rc;
  const one_paged_tokens& x = *tokens;
  if (x.n < 1 || (x.q && x.hq < 1)) return fail(ONE_ERR_INVALID, "paged append: sizes must be positive");
  if (x.cos && x.cos_batch != 1 && x.cos_batch != cache->b) return fail(ONE_ERR_INVALID, "cos_batch must be 1 or b");
  QuantAppendParams p = {};
  p.scales = m.scales; p.s_stride = m.s_stride; p.row = m.row; p.groups = m.groups;
  p.a.c = m.c; p.a.k = x.k; p.a.v = x.v; p.a.q = x.q;
  for (int i = 0; i < 3; ++i) {
    p.a.ks[i] = x.k_strides[i];
    p.a.vs[i] = x.v_strides[i];
    p.a.qs[i] = x.q_strides[i];
  }
  p.a.cosv = x.cos; p.a.sinv = x.sin; p.a.cos_bs = x.cos_batch == 1 ? 0 : (int64_t)x.n * cache->dh; p.a.counts = x.counts;
  p.a.mass = cache->mass; p.a.mass_width = cache->mass_width; p.a.q_out = x.q_out; p.a.N = x.n; p.a.Hq = x.hq;
  // whole 16-byte pieces of rows; anything else goes element by element
  const int64_t unit = 16 / elem_bytes(dtype);
  auto aligned = [&](const void* at, const int64_t* s) {
    return (reinterpret_cast<uintptr_t>(at) & 15) == 0 && s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0;
  };
  const bool vec = aligned(x.k, x.k_strides) && aligned(x.v, x.v_strides) && (!x.q || aligned(x.q, x.q_strides)) &&
                   ((reinterpret_cast<uintptr_t>(x.q_out) | reinterpret_cast<uintptr_t>(x.cos) | reinterpret_cast<uintptr_t>(x.sin)) & 15) == 0;
  const int64_t hq = x.q ? x.hq : 0, per = 32 / (cache->dh / 8), rows = dtype == ONE_DTYPE_F32 ? kQuantRows<float> : kQuantRows<__nv_bfloat16>;
  auto groups = [&](int64_t heads) { return (heads + rows - 1) / rows; };
  const int64_t all = x.n * (2 * (int64_t)cache->hkv + hq), kinds = 2 * groups(cache->hkv) + groups(hq);
  if (all > 0x7fffffff / 32 || kinds > 65535) return fail(ONE_ERR_UNSUPPORTED, "paged append: too many rows");
  p.per = (int)per;
  p.lane_m = (1024 + cache->dh / 8 - 1) / (cache->dh / 8);
  const int64_t warps = (x.n + per - 1) / per, block = std::min<int64_t>(8, warps);  // of a kind and group of heads
  const dim3 grid = vec ? dim3((unsigned)((warps + block - 1) / block), cache->b, (unsigned)kinds) : dim3((unsigned)((all + 7) / 8), cache->b);
  const dim3 threads((unsigned)(vec ? 32 * block : 256));
  cudaStream_t st = (cudaStream_t)stream;
  auto append = [&](auto t, auto c) {
    using T = decltype(t);
    using C = decltype(c);
    if (cache->bits == 4)
      return vec ? launch(quant_append_kernel<T, C, 4>, grid, threads, 0, st, p) : launch(quant_append_any_kernel<T, C, 4>, grid, threads, 0, st, p);
    return vec ? launch(quant_append_kernel<T, C, 8>, grid, threads, 0, st, p) : launch(quant_append_any_kernel<T, C, 8>, grid, threads, 0, st, p);
  };
  return launched(dtype == ONE_DTYPE_F32   ? append(float(0), float(0))
                  : x.cos && x.tables_fp32 ? append(__nv_bfloat16(), float(0))
                                           : append(__nv_bfloat16(), __nv_bfloat16()),
                  "paged append");
}

extern "C" int one_paged_quant_read(const one_paged_quant_cache* cache, const int32_t* starts, int32_t n, int32_t dtype, void* k,
                                    void* v, void* stream) {
  if (!k || !v) return fail(ONE_ERR_INVALID, "paged read: null argument");
  QuantReadParams p = {};
  int rc = check_quant(p.m, cache);
  if (!rc) rc = check_dtype(dtype);
  if (rc) return rc;
  if (n < 1) return fail(ONE_ERR_INVALID, "paged read: sizes must be positive");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
    return fail(ONE_ERR_INVALID, "paged read: k and v must start on 16-byte boundaries");
  p.starts = starts; p.k = k; p.v = v; p.N = n;
  const int64_t threads = (int64_t)n * (cache->dh / 8), heads = (cache->hkv + kReadHeads - 1) / kReadHeads;
  if (threads > 0x7fffffff) return fail(ONE_ERR_UNSUPPORTED, "paged read: too many rows");
  const dim3 grid((unsigned)((threads + 255) / 256), cache->b, (unsigned)heads);
  cudaStream_t st = (cudaStream_t)stream;
  auto read = [&](auto t) {
    using T = decltype(t);
    return cache->bits == 4 ? launch(quant_read_kernel<T, 4>, grid, dim3(256), 0, st, p)
                            : launch(quant_read_kernel<T, 8>, grid, dim3(256), 0, st, p);
  };
  return launched(dtype == ONE_DTYPE_F32 ? read(float(0)) : read(__nv_bfloat16()), "paged read");
}

namespace {

// Query heads that one pass over a kv head's cache serves.
int quant_rows(int dtype, int G) { return G <= 4 ? 4 : dtype == ONE_DTYPE_F32 || G <= 8 ? 8 : 16; }

template <int BITS>
int attend_bits(PagedAttn& p, bool split, int dtype, int rows, cudaStream_t st) {
  auto dims = [&](auto dh) -> int {
    constexpr int DH = decltype(dh)::value;
    if (dtype == ONE_DTYPE_F32)
      return rows == 4 ? attend<PaQuant<DH, BITS, PQ_PAIR4>>(p, split, st) : attend<PaQuant<DH, BITS, PQ_PAIR8>>(p, split, st);
    return rows == 16  ? attend<PaQuant<DH, BITS, PQ_16>>(p, split, st)
           : rows == 8 ? attend<PaQuant<DH, BITS, PQ_8>>(p, split, st)
                       : attend<PaQuant<DH, BITS, PQ_4>>(p, split, st);
  };
  switch (pad_dh(p.c.Dh)) {
    case 32: return dims(Int<32>());
    case 64: return dims(Int<64>());
    case 96: return dims(Int<96>());
    default: return dims(Int<128>());
  }
}

}  // namespace

extern "C" size_t one_paged_quant_attention_workspace_bytes(int32_t b, int32_t hq, int32_t hkv, int32_t dh, int32_t page_size,
                                                            int32_t max_pages, int32_t dtype, int32_t with_mass) {
  if (hq < 1 || hkv < 1) return 0;
  return attention_bytes(b, hq, hkv, dh, quant_rows(dtype, hq / hkv), page_size, max_pages, with_mass != 0, 4 * kPaWarps);
}

extern "C" int one_paged_quant_attention(const one_paged_quant_cache* cache, const void* q, int64_t q_batch_stride,
                                         int64_t q_head_stride, int32_t hq, float scale, int32_t dtype, void* out,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !out) return fail(ONE_ERR_INVALID, "paged attention: null argument");
  PagedQuant m = {};
  int rc = check_quant(m, cache);
  if (!rc) rc = check_dtype(dtype);
  if (rc) return rc;
  const int b = cache->b, hkv = cache->hkv, dh = cache->dh;
  if (hq < 1 || hq % hkv) return fail(ONE_ERR_INVALID, "paged attention: the query heads must be a multiple of the kv heads");
  const int rows = quant_rows(dtype, hq / hkv);
  const size_t need = one_paged_quant_attention_workspace_bytes(b, hq, hkv, dh, cache->page_size, cache->max_pages, dtype, cache->mass != nullptr);
  PagedAttn p = {};
  p.c = m.c; p.scales = (const uint8_t*)m.scales; p.s_stride = 2 * m.s_stride; p.row = m.row;
  const int64_t at = reinterpret_cast<uintptr_t>(m.c.k) | reinterpret_cast<uintptr_t>(m.c.v) | m.c.k_stride | m.c.v_stride;
  p.vec16 = ((at | m.row) & 15) == 0;
  // and places in a pool count in 32 bits of 16 bytes
  p.run = ((at | reinterpret_cast<uintptr_t>(m.scales) | p.s_stride) & 15) == 0 &&
          cache->num_pages * std::max({m.c.k_stride, m.c.v_stride, p.s_stride}) < 0xfffffff0ll * 16;
  bool split;
  rc = plan_attention(p, split, cache, q, q_batch_stride, q_head_stride, hq, rows, 4 * kPaWarps, kQuantUnits, 32, scale, out, workspace, workspace_bytes, need);
  if (rc) return rc;
  return cache->bits == 4 ? attend_bits<4>(p, split, dtype, rows, (cudaStream_t)stream)
                          : attend_bits<8>(p, split, dtype, rows, (cudaStream_t)stream);
}

extern "C" int one_paged_quant_evict(const one_paged_quant_cache* cache, const int32_t* dst_table, int64_t dst_stride,
                                     int32_t dst_max_pages, int32_t budget, int32_t recent, int32_t sink, float* mass_out,
                                     int64_t mass_out_width, int32_t* kept, void* stream) {
  if (!cache || !cache->mass) return fail(ONE_ERR_INVALID, "paged evict: null argument");
  PagedQuant m = {};
  const int rc = check_quant(m, cache);
  if (rc) return rc;
  PagedEvictParams p = {};
  p.c = m.c; p.scales = (uint32_t*)m.scales; p.s_stride = m.s_stride / 2; p.words = m.groups;
  return evict<uint2>(p, cache, m.row / 8, dst_table, dst_stride, dst_max_pages, budget, recent, sink, mass_out, mass_out_width,
                      kept, (cudaStream_t)stream);
}
