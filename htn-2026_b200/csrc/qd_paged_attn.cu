// Causal grouped-query attention of a ragged batch's new tokens over cache pages.
//
// One warp per (token, query head): each lane holds D / 32 dims of the query and of the output, every key
// is one dot product (a butterfly over the warp) and one step of the running softmax
//   m' = max(m, s),  l = l e^(m - m') + e^(s - m'),  o = o e^(m - m') + e^(s - m') v.
#include "qd_host.h"
#include "qd_paged_dev.cuh"

namespace qd {

struct PagedAttnArgs {
  PagedBatch b;
  const char *q, *k_pages, *v_pages;
  char* out;
  float* lse;
  int64_t ldq, ldo, ld_lse;
  float scale;
};

constexpr int kSimpleThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kSimpleThreads) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int kPer = D / 64;  // 32-bit words (pairs of dims) per lane
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kSimpleThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = unit / a.b.nq;
  if (t >= a.b.tokens) return;
  const int h = (int)(unit - t * a.b.nq), kvh = h / (a.b.nq / a.b.nkv);
  const int i = warp_find_request(a.b.cu, a.b.batch, (int)t, lane);
  if (i >= a.b.batch) return;
  int kv = a.b.kv_len[i];
  const int pos = kv - a.b.cu[i + 1] + (int)t;
  if (kv > (int64_t)a.b.max_pages * a.b.page_size) {
    kv = a.b.max_pages * a.b.page_size;
    if (lane == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
  }
  const int n = min(kv, pos + 1);
  float2 q[kPer], o[kPer];
  const uint32_t* qp = reinterpret_cast<const uint32_t*>(a.q + (t * a.ldq + (int64_t)h * D) * 2);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    q[e] = Elem<T>::unpack(qp[lane + 32 * e]);
    o[e] = make_float2(0.f, 0.f);
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < n; ++j) {
    const int page = a.b.table[i * a.b.ld_table + (j >> a.b.page_shift)];
    const bool in = page >= 0 && page < a.b.n_pages;
    if (!in && lane == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
    const int64_t at = ((in ? page : 0) * a.b.ps_page + kvh * a.b.ps_head + (int64_t)(j & (a.b.page_size - 1)) * D) * 2;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(a.k_pages + at);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(a.v_pages + at);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float2 k = Elem<T>::unpack(in ? kp[lane + 32 * e] : 0u);
      s = fmaf(q[e].x, k.x, fmaf(q[e].y, k.y, s));
    }
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s);
    const float up = m == mn ? 1.f : expf(m - mn), p = s == mn ? 1.f : expf(s - mn);
    m = mn;
    l = l * up + p;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float2 v = Elem<T>::unpack(in ? vp[lane + 32 * e] : 0u);
      o[e].x = o[e].x * up + p * v.x;
      o[e].y = o[e].y * up + p * v.y;
    }
  }
  const float inv = n > 0 ? 1.f / l : 0.f;
  uint32_t* op = reinterpret_cast<uint32_t*>(a.out + (t * a.ldo + (int64_t)h * D) * 2);
#pragma unroll
  for (int e = 0; e < kPer; ++e) op[lane + 32 * e] = Elem<T>::pack(o[e].x * inv, o[e].y * inv);
  if (a.lse && lane == 0) a.lse[t * a.ld_lse + h] = n > 0 ? m + logf(l) : -INFINITY;
}

}  // namespace qd

using namespace qd;

extern "C" int qd_paged_attn_plan(int nq_heads, int nkv_heads, int head_dim, int grid_hint, int* grid,
                                  int64_t* scratch_bytes) {
  if (!grid || !scratch_bytes) return set_error(QD_ERR_ARG, "paged attention plan: null result");
  if (nkv_heads < 1 || nq_heads < nkv_heads || nq_heads % nkv_heads || (head_dim != 64 && head_dim != 128))
    return set_error(QD_ERR_UNSUPPORTED, "paged attention: %d query heads over %d KV heads of %d", nq_heads,
                     nkv_heads, head_dim);
  *grid = grid_hint > 0 ? grid_hint : host_sm_count();
  *scratch_bytes = 16;
  return QD_OK;
}

extern "C" int qd_paged_attn(const void* q, int64_t ldq, int dtype, int64_t tokens, int nq_heads, int nkv_heads,
                             int head_dim, const void* k_pages, const void* v_pages, int64_t n_pages, int page_size,
                             int64_t ps_page, int64_t ps_head, const int32_t* cu_tokens, const int32_t* kv_len,
                             int batch, const int32_t* page_table, int64_t ld_table, int max_pages, float scale,
                             void* out, int64_t ldo, float* lse, int64_t ld_lse, int grid, void* scratch,
                             int64_t scratch_bytes, int* err, int pdl, cudaStream_t stream) {
  PagedAttnArgs a = {};
  const int rc = paged_batch_check("paged attention", dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages, v_pages,
                                   n_pages, page_size, ps_page, ps_head, cu_tokens, kv_len, batch, page_table,
                                   ld_table, max_pages, err, &a.b);
  if (rc != QD_OK) return rc;
  if (!q || !out || !aligned16(q) || !aligned16(out) || ldq % 8 || ldo % 8 || ldq < (int64_t)nq_heads * head_dim ||
      ldo < (int64_t)nq_heads * head_dim || (lse && ld_lse < nq_heads) || !(scale > 0.f))
    return set_error(QD_ERR_ARG, "paged attention: q / out / lse null, misaligned or with a bad stride (%lld, %lld, %lld), or scale %g",
                     (long long)ldq, (long long)ldo, (long long)ld_lse, (double)scale);
  if (grid < 1 || !scratch || scratch_bytes < 16)
    return set_error(QD_ERR_SCRATCH, "paged attention: grid %d, %lld scratch bytes", grid, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  a.q = static_cast<const char*>(q);
  a.k_pages = static_cast<const char*>(k_pages);
  a.v_pages = static_cast<const char*>(v_pages);
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.ldq = ldq;
  a.ldo = ldo;
  a.ld_lse = ld_lse;
  a.scale = scale;
  const int64_t blocks = (tokens * nq_heads + kSimpleThreads / 32 - 1) / (kSimpleThreads / 32);
  if (blocks > INT32_MAX) return set_error(QD_ERR_UNSUPPORTED, "paged attention: %lld tokens", (long long)tokens);
  const void* fn = dtype == QD_BF16 ? (head_dim == 128 ? (const void*)paged_attn_kernel<__nv_bfloat16, 128>
                                                       : (const void*)paged_attn_kernel<__nv_bfloat16, 64>)
                                    : (head_dim == 128 ? (const void*)paged_attn_kernel<__half, 128>
                                                       : (const void*)paged_attn_kernel<__half, 64>);
  return launch_kernel(fn, dim3((unsigned)blocks), dim3(kSimpleThreads), 0, pdl, stream, &a);
}
