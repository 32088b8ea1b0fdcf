// Causal grouped-query attention of a ragged batch's new tokens over cache pages of 8 bits.
//
// The simplest kernel that is right: a warp per token and query head walks the keys that the token sees; a lane has
// D / 32 dims of the query, of a key and of the sum. The running maximum and sum of the softmax are fp32.
#include <cuda_fp8.h>

#include <climits>

#include "qd_host.h"
#include "qd_paged_attn8.h"

namespace qd {

struct Attn8Args {
  PagedBatch b;
  const char* q;
  const uint8_t *k_pages, *v_pages, *k_scale, *v_scale;
  char* out;
  float* lse;
  int64_t ldq, ldo, ld_lse, ss_page, ss_head;
  float scale;
  int least;  // requests of fewer tokens are another kernel's
};

__device__ __forceinline__ float held_value(uint8_t code) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(code, __NV_E4M3);
  return __half2float(__half(h));
}

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attn8_kernel(const __grid_constant__ Attn8Args a) {
  constexpr int kOwn = D / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t t = w / a.b.nq;
  if (t >= a.b.tokens) return;
  const int h = (int)(w - t * a.b.nq), kvh = h / (a.b.nq / a.b.nkv);
  const int i = warp_find_request(a.b.cu, a.b.batch, (int)t, lane);
  if (i >= a.b.batch) return;
  if (ld_i32(a.b.cu + i + 1) - ld_i32(a.b.cu + i) < a.least) return;
  const int kv_len = max(ld_i32(a.b.kv_len + i), 0), pos = kv_len - ld_i32(a.b.cu + i + 1) + (int)t;
  const int64_t room = (int64_t)a.b.max_pages << a.b.page_shift;
  if (kv_len > room && lane == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
  const int keys = (int)min((int64_t)min(pos + 1, kv_len), room);
  float q[kOwn], o[kOwn] = {}, m = -INFINITY;
  double l = 0.;  // (as many additions as keys, one after the other)
  const T* row = reinterpret_cast<const T*>(a.q) + t * a.ldq + (int64_t)h * D + lane * kOwn;
#pragma unroll
  for (int d = 0; d < kOwn; ++d) q[d] = (float)row[d] * a.scale;
  for (int p = 0; p < keys; ++p) {
    const int page = ld_i32(a.b.table + i * a.b.ld_table + (p >> a.b.page_shift)), r = p & (a.b.page_size - 1);
    const bool in = page >= 0 && page < a.b.n_pages;
    if (!in && lane == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
    const int64_t at = page * a.b.ps_page + kvh * a.b.ps_head + (int64_t)r * D + lane * kOwn;
    const int64_t sc = page * a.ss_page + kvh * a.ss_head + r;
    const float ks = in ? exp2f((float)a.k_scale[sc] - 127.f) : 0.f, vs = in ? exp2f((float)a.v_scale[sc] - 127.f) : 0.f;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < kOwn; ++d) s = fmaf(q[d], in ? held_value(a.k_pages[at + d]) * ks : 0.f, s);
    s = warp_sum(s);
    const float mn = s > m ? s : m, f = m == -INFINITY ? 0.f : expf(m - mn), e = mn == -INFINITY ? s - s : expf(s - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int d = 0; d < kOwn; ++d) o[d] = o[d] * f + (in ? e * held_value(a.v_pages[at + d]) * vs : 0.f);
  }
  const float inv = l == 0. ? 0.f : (float)(1. / l);
  T* to = reinterpret_cast<T*>(a.out) + t * a.ldo + (int64_t)h * D + lane * kOwn;
#pragma unroll
  for (int d = 0; d < kOwn; ++d) to[d] = (T)(o[d] * inv);
  if (a.lse && lane == 0) a.lse[t * a.ld_lse + h] = l == 0. ? -INFINITY : m + (float)log(l);
}

}  // namespace qd

using namespace qd;

extern "C" int qd_paged_attn8_plan(int nq_heads, int nkv_heads, int head_dim, int grid_hint, int* grid,
                                   int64_t* scratch_bytes) {
  return qd_paged_attn_plan(nq_heads, nkv_heads, head_dim, grid_hint, grid, scratch_bytes);
}

extern "C" int qd_paged_attn8(const void* q, int64_t ldq, int dtype, int64_t tokens, int nq_heads, int nkv_heads,
                              int head_dim, const void* k_pages, const void* v_pages, const void* k_scale,
                              const void* v_scale, int64_t n_pages, int page_size, int64_t ps_page, int64_t ps_head,
                              int64_t ss_page, int64_t ss_head, const int32_t* cu_tokens, const int32_t* kv_len,
                              int batch, const int32_t* page_table, int64_t ld_table, int max_pages, int max_new,
                              float scale, void* out, int64_t ldo, float* lse, int64_t ld_lse, int grid, void* scratch,
                              int64_t scratch_bytes, int* err, int pdl, cudaStream_t stream) {
  constexpr const char* what = "paged attention (8 bits)";
  Attn8Args a = {};
  const int rc = paged_batch_check8(what, dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages, v_pages, k_scale, v_scale,
                                    n_pages, page_size, ps_page, ps_head, ss_page, ss_head, cu_tokens, kv_len, batch,
                                    page_table, ld_table, max_pages, err, &a.b);
  if (rc != QD_OK) return rc;
  if ((tokens > 0 && (!q || !out)) || !aligned16(q) || !aligned16(out) || ldq % 8 || ldo % 8 ||
      ldq < (int64_t)nq_heads * head_dim || ldo < (int64_t)nq_heads * head_dim || (lse && ld_lse < nq_heads) || !(scale > 0.f))
    return set_error(QD_ERR_ARG, "%s: q / out / lse null, misaligned or with a bad stride (%lld, %lld, %lld), or scale %g",
                     what, (long long)ldq, (long long)ldo, (long long)ld_lse, (double)scale);
  int64_t need = 0;
  int g = 0;
  qd_paged_attn8_plan(nq_heads, nkv_heads, head_dim, grid < 1 ? 1 : grid, &g, &need);
  if (grid < 1 || !scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 31))
    return set_error(QD_ERR_SCRATCH, "%s: grid %d needs %lld B of 32-byte aligned scratch (have %lld)", what, grid,
                     (long long)need, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  // Requests of at most `few` tokens have a kernel of their own, and the others one.
  const int few = kFewRows / (nq_heads / nkv_heads);
  const bool only_few = (max_new > 0 && max_new <= few) || tokens <= few;
  if (few > 0) {
    Paged8Call c = {a.b, q, k_pages, v_pages, k_scale, v_scale, out, lse, ldq, ldo, ld_lse, ss_page, ss_head, dtype, head_dim,
                    grid, pdl, scale, scratch, stream};
    const int rf = launch_few8(c, only_few);
    if (rf != QD_OK || only_few) return rf;
  }
  a.least = few + 1;
  a.q = static_cast<const char*>(q);
  a.k_pages = static_cast<const uint8_t*>(k_pages);
  a.v_pages = static_cast<const uint8_t*>(v_pages);
  a.k_scale = static_cast<const uint8_t*>(k_scale);
  a.v_scale = static_cast<const uint8_t*>(v_scale);
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.ldq = ldq;
  a.ldo = ldo;
  a.ld_lse = ld_lse;
  a.ss_page = ss_page;
  a.ss_head = ss_head;
  a.scale = scale;
  const int64_t blocks = (tokens * nq_heads + 3) / 4;
  if (blocks > INT_MAX) return set_error(QD_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)tokens);
  const void* fn = dtype == QD_BF16 ? (head_dim == 128 ? (const void*)paged_attn8_kernel<__nv_bfloat16, 128> : (const void*)paged_attn8_kernel<__nv_bfloat16, 64>)
                                    : (head_dim == 128 ? (const void*)paged_attn8_kernel<__half, 128> : (const void*)paged_attn8_kernel<__half, 64>);
  return launch_kernel(fn, dim3((unsigned)blocks), dim3(128), 0, pdl, stream, &a);
}
