// Attention of a ragged batch whose requests share their beginnings in groups: each group's common keys are read once.
//
// For a row with the keys C (common) and R (its request's own), with o_X, z_X the softmax's result and log-sum-exp over X,
//   z = log(e^z_C + e^z_R),   out = o_C e^(z_C - z) + o_R e^(z_R - z),
// so the two parts can be computed apart. Three launches:
//   plan   one CTA turns the batch into rows of work (PgShared): for a group, all its requests' tokens over its common
//          keys, without a causal mask, since every one of them is before every new token; for a request, its tokens over
//          the rest of its keys. Common are whole blocks of 128 keys.
//   attn   the 16-bit paged attention (qd_paged_attn.cu) over these rows of work on one line: 64 decoding requests of 4
//          query heads a KV head are a pair of tiles there, so a block of common keys is read, and multiplied, once for
//          all, and both kinds of work fill the SMs together. The results go to fp32 rows, two layers of them, as a second
//          rounding to 16 bits would cost as much as the last.
//   merge  joins the layers' rows, a warp for 8 heads of a token.
// A group is taken apart again (its requests read all keys, straight to out) where sharing would not pay: see the plan.
#include "qd_host.h"
#include "qd_paged_attn8.h"

namespace qd {

constexpr int kPlanThreads = 1024, kMergeWarps = 8, kMergeHeads = 8;

struct PrefixPlanArgs {
  PagedBatch b;
  PgShape s;
  const int32_t *cu_groups, *prefix_len;
  PgShared* shared;  // the groups', then the requests'
  int n_groups, room;
};

// places of a key block of a request's tile pairs, all together (pg_weight)
__device__ __forceinline__ int64_t block_weight(const PgShape& s, int n) {
  PgReq r = {};
  r.n = n;
  const int pairs = (n + 2 * s.tpt - 1) / (2 * s.tpt);
  return pairs ? (int64_t)(pairs - 1) * kPgPairCost + pg_weight(s, r, pairs - 1) : 0;
}

__global__ void __launch_bounds__(kPlanThreads) prefix_plan_kernel(const __grid_constant__ PrefixPlanArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, batch = a.b.batch;
  auto request = [&](int i) {
    return pg_make_request(a.s, ld_i32(a.b.cu + i), ld_i32(a.b.cu + i + 1), ld_i32(a.b.kv_len + i), (int)a.b.tokens, a.room);
  };
  for (int i = threadIdx.x; i < batch; i += kPlanThreads) {
    const PgReq r = request(i);
    if (r.n > 0 && r.kv != r.pos0 + r.n) flag_error(a.b.err, QD_DEVERR_PAGE);
    a.shared[a.n_groups + i] = PgShared{r.row0, r.n, r.pos0, r.kv, 0, i, -1, 0};
  }
  __syncthreads();
  for (int g = warp; g < a.n_groups; g += kPlanThreads / 32) {
    const int lo = min(max(ld_i32(a.cu_groups + g), 0), batch), hi = min(max(ld_i32(a.cu_groups + g + 1), lo), batch);
    int least = INT32_MAX, some = 0, first = INT32_MAX, last = 0;  // first new position; requests with tokens; token rows
    int64_t apart = 0;  // places of a block of common keys, if each request reads it
    for (int i = lo + lane; i < hi; i += 32) {
      const PgReq r = request(i);
      if (r.n == 0) continue;
      least = min(least, r.pos0);
      first = min(first, r.row0);
      last = max(last, r.row0 + r.n);
      apart += block_weight(a.s, r.n);
      ++some;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    first = __reduce_min_sync(0xffffffffu, first);
    last = __reduce_max_sync(0xffffffffu, last);
    some = __reduce_add_sync(0xffffffffu, some);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) apart += __shfl_xor_sync(0xffffffffu, apart, o);
    const int n = some ? last - first : 0;
    // (positions up to the last common key's and the number of tokens together stay within 32 bits)
    const int keys = min(min(ld_i32(a.prefix_len + g), least), min(a.room, kPgMaxKeys - n));
    int blocks = some > 1 && keys > 0 ? keys / kPgKeys : 0;
    // Sharing pays where the places that it saves are more than its own: a unit's fixed cost for each pair of tiles, and
    // as much for the rows' way through memory once more.
    const int pairs = (n + 2 * a.s.tpt - 1) / (2 * a.s.tpt);
    if (blocks * (apart - block_weight(a.s, n)) <= 2 * kPgUnitCost * (int64_t)pairs) blocks = 0;
    if (lane == 0)
      a.shared[g] = blocks ? PgShared{first, n, blocks * kPgKeys - 1, blocks * kPgKeys, 0, lo, 0, 0} : PgShared{};
    if (blocks)
      for (int i = lo + lane; i < hi; i += 32)
        if (request(i).n > 0) {
          a.shared[a.n_groups + i].jb = blocks;
          a.shared[a.n_groups + i].layer = 1;
        }
  }
}

struct PrefixMergeArgs {
  PagedBatch b;
  const PgShared* requests;
  const float *rows, *rows_lse;
  char* out;
  float* lse;
  int64_t ldo, ld_lse;
};

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_kernel(const __grid_constant__ PrefixMergeArgs a) {
  constexpr int kOwn = D / 32;  // dims of a lane
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, per = (a.b.nq + kMergeHeads - 1) / kMergeHeads;
  const int64_t w = (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5), t = w / per;
  if (t >= a.b.tokens) return;
  const int h0 = (int)(w - t * per) * kMergeHeads, heads = min(a.b.nq - h0, kMergeHeads);
  const int i = warp_find_request(a.b.cu, a.b.batch, (int)t, lane);
  if (i >= a.b.batch || ld_i32(&a.requests[i].layer) != 1) return;
  const int64_t row = t * a.b.nq + h0, layer = a.b.tokens * a.b.nq;
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  Vec c[kMergeHeads], o[kMergeHeads];
  float zc[kMergeHeads], zo[kMergeHeads];
#pragma unroll
  for (int k = 0; k < kMergeHeads; ++k) {  // (past the last head: that one again)
    const int64_t at = row + min(k, heads - 1);
    c[k] = __ldcs(reinterpret_cast<const Vec*>(a.rows + at * D) + lane);
    o[k] = __ldcs(reinterpret_cast<const Vec*>(a.rows + (layer + at) * D) + lane);
    zc[k] = __ldcs(a.rows_lse + at);
    zo[k] = __ldcs(a.rows_lse + layer + at);
  }
#pragma unroll
  for (int k = 0; k < kMergeHeads; ++k) {
    if (k >= heads) break;
    const float m = fmaxf(zc[k], zo[k]), base = m == -INFINITY ? 0.f : m;
    const float ec = expf(zc[k] - base), eo = expf(zo[k] - base), sum = ec + eo, inv = sum == 0.f ? 0.f : 1.f / sum;
    const float* const x = reinterpret_cast<const float*>(&c[k]);
    const float* const y = reinterpret_cast<const float*>(&o[k]);
    uint32_t v[kOwn / 2];
#pragma unroll
    for (int d = 0; d < kOwn / 2; ++d)
      v[d] = Elem<T>::pack((x[2 * d] * ec + y[2 * d] * eo) * inv, (x[2 * d + 1] * ec + y[2 * d + 1] * eo) * inv);
    T* const to = reinterpret_cast<T*>(a.out) + t * a.ldo + (int64_t)(h0 + k) * D + lane * kOwn;
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(to) = make_uint2(v[0], v[1]);
    else
      *reinterpret_cast<uint32_t*>(to) = v[0];
    if (lane == 0 && a.lse) a.lse[t * a.ld_lse + h0 + k] = sum == 0.f ? -INFINITY : base + logf(sum);
  }
}

// After the attention's own scratch: the rows of work, and the two layers.
struct PrefixPlan {
  int64_t off_shared, off_rows, off_lse, bytes;
};
static PrefixPlan prefix_plan(int grid, int head_dim, int nq, int64_t tokens, int64_t entries) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  PrefixPlan p;
  p.off_shared = up(paged_attn_plan(grid, head_dim).bytes);
  p.off_rows = p.off_shared + up(entries * (int64_t)sizeof(PgShared));
  p.off_lse = p.off_rows + up(2 * tokens * nq * head_dim * 4);
  p.bytes = p.off_lse + up(2 * tokens * nq * 4);
  return p;
}

}  // namespace qd

using namespace qd;

extern "C" int qd_prefix_attn_plan(int nq_heads, int nkv_heads, int head_dim, int64_t max_tokens, int max_requests,
                                   int grid_hint, int* grid, int64_t* scratch_bytes) {
  const int rc = qd_paged_attn_plan(nq_heads, nkv_heads, head_dim, grid_hint, grid, scratch_bytes);
  if (rc != QD_OK) return rc;
  if (max_tokens < 0 || max_tokens > INT32_MAX || max_requests < 0)
    return set_error(QD_ERR_ARG, "prefix attention plan: %lld tokens, %d requests", (long long)max_tokens, max_requests);
  *scratch_bytes = prefix_plan(*grid, head_dim, nq_heads, max_tokens, 2 * (int64_t)max_requests).bytes;
  return QD_OK;
}

extern "C" int qd_prefix_attn(const void* q, int64_t ldq, int dtype, int64_t tokens, int nq_heads, int nkv_heads,
                              int head_dim, const void* k_pages, const void* v_pages, int64_t n_pages, int page_size,
                              int64_t ps_page, int64_t ps_head, const int32_t* cu_tokens, const int32_t* kv_len,
                              int batch, const int32_t* page_table, int64_t ld_table, int max_pages,
                              const int32_t* cu_groups, const int32_t* prefix_len, int n_groups, float scale, void* out,
                              int64_t ldo, float* lse, int64_t ld_lse, int grid, void* scratch, int64_t scratch_bytes,
                              int* err, int pdl, cudaStream_t stream) {
  constexpr const char* what = "prefix attention";
  PrefixPlanArgs p = {};
  const int rc = paged_batch_check(what, dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages, v_pages, n_pages, page_size,
                                   ps_page, ps_head, cu_tokens, kv_len, batch, page_table, ld_table, max_pages, err, &p.b);
  if (rc != QD_OK) return rc;
  if ((tokens > 0 && (!q || !out)) || !aligned16(q) || !aligned16(out) || ldq % 8 || ldo % 8 || ldq < (int64_t)nq_heads * head_dim ||
      ldo < (int64_t)nq_heads * head_dim || (lse && ld_lse < nq_heads) || !(scale > 0.f))
    return set_error(QD_ERR_ARG, "%s: q / out / lse null, misaligned or with a bad stride (%lld, %lld, %lld), or scale %g",
                     what, (long long)ldq, (long long)ldo, (long long)ld_lse, (double)scale);
  if (ps_head % (8 * head_dim))
    return set_error(QD_ERR_ARG, "%s: head stride %lld (whole groups of 8 rows)", what, (long long)ps_head);
  if (n_groups < 0 || n_groups > batch || (n_groups > 0 && tokens > 0 && (!cu_groups || !prefix_len)))
    return set_error(QD_ERR_ARG, "%s: %d groups of %d requests, or null groups", what, n_groups, batch);
  const PrefixPlan plan = prefix_plan(grid < 1 ? 1 : grid, head_dim, nq_heads, tokens, (int64_t)batch + n_groups);
  if (grid < 1 || !scratch || scratch_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(scratch) & 31))
    return set_error(QD_ERR_SCRATCH, "%s: grid %d, %lld tokens, %d requests and %d groups need %lld B of 32-byte aligned scratch (have %lld)",
                     what, grid, (long long)tokens, batch, n_groups, (long long)plan.bytes, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  char* const base = static_cast<char*>(scratch);
  p.s = pg_shape(nq_heads, nkv_heads);
  p.cu_groups = cu_groups;
  p.prefix_len = prefix_len;
  p.shared = reinterpret_cast<PgShared*>(base + plan.off_shared);
  p.n_groups = n_groups;
  p.room = pg_room(p.b);
  float *const rows = reinterpret_cast<float*>(base + plan.off_rows), *const rows_lse = reinterpret_cast<float*>(base + plan.off_lse);
  const int rp = launch_kernel((const void*)prefix_plan_kernel, dim3(1), dim3(kPlanThreads), 0, pdl, stream, &p);
  if (rp != QD_OK) return rp;
  const int ra = launch_shared(p.b, p.shared, batch + n_groups, rows, rows_lse, q, ldq, dtype, head_dim, k_pages, v_pages, scale,
                               out, ldo, lse, ld_lse, grid, scratch, pdl, stream);
  if (ra != QD_OK || n_groups == 0) return ra;
  PrefixMergeArgs m = {p.b, p.shared + n_groups, rows, rows_lse, static_cast<char*>(out), lse, ldo, ld_lse};
  const int64_t warps = tokens * ((nq_heads + kMergeHeads - 1) / kMergeHeads), ctas = (warps + kMergeWarps - 1) / kMergeWarps;
  if (ctas > INT32_MAX) return set_error(QD_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)tokens);
  const bool bf = dtype == QD_BF16;
  const void* fn = head_dim == 128 ? (bf ? (const void*)prefix_merge_kernel<__nv_bfloat16, 128> : (const void*)prefix_merge_kernel<__half, 128>)
                                   : (bf ? (const void*)prefix_merge_kernel<__nv_bfloat16, 64> : (const void*)prefix_merge_kernel<__half, 64>);
  return launch_kernel(fn, dim3((unsigned)ctas), dim3(kMergeWarps * 32), 0, pdl, stream, &m);
}
