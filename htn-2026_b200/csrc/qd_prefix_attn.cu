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
//   merge  joins the layers' rows and the pieces that units of common keys were cut into, a warp per token and head.
// Measured, 32 query and 8 KV heads of 128: 64 users, 4 k common and up to 1 k own keys each, 78 to 84 us, of which the
// plan is 3.5 and the merge some 3 (dependent loads); 4 documents of 16 k keys with 4 answers each 76 to 79 us. The floors
// are 36 and 38; the rest is what the attention kernel loses on short units.
// A group is taken apart again (its requests read all keys, straight to out) where sharing would not pay: see the plan.
#include "qd_host.h"
#include "qd_paged_attn8.h"

namespace qd {

constexpr int kPlanThreads = 1024, kMergeWarps = 8, kMergePieces = 4;

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
    int reader = INT32_MAX;  // the first request with tokens: a row of the page table without any may hold anything
    int64_t apart = 0;  // places of a block of common keys, if each request reads it
    for (int i = lo + lane; i < hi; i += 32) {
      const PgReq r = request(i);
      if (r.n == 0) continue;
      reader = min(reader, i);
      least = min(least, r.pos0);
      first = min(first, r.row0);
      last = max(last, r.row0 + r.n);
      apart += block_weight(a.s, r.n);
      ++some;
    }
    reader = __reduce_min_sync(0xffffffffu, reader);
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
      a.shared[g] = blocks ? PgShared{first, n, blocks * kPgKeys - 1, blocks * kPgKeys, 0, reader, 0, 0} : PgShared{};
    if (blocks)
      for (int i = lo + lane; i < hi; i += 32)
        if (request(i).n > 0) {
          a.shared[a.n_groups + i].jb = blocks;
          a.shared[a.n_groups + i].layer = 1;
          a.shared[a.n_groups + i].group_row0 = first;
        }
  }
}

struct PrefixMergeArgs {
  PagedBatch b;
  PgShape s;
  const PgShared* requests;
  const PgUnit* units;
  const float *partials, *rows, *rows_lse;
  char* out;
  float* lse;
  int64_t ldo, ld_lse;
  int grid;  // of the attention
};

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_kernel(const __grid_constant__ PrefixMergeArgs a) {
  constexpr int kOwn = D / 32;  // dims of a lane
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5), t = w / a.b.nq;
  if (t >= a.b.tokens) return;
  const int h = (int)(w - t * a.b.nq), kvh = h / a.s.group;
  const int i = warp_find_request(a.b.cu, a.b.batch, (int)t, lane);
  if (i >= a.b.batch) return;
  const PgShared request = a.requests[i];
  if (request.layer != 1) return;
  // the token's unit of common keys, and where in it its row is
  const int at = max((int)t - request.group_row0, 0), in_pair = at % (2 * a.s.tpt);
  const int x = in_pair >= a.s.tpt ? 1 : 0, row = (in_pair - x * a.s.tpt) * a.s.group + h - kvh * a.s.group;
  const float2* const pm = reinterpret_cast<const float2*>(a.partials + (int64_t)2 * a.grid * 2 * 128 * D);
  const int64_t layer = a.b.tokens * a.b.nq, out_row = t * a.b.nq + h;
  const PgUnit unit = a.units[((int)t - in_pair < 0 ? 0 : (int)t - in_pair) * (int64_t)a.b.nkv + kvh];
  const bool few = unit.pieces & PgUnit::kFew;
  int pieces = unit.pieces & ~PgUnit::kFew;
  if (unit.cta < 0 || pieces < 0 || pieces > a.grid - unit.cta) pieces = 0;  // (groups that overlap)
  // the sum of what there is, each part with its weight 2^(m - M); the own part first
  float acc[kOwn], M = a.rows_lse[layer + out_row] * 1.4426950408889634f, L = M == -INFINITY ? 0.f : 1.f;
  auto take = [&](const Vec& v, float* f) {
    const float* const e = reinterpret_cast<const float*>(&v);
#pragma unroll
    for (int d = 0; d < kOwn; ++d) f[d] = e[d];
  };
  auto add = [&](const Vec& v, float m, float l) {  // v: the sum of 2^(score - m) V, l of 2^(score - m)
    if (l == 0.f) return;                           // (no key seen)
    const float mn = fmaxf(M, m), fa = M == -INFINITY && L == 0.f ? 0.f : exp2f(M - mn), fb = exp2f(m - mn);
    const float* const e = reinterpret_cast<const float*>(&v);
    M = mn;
    L = L * fa + l * fb;
#pragma unroll
    for (int d = 0; d < kOwn; ++d) acc[d] = acc[d] * fa + e[d] * fb;
  };
  take(__ldcs(reinterpret_cast<const Vec*>(a.rows + (layer + out_row) * D) + lane), acc);
  if (pieces == 0) {
    const float z = a.rows_lse[out_row] * 1.4426950408889634f;
    add(__ldcs(reinterpret_cast<const Vec*>(a.rows + out_row * D) + lane), z, z == -INFINITY ? 0.f : 1.f);
  }
#pragma unroll 1
  for (int q0 = 0; q0 < pieces; q0 += kMergePieces) {
    float2 ml[kMergePieces];
    Vec v[kMergePieces];
#pragma unroll
    for (int q = 0; q < kMergePieces; ++q) {
      const int qq = min(q0 + q, pieces - 1);  // past the last piece: the last again, not counted
      const int64_t tile = (int64_t)(2 * (unit.cta + qq) + (qq == 0 ? 1 : 0)) * 2 + x;
      ml[q] = pm[tile * 128 + row];
      // few rows: [row][D]; tiles: [D / 4][128 rows][4], of which neighbouring heads share the sectors
      v[q] = few ? reinterpret_cast<const Vec*>(a.partials + (tile * 128 + row) * D)[lane]
                 : *reinterpret_cast<const Vec*>(a.partials + ((tile * (D / 4) + lane * kOwn / 4) * 128 + row) * 4 + lane * kOwn % 4);
    }
#pragma unroll
    for (int q = 0; q < kMergePieces; ++q)
      if (q0 + q < pieces) add(v[q], ml[q].x, ml[q].y);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t o[kOwn / 2];
#pragma unroll
  for (int d = 0; d < kOwn / 2; ++d) o[d] = Elem<T>::pack(acc[2 * d] * inv, acc[2 * d + 1] * inv);
  T* const to = reinterpret_cast<T*>(a.out) + t * a.ldo + (int64_t)h * D + lane * kOwn;
  if constexpr (D == 128)
    *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
  else
    *reinterpret_cast<uint32_t*>(to) = o[0];
  if (lane == 0 && a.lse) a.lse[t * a.ld_lse + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

// After the attention's own scratch: the rows of work, and the two layers.
struct PrefixPlan {
  int64_t off_shared, off_rows, off_lse, off_units, bytes;
};
static PrefixPlan prefix_plan(int grid, int head_dim, int nq, int nkv, int64_t tokens, int64_t entries) {
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  PrefixPlan p;
  p.off_shared = up(paged_attn_plan(grid, head_dim).bytes);
  p.off_rows = p.off_shared + up(entries * (int64_t)sizeof(PgShared));
  p.off_lse = p.off_rows + up(2 * tokens * nq * head_dim * 4);
  p.off_units = p.off_lse + up(2 * tokens * nq * 4);
  p.bytes = p.off_units + up(tokens * nkv * (int64_t)sizeof(PgUnit));
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
  *scratch_bytes = prefix_plan(*grid, head_dim, nq_heads, nkv_heads, max_tokens, 2 * (int64_t)max_requests).bytes;
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
  const PrefixPlan plan = prefix_plan(grid < 1 ? 1 : grid, head_dim, nq_heads, nkv_heads, tokens, (int64_t)batch + n_groups);
  if (grid < 1 || !scratch || scratch_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(scratch) & 31))
    return set_error(QD_ERR_SCRATCH, "%s: grid %d, %lld tokens, %d requests and %d groups need %lld B of 32-byte aligned scratch (have %lld)",
                     what, grid, (long long)tokens, batch, n_groups, (long long)plan.bytes, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  const int64_t merge_ctas = (tokens * nq_heads + kMergeWarps - 1) / kMergeWarps;
  if (merge_ctas > INT32_MAX || (int64_t)batch + n_groups > INT32_MAX)
    return set_error(QD_ERR_UNSUPPORTED, "%s: %lld tokens, %d requests and %d groups", what, (long long)tokens, batch, n_groups);
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
  PgUnit* const units = reinterpret_cast<PgUnit*>(base + plan.off_units);
  const int ra = launch_shared(p.b, p.shared, batch + n_groups, rows, rows_lse, units, q, ldq, dtype, head_dim, k_pages, v_pages, scale,
                               out, ldo, lse, ld_lse, grid, scratch, pdl, stream);
  if (ra != QD_OK || n_groups == 0) return ra;
  const float* const partials = reinterpret_cast<const float*>(base + paged_attn_plan(grid, head_dim).off_partials);
  PrefixMergeArgs m = {p.b, p.s, p.shared + n_groups, units, partials, rows, rows_lse, static_cast<char*>(out),
                       lse, ldo, ld_lse, grid};
  const bool bf = dtype == QD_BF16;
  const void* fn = head_dim == 128 ? (bf ? (const void*)prefix_merge_kernel<__nv_bfloat16, 128> : (const void*)prefix_merge_kernel<__half, 128>)
                                   : (bf ? (const void*)prefix_merge_kernel<__nv_bfloat16, 64> : (const void*)prefix_merge_kernel<__half, 64>);
  return launch_kernel(fn, dim3((unsigned)merge_ctas), dim3(kMergeWarps * 32), 0, pdl, stream, &m);
}
