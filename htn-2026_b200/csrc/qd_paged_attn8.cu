// Causal grouped-query attention of a ragged batch's new tokens over cache pages of 8 bits: the entry points. Requests of
// at most 16 query rows a KV head (single tokens) run in qd_paged_few8.cu, the others in tiles of 128 rows in
// qd_paged_attn.cu. Two launches, since what bounds them differs (the memory, and the tensor cores with the softmax) and
// with it all of their shared memory and warps. The second does not wait for the first, which waits for what came before
// both, but for its end: its first CTAs run on the SMs that the first leaves, and keep them until the first has ended, so
// the rest of them, which find no room, come after it. A caller that knows that there are no longer requests saves a
// launch.
#include "qd_paged_attn8.h"

using namespace qd;

extern "C" int qd_paged_attn8_plan(int nq_heads, int nkv_heads, int head_dim, int grid_hint, int* grid,
                                   int64_t* scratch_bytes) {
  const int rc = qd_paged_attn_plan(nq_heads, nkv_heads, head_dim, grid_hint, grid, scratch_bytes);
  if (rc == QD_OK) *scratch_bytes = paged8_plan(*grid, head_dim).bytes;
  return rc;
}

extern "C" int qd_paged_attn8(const void* q, int64_t ldq, int dtype, int64_t tokens, int nq_heads, int nkv_heads,
                              int head_dim, const void* k_pages, const void* v_pages, const void* k_scale,
                              const void* v_scale, int64_t n_pages, int page_size, int64_t ps_page, int64_t ps_head,
                              int64_t ss_page, int64_t ss_head, const int32_t* cu_tokens, const int32_t* kv_len,
                              int batch, const int32_t* page_table, int64_t ld_table, int max_pages, int max_new,
                              float scale, void* out, int64_t ldo, float* lse, int64_t ld_lse, int grid, void* scratch,
                              int64_t scratch_bytes, int* err, int pdl, cudaStream_t stream) {
  constexpr const char* what = "paged attention (8 bits)";
  Paged8Call c = {};
  const int rc = paged_batch_check8(what, dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages, v_pages, k_scale, v_scale,
                                    n_pages, page_size, ps_page, ps_head, ss_page, ss_head, cu_tokens, kv_len, batch,
                                    page_table, ld_table, max_pages, err, &c.b);
  if (rc != QD_OK) return rc;
  if ((tokens > 0 && (!q || !out)) || !aligned16(q) || !aligned16(out) || ldq % 8 || ldo % 8 ||
      ldq < (int64_t)nq_heads * head_dim || ldo < (int64_t)nq_heads * head_dim || (lse && ld_lse < nq_heads) || !(scale > 0.f))
    return set_error(QD_ERR_ARG, "%s: q / out / lse null, misaligned or with a bad stride (%lld, %lld, %lld), or scale %g",
                     what, (long long)ldq, (long long)ldo, (long long)ld_lse, (double)scale);
  const int64_t need = paged8_plan(grid < 1 ? 1 : grid, head_dim).bytes;
  if (grid < 1 || !scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 31))
    return set_error(QD_ERR_SCRATCH, "%s: grid %d needs %lld B of 32-byte aligned scratch (have %lld)", what, grid,
                     (long long)need, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  c.q = q;
  c.k_pages = k_pages;
  c.v_pages = v_pages;
  c.k_scale = k_scale;
  c.v_scale = v_scale;
  c.out = out;
  c.lse = lse;
  c.ldq = ldq;
  c.ldo = ldo;
  c.ld_lse = ld_lse;
  c.ss_page = ss_page;
  c.ss_head = ss_head;
  c.dtype = dtype;
  c.head_dim = head_dim;
  c.grid = grid;
  c.pdl = pdl;
  c.scale = scale;
  c.scratch = scratch;
  c.stream = stream;
  const int few = kFewRows / (nq_heads / nkv_heads);  // tokens of a request of few rows
  const bool only_few = (max_new > 0 && max_new <= few) || tokens <= few;
  if (!only_few || few == 0) {
    const int rt = launch_tiles8(c, few + 1);
    if (rt != QD_OK || few == 0) return rt;
  }
  return launch_few8(c, !only_few);
}
