// The two kernels of the attention over pages of 8 bits, for requests of few rows and of tiles of them.
#pragma once

#include "qd_host.h"
#include "qd_paged_dev.cuh"
#include "qd_paged_line.h"

namespace qd {

// Scratch of the paged attentions: tickets [grid][2], then the pieces of cut units, as large as two tiles' at most.
struct PagedAttnPlan {
  int64_t off_partials, bytes;
};
inline PagedAttnPlan paged_attn_plan(int grid, int head_dim) {
  PagedAttnPlan p;
  p.off_partials = ((int64_t)grid * 2 * 4 + 255) / 256 * 256;  // the tickets first
  p.bytes = p.off_partials + (int64_t)2 * grid * 2 * 128 * (head_dim * 4 + 8);
  return p;
}

// Of the attention over pages of 8 bits, whose two kernels may run at once: the tickets of both ([grid][2] each), then the
// pieces of each.
constexpr int kF8Resident = 2;  // CTAs an SM of the kernel for few rows
struct Paged8Plan {
  int64_t off_few_tickets, off_tiles, off_few, bytes;
};
inline Paged8Plan paged8_plan(int grid, int head_dim) {
  Paged8Plan p;
  p.off_few_tickets = (int64_t)grid * 2 * 4;
  p.off_tiles = ((int64_t)grid * 4 * 4 + 255) / 256 * 256;
  p.off_few = p.off_tiles + (int64_t)2 * grid * 2 * 128 * (head_dim * 4 + 8);
  p.bytes = p.off_few + (int64_t)2 * grid * kF8Resident * kFewRows * (head_dim * 4 + 8);
  return p;
}

// positions in a row of the page table, as many as are attended to
inline int pg_room(const PagedBatch& b) {
  const int64_t room = (int64_t)b.max_pages * b.page_size;
  return room < kPgMaxKeys ? (int)room : kPgMaxKeys;
}

// A row of work of the attention over shared beginnings: token rows row0 .. row0 + n - 1, the first at position pos0, over
// the keys from block jb to kv of the page table's row table_row. layer: the fp32 rows that the results go to (0: of keys
// that are shared, 1: of a request's own), or -1: straight out.
struct alignas(16) PgShared {
  int row0, n, pos0, kv;
  int jb, table_row, layer, group_row0;  // (the last: a request's, where layer is 1)
};
// A unit of common keys, known by its first token row and KV head: its first CTA and the number of its pieces in the
// scratch (0: it was not cut, and is in the rows). Piece p has slot 2 (cta + p) + (p == 0).
struct alignas(8) PgUnit {
  int cta, pieces;  // (kFew: the pieces are of few rows)
  static constexpr int kFew = 1 << 30;
};
// The 16-bit attention over `entries` such rows of work; rows and rows_lse: 2 layers of [tokens][nq] rows.
int launch_shared(const PagedBatch& b, const PgShared* shared, int entries, float* rows, float* rows_lse, PgUnit* units,
                  const void* q, int64_t ldq, int dtype, int head_dim, const void* k_pages, const void* v_pages, float scale, void* out,
                  int64_t ldo, float* lse, int64_t ld_lse, int grid, void* scratch, int pdl, cudaStream_t stream);

// A checked call over pages of 8 bits.
struct Paged8Call {
  PagedBatch b;
  const void *q, *k_pages, *v_pages, *k_scale, *v_scale;
  void* out;
  float* lse;
  int64_t ldq, ldo, ld_lse, ss_page, ss_head;
  int dtype, head_dim, grid, pdl;
  float scale;
  void* scratch;
  cudaStream_t stream;
};
// The requests of at most 16 query rows a KV head (of none, where a group of heads is larger). `beside`: launch_tiles8
// came right before, for the rest; without it their rows are left as they are and flagged.
int launch_few8(const Paged8Call& c, bool beside);
// The requests of `least` tokens and more, in tiles of 128 query rows.
int launch_tiles8(const Paged8Call& c, int least);
// Maps of the values: a box is a page of a KV head as rows of `row` bytes (head_dim or 128), swizzled over as many.
int map_pools8(const Paged8Call& c, PFN_cuTensorMapEncodeTiled_v12000 encode, int row, CUtensorMap* tk, CUtensorMap* tv);

}  // namespace qd
