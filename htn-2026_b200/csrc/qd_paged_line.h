// The line of work of the paged attention: the key blocks of all its units one after the other, in places, cut
// evenly over the CTAs. Plain C++ for the host too, so that its sums can be checked at sizes that would take the
// GPU minutes.
//
// Places are counted in 64 bits: a prompt of 938,000 tokens with 8 KV heads of 4 query heads each passes 2^31, and
// so do one of 470,000 with 71 query heads on one KV head (heads of 64: 5.4 s on the GPU) and calls of many
// requests. A unit alone stays below 2^27 (2^24 key blocks).
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define QD_LINE_FN __host__ __device__ __forceinline__
#else
#define QD_LINE_FN inline
#endif

namespace qd {

constexpr int kPgKeys = 128;               // keys per block
constexpr int kPgMaxKeys = 0x7fffff00;     // of a request: whole blocks, and one more stays within 32 bits
constexpr int kFewRows = 16;               // rows of a few-row unit (MMA N)
// A key block of a pair of tiles takes 5 places, one of a single tile 4, one of few rows 2 (measured 2.5, 1.8 and
// 1.3 us; the tiles a little more, since their pieces take longer to join), and a unit of tiles 8 more for Q and its
// rows' way out (some 5 us), which few rows' units do not show. 30 single tokens and 2 chunks of 251 after up to
// 2 k keys take 98 us; with 3, 2, 2 and 7 for every unit 128. A CTA takes whole blocks.
constexpr int kPgPairCost = 5, kPgTileCost = 4, kPgBlockCost = 2, kPgUnitCost = 8;
constexpr int kPgPiece = 12;  // places that a CTA takes at least, where units are whole tiles

template <typename T>
QD_LINE_FN T pg_min(T x, T y) {
  return x < y ? x : y;
}
template <typename T>
QD_LINE_FN T pg_max(T x, T y) {
  return x < y ? y : x;
}

// The units of a head layout.
struct PgShape {
  int nkv, group, tpt, tpf;   // heads per KV head; tokens per tile and per 16 rows (0: a group is larger)
  int period, period_blocks;  // ceil sums over tile pairs repeat every `period` pairs, `period_blocks` blocks on
  int few_cost;               // a few-row unit's fixed cost
};
inline PgShape pg_shape(int nq, int nkv) {
  PgShape s;
  s.nkv = nkv;
  s.group = nq / nkv;
  s.tpt = 128 / s.group;
  s.tpf = kFewRows / s.group;
  const int pair = 2 * s.tpt, two = pair & -pair, g = two < kPgKeys ? two : kPgKeys;  // g = gcd(pair, 128)
  s.period = kPgKeys / g;
  s.period_blocks = pair / g;
  s.few_cost = 0;
  return s;
}

// One request on the line.
struct PgReq {
  int row0, n, pos0, kv;  // token rows, the first one's position, keys (cut to `room`)
  int pairs;              // tile pairs
  int jb;                 // key blocks before its first: of keys that other rows of work cover
};
// Token rows begin .. end - 1 of `tokens`; `room` positions in a row of the page table, at most kPgMaxKeys.
QD_LINE_FN PgReq pg_make_request(const PgShape& s, int begin, int end, int kv_len, int tokens, int room) {
  PgReq r;
  end = pg_min(pg_max(end, 0), tokens);
  r.row0 = pg_min(pg_max(begin, 0), end);
  r.n = end - r.row0;
  const int kv = pg_max(kv_len, 0);
  r.pos0 = kv - r.n;
  r.kv = pg_min(kv, room);
  r.pairs = (r.n + 2 * s.tpt - 1) / (2 * s.tpt);
  r.jb = 0;
  return r;
}
// key blocks of tile pair k: up to its last token's position (at least one, so that rows without keys are
// written too)
QD_LINE_FN int pg_blocks(const PgShape& s, const PgReq& r, int k) {
  const int keys = pg_min(r.kv, r.pos0 + pg_min(r.n, (k + 1) * 2 * s.tpt));
  return pg_max((keys + kPgKeys - 1) / kPgKeys - r.jb, 1);
}
// places of a key block of tile pair k
QD_LINE_FN int pg_weight(const PgShape& s, const PgReq& r, int k) {
  const int tok = r.n - k * 2 * s.tpt;
  return tok > s.tpt ? kPgPairCost : tok > s.tpf ? kPgTileCost : kPgBlockCost;
}
// and of its fixed cost
QD_LINE_FN int pg_fixed(const PgShape& s, const PgReq& r, int k) {
  return r.n - k * 2 * s.tpt > s.tpf ? kPgUnitCost : s.few_cost;
}
QD_LINE_FN int pg_cost(const PgShape& s, const PgReq& r, int k) {
  return pg_fixed(s, r, k) + pg_weight(s, r, k) * pg_blocks(s, r, k);
}
// sum of pg_cost over the request's pairs. Where nothing is cut the terms are ceil((pos0 + 2 tpt k) / 128),
// which grow by period_blocks every `period` pairs: one pass over a period suffices (all but the last are pairs).
QD_LINE_FN int64_t pg_sum_cost(const PgShape& s, const PgReq& r) {
  if (r.pairs <= 1) return r.pairs ? pg_cost(s, r, 0) : 0;
  int64_t sum = 0;
  if (r.pos0 >= 0 && r.kv == r.pos0 + r.n) {
    const int m = r.pairs - 1, q = m / s.period, rest = m - q * s.period;
#pragma unroll 1
    for (int j = 1; j <= pg_min(s.period, m); ++j) {
      const int64_t cnt = q + (j <= rest);
      sum += cnt * ((r.pos0 + 2 * s.tpt * j + kPgKeys - 1) / kPgKeys) + s.period_blocks * (cnt * (cnt - 1) / 2);
    }
    return (int64_t)kPgUnitCost * m + kPgPairCost * (sum - (int64_t)m * r.jb) + pg_cost(s, r, m);
  }
#pragma unroll 1
  for (int k = 0; k < r.pairs; ++k) sum += pg_cost(s, r, k);
  return sum;
}
// Where place w of a request is: tile pair, KV head and place in that unit (`whole`: a place per unit).
struct PgPlace {
  int k, h, o;
};
QD_LINE_FN PgPlace pg_place(const PgShape& s, const PgReq& r, int64_t w, bool whole) {
  int k = 0, len = whole ? 1 : pg_cost(s, r, 0);
  while (w >= (int64_t)s.nkv * len) {
    w -= (int64_t)s.nkv * len;
    ++k;
    len = whole ? 1 : pg_cost(s, r, k);
  }
  const int h = (int)(w / len);
  return PgPlace{k, h, (int)(w - (int64_t)h * len)};
}
// The line of `total` places over `ctas` CTAs: the first total % ctas take one more than the others.
struct PgLine {
  int64_t each;
  int more, ctas;
  QD_LINE_FN int64_t begin(int c) const { return c * each + pg_min(c, more); }
  QD_LINE_FN int owner(int64_t at) const {
    const int64_t big = more * (each + 1);
    return at < big ? (int)(at / (each + 1)) : more + (int)((at - big) / each);
  }
};
// With little work the first CTAs take `least` places each, the rest nothing.
QD_LINE_FN PgLine pg_line(int64_t total, int grid, int least) {
  PgLine line;
  line.ctas = (int)pg_min((int64_t)grid, pg_max(total / least, pg_min(total, (int64_t)1)));
  line.each = line.ctas ? total / line.ctas : 0;
  line.more = line.ctas ? (int)(total - line.each * line.ctas) : 0;
  return line;
}

}  // namespace qd
