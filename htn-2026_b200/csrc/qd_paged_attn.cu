// Causal grouped-query attention of a ragged batch's new tokens over cache pages, on the tcgen05 tensor cores.
//
// Rows. The query heads of one KV head share its keys, so a tile of 128 MMA rows holds tpt = 128 / group
// tokens x group heads (row = token * group + head), and a work unit is (request, tile pair, KV head): up to
// two such tiles (A, B) that read the same key blocks. A single token fills one tile's first group rows.
// Per block of 128 keys, for each tile x:
//   S_x = Q_x K^T   tcgen05.mma M = 128 rows, N = 128 keys, fp32 in tensor memory
//   softmax         a warpgroup per tile, thread = row: running maximum and sum in fp32,
//                   P = exp2(s * scale * log2 e - m) written over S_x as 16-bit pairs
//   O_x += P_x V    M = 128 rows, N = head_dim, P from tensor memory, V an MN-major operand
// While one warpgroup turns its S into P the tensor cores run the other tile's products. The maximum only
// moves when a row's grows by more than 2^8 (then the warp rescales O_x in tensor memory): O / l does not
// depend on which maximum is used, and 2^8 leaves the fp32 sums and the 16-bit P far from overflow.
//
// Keys and values come page by page: a box of a page's rows x 64 dims per copy (TMA, 128-byte swizzle), the
// lanes of the producer warp issuing one each, into a ring of slots that K and V blocks take in turn. Rows
// past the request's last key hold anything, NaN included: their scores are replaced by -inf before any
// arithmetic, and the MMA warp zeroes their V rows in shared memory (0 x NaN would be NaN).
//
// Split. The key blocks of all units form one line, cut evenly over the CTAs (one per SM) wherever the cuts
// fall: single tokens over long caches, whole prompts and mixtures of them balance alike. A unit that is cut
// leaves fp32 partials (O, m, l) in the scratch, and the CTA that finishes last (a ticket per cut unit)
// joins them in the order of the keys, so results repeat bit for bit. Every CTA finds its place on the line
// from cu_tokens and kv_len itself: no planning launch, and no length is needed on the host.
#include "qd_host.h"
#include "qd_paged_dev.cuh"
#include "qd_umma.cuh"

namespace qd {

constexpr int kPgThreads = 384;  // warps 0-3 softmax A, 4-7 softmax B, 8 producer, 9 MMA, 10-11 only start up
// registers per thread after the start: 2 * 208 + 88 = 3 * 168, what the launch gave the three warpgroups
constexpr int kPgSoftmaxRegs = 208, kPgOtherRegs = 88;
constexpr int kPgKeys = 128;     // keys per block
constexpr int kPgBox = 128 * 128;  // [128 rows][64 dims] of 16 bits
constexpr int kPgUnitCost = 1;     // a unit's fixed cost (Q, epilogue) in key blocks, for the split

struct alignas(64) PagedAttnArgs {
  CUtensorMap tq, tq1, tk, tv;  // tq: a whole tile's rows; tq1: one token's
  PagedBatch b;
  char* out;
  float* lse;
  int64_t ldo, ld_lse;
  int group, tpt;            // heads per KV head, tokens per tile
  int period, period_blocks;  // ceil sums over tile pairs repeat every `period` pairs, `period_blocks` blocks on
  float scale_log2;
  float* partials;  // [2 * grid slots][2 tiles][D / 4][128] float4, then [slots][2][128] float2
  int* tickets;     // [grid][2]
};

template <int D>
struct PgLayout {
  static constexpr int kItem = D / 64 * kPgBox;  // a K or V block, and a Q tile
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int q = 0;
  static constexpr int kv = q + 2 * kItem;
  static constexpr int bars = kv + kSlots * kItem;
  // qfull[2], qempty[2], sfull[2], pfull[2], odone[2], ofree[2], group[2], segfull[4], segempty[4],
  // full[slots], empty[slots]
  static constexpr int nbars = 22 + 2 * kSlots;
  static constexpr int seg = bars + nbars * 8;  // segment ring
  static constexpr int misc = seg + 4 * 64;     // tmem slot, abort, line start, flags, drain counts
  static constexpr int total = misc + 192;
};

// A CTA's piece of a unit: what every warp needs to know of it.
struct PgSeg {
  int row0, ntok, pos0, kv;  // first token row, tokens, the first's position, keys of the request
  int head, j0, nb;          // KV head, first key block, blocks; nb = 0 ends the CTA's list
  int whole;                 // this piece is the whole unit (no partials)
  int slot, c0, nc;          // partial slot, first CTA and number of CTAs of the unit
  int region;                // Q region of a single tile, or -1: both tiles
};
static_assert(sizeof(PgSeg) <= 64, "segment ring entry");

__device__ __forceinline__ void pg_tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ float pg_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float pg_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// One request on the line of key blocks.
struct PgReq {
  int row0, n, pos0, kv;  // token rows, the first one's position, keys (cut to the table row)
  int pairs;              // tile pairs
};
__device__ __forceinline__ PgReq pg_request(const PagedAttnArgs& a, int i) {
  PgReq r;
  const int tok = (int)a.b.tokens;
  const int end = min(max(ld_i32(a.b.cu + i + 1), 0), tok);
  r.row0 = min(max(ld_i32(a.b.cu + i), 0), end);
  r.n = end - r.row0;
  const int kv = max(ld_i32(a.b.kv_len + i), 0);
  r.pos0 = kv - r.n;
  r.kv = (int)min((int64_t)kv, (int64_t)a.b.max_pages * a.b.page_size);
  r.pairs = (r.n + 2 * a.tpt - 1) / (2 * a.tpt);
  return r;
}
// key blocks of tile pair k: up to its last token's position (at least one, so that rows without keys are
// written too)
__device__ __forceinline__ int pg_blocks(const PagedAttnArgs& a, const PgReq& r, int k) {
  const int keys = min(r.kv, r.pos0 + min(r.n, (k + 1) * 2 * a.tpt));
  return max((keys + kPgKeys - 1) / kPgKeys, 1);
}
// sum of pg_blocks over the request's pairs. Where nothing is cut the terms are ceil((pos0 + 2 tpt k) / 128),
// which grow by period_blocks every `period` pairs: one pass over a period suffices.
__device__ __forceinline__ int64_t pg_sum_blocks(const PagedAttnArgs& a, const PgReq& r) {
  if (r.pairs == 0) return 0;
  if (r.pairs == 1) return pg_blocks(a, r, 0);
  int64_t sum = 0;
  if (r.pos0 >= 0 && r.kv == r.pos0 + r.n) {
    const int m = r.pairs - 1, q = m / a.period, rest = m - q * a.period;
    for (int j = 1; j <= min(a.period, m); ++j) {
      const int64_t cnt = q + (j <= rest);
      sum += cnt * ((r.pos0 + 2 * a.tpt * j + kPgKeys - 1) / kPgKeys) + a.period_blocks * (cnt * (cnt - 1) / 2);
    }
    return sum + pg_blocks(a, r, m);
  }
  for (int k = 0; k < r.pairs; ++k) sum += pg_blocks(a, r, k);
  return sum;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPgThreads, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  using Lay = PgLayout<D>;
  constexpr int kHalves = D / 64, kSlots = Lay::kSlots;
  grid_dep_wait();
  extern __shared__ __align__(1024) char smem[];
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need 1 KiB alignment, and there is no room to realign
    if (threadIdx.x == 0 && blockIdx.x == 0) flag_error(a.b.err, kErrSmem);
    return;
  }
  const uint32_t sb = smem_u32(smem), bars = sb + Lay::bars;
  auto qfull = [&](int r) { return bars + 8u * r; };
  auto qempty = [&](int r) { return bars + 16 + 8u * r; };
  auto sfull = [&](int x) { return bars + 32 + 8u * x; };
  auto pfull = [&](int x) { return bars + 48 + 8u * x; };
  auto odone = [&](int x) { return bars + 64 + 8u * x; };
  auto ofree = [&](int x) { return bars + 80 + 8u * x; };
  auto group = [&](int x) { return bars + 96 + 8u * x; };
  auto segfull = [&](int k) { return bars + 112 + 8u * (k & 3); };
  auto segempty = [&](int k) { return bars + 144 + 8u * (k & 3); };
  auto full = [&](int s) { return bars + 176 + 8u * s; };
  auto empty = [&](int s) { return bars + 176 + 8u * (kSlots + s); };
  PgSeg* segs = reinterpret_cast<PgSeg*>(smem + Lay::seg);
  int* misc = reinterpret_cast<int*>(smem + Lay::misc);
  int* abort = misc + 1;
  int64_t* scan = reinterpret_cast<int64_t*>(misc + 16);  // warp totals [12]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int unit_cost = kPgUnitCost;
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(qfull(x), 1);
      mbar_init(qempty(x), 1);
      mbar_init(sfull(x), 1);
      mbar_init(pfull(x), 4);
      mbar_init(odone(x), 1);
      mbar_init(ofree(x), 4);
      mbar_init(group(x), 4);
    }
    for (int k = 0; k < 4; ++k) {
      mbar_init(segfull(k), 1);
      mbar_init(segempty(k), 9);  // the MMA warp and eight softmax warps
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_mbar_init();
    for (int m = 1; m < 16; ++m) misc[m] = 0;
  }
  if (warp == 9) tmem_alloc(smem_u32(misc), 512);

  // ---- this CTA's place on the line: a prefix sum over the requests, and a walk from the one it starts in
  int64_t mine = 0;
  const int per = (a.b.batch + kPgThreads - 1) / kPgThreads;
  const int i0 = min(tid * per, a.b.batch), i1 = min(i0 + per, a.b.batch);
  bool cut = false;
  for (int i = i0; i < i1; ++i) {
    const PgReq r = pg_request(a, i);
    cut |= r.kv != r.pos0 + r.n && r.n > 0;
    mine += a.b.nkv * ((int64_t)unit_cost * r.pairs + pg_sum_blocks(a, r));
  }
  if (cut && blockIdx.x == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_launch();
  int64_t before = 0, W = 0;
  for (int w = 0; w < kPgThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    W += scan[w];
  }
  before += incl - mine;
  // with less than one piece per CTA the first W CTAs take one each, and the rest nothing
  const int G = (int)min((int64_t)gridDim.x, W), cta = blockIdx.x;
  const int64_t begin = cta < G ? part_begin(W, G, cta) : W, end = cta < G ? part_begin(W, G, cta + 1) : W;
  if (mine > 0 && begin >= before && begin < before + mine && begin < end) {
    int64_t w = begin - before;
    int i = i0;
    PgReq r = pg_request(a, i);
    for (;;) {
      const int64_t c = a.b.nkv * ((int64_t)unit_cost * r.pairs + pg_sum_blocks(a, r));
      if (w < c) break;
      w -= c;
      r = pg_request(a, ++i);
    }
    int k = 0;
    for (;; ++k) {
      const int64_t c = (int64_t)a.b.nkv * (unit_cost + pg_blocks(a, r, k));
      if (w < c) break;
      w -= c;
    }
    const int len = unit_cost + pg_blocks(a, r, k);
    misc[2] = i;
    misc[3] = k;
    misc[4] = (int)(w / len);  // KV head
    misc[5] = (int)(w % len);  // place in the unit
  }
  __syncthreads();
  const uint32_t tmem = (uint32_t)misc[0];
  auto tS = [&](int x) { return tmem + 128u * x; };
  auto tO = [&](int x) { return tmem + 256u + 128u * x; };

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPgOtherRegs));
  if (warp == 8) {
    // ------------------------------------------------------------ producer: all lanes walk the line
    const uint64_t pol = policy_evict_normal();
    int64_t at = begin;
    int i = misc[2], k = misc[3], h = misc[4], o = misc[5];
    const int box_rows = min(a.b.page_size, kPgKeys);
    const int boxes = kPgKeys / box_rows * kHalves, box_bytes = box_rows * 128;
    const int my_page = lane / kHalves, my_half = lane % kHalves;
    int seg = 0, item = 0, next_region = 0, qfills[2] = {0, 0};
    bool ok = true;
    PgReq r = {};
    if (at < end) r = pg_request(a, i);
    while (at < end && ok) {
      const int nblk = pg_blocks(a, r, k);
      const int take = (int)min(end - at, (int64_t)(unit_cost + nblk - o));
      const int j0 = max(o - unit_cost, 0), j1 = max(o + take - unit_cost, 0);
      if (j1 > j0) {
        const int64_t first = at - o + unit_cost;  // place of the unit's first block
        const int c0 = part_owner(W, G, first), c1 = part_owner(W, G, first + nblk - 1);
        const int t0 = k * 2 * a.tpt, ntok = min(2 * a.tpt, r.n - t0);
        const bool two = ntok > a.tpt;
        const int ra = two ? 0 : next_region;
        // Q: the regions this unit takes, once their last users' S products are done
        for (int x = 0; x <= (two ? 1 : 0) && ok; ++x) {
          const int reg = two ? x : ra;
          if (qfills[reg] > 0 && !mbar_wait_abort(qempty(reg), (qfills[reg] - 1) & 1, a.b.err, kErrWaitEmpty, abort))
            ok = false;
        }
        if (ok && seg >= 4) ok = mbar_wait_abort(segempty(seg), ((seg >> 2) - 1) & 1, a.b.err, kErrWaitEmpty, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          PgSeg* s = segs + (seg & 3);
          s->row0 = r.row0 + t0;
          s->ntok = ntok;
          s->pos0 = r.pos0 + t0;
          s->kv = r.kv;
          s->head = h;
          s->j0 = j0;
          s->nb = j1 - j0;
          s->whole = j0 == 0 && j1 == nblk;
          s->slot = 2 * cta + (j0 > 0 ? 0 : 1);
          s->c0 = c0;
          s->nc = c1 - c0 + 1;
          s->region = two ? -1 : ra;
          mbar_arrive(segfull(seg));
          for (int x = 0; x <= (two ? 1 : 0); ++x) {
            const int reg = two ? x : ra;
            const bool one = ntok - x * a.tpt == 1;
            mbar_arrive_expect_tx(qfull(reg), kHalves * a.group * (one ? 1 : a.tpt) * 128);
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
              pg_tma_4d(sb + Lay::q + reg * Lay::kItem + hf * kPgBox, one ? &a.tq1 : &a.tq, 64 * hf, 0, h,
                        r.row0 + t0 + x * a.tpt, qfull(reg), pol);
            misc[6 + reg] = qfills[reg] + 1;
          }
        }
        for (int x = 0; x <= (two ? 1 : 0); ++x) ++qfills[two ? x : ra];
        next_region = two ? 0 : 1 - ra;
        ++seg;
        // K and V blocks in turn
        const int32_t* trow = a.b.table + i * a.b.ld_table;
        auto page_of = [&](int j) {  // this lane's page of block j; -2: no box (past the last key)
          const int key = j * kPgKeys + my_page * box_rows;
          return lane < boxes && key < r.kv ? ld_i32(trow + (key >> a.b.page_shift)) : -2;
        };
        int page = page_of(j0);
        for (int j = j0; j < j1 && ok; ++j) {
          const int next = j + 1 < j1 ? page_of(j + 1) : -2;
          const int key = j * kPgKeys + my_page * box_rows;
          const bool need = lane < boxes && key < r.kv;
          const int n_need = __popc(__ballot_sync(0xffffffffu, need));
          if (need && (page < 0 || page >= a.b.n_pages)) {
            flag_error(a.b.err, QD_DEVERR_PAGE);
            page = -1;  // outside the tensor map: the copy fills zeros
          }
          for (int kv = 0; kv < 2; ++kv, ++item) {
            const int s = item % kSlots;
            if (item >= kSlots) {
              const bool got = mbar_wait_abort(empty(s), (item / kSlots - 1) & 1, a.b.err, kErrWaitEmpty, abort);
              if (!__all_sync(0xffffffffu, got)) {
                ok = false;
                break;
              }
            }
            if (lane == 0) {
              mbar_arrive_expect_tx(full(s), n_need * box_bytes);
              misc[8] = item + 1;
            }
            __syncwarp();
            if (need)
              pg_tma_4d(sb + Lay::kv + s * Lay::kItem + my_half * kPgBox + my_page * box_bytes, kv ? &a.tv : &a.tk,
                        64 * my_half, 0, h, page, full(s), pol);
          }
          page = next;
        }
      }
      at += take;
      o = 0;
      if (at < end && ++h == a.b.nkv) {
        h = 0;
        if (++k == r.pairs) {
          k = 0;
          do r = pg_request(a, ++i);
          while (r.pairs == 0);
        }
      }
    }
    // the end of the list: a segment without blocks
    if (ok && seg >= 4) ok = mbar_wait_abort(segempty(seg), ((seg >> 2) - 1) & 1, a.b.err, kErrWaitEmpty, abort);
    if (ok && lane == 0) {
      segs[seg & 3].nb = 0;
      mbar_arrive(segfull(seg));
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA: lane 0 waits and issues
    constexpr uint32_t kTypes = (7u << 7) | (7u << 10), kind = Elem<T>::kBf16 ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t id_s = (umma_idesc_bf16(kPgKeys) & ~kTypes) | kind;
    constexpr uint32_t id_o = (umma_idesc_bf16(D, false, true) & ~kTypes) | kind;
    int item = 0, uses[2] = {0, 0}, sc[2] = {0, 0}, pc[2] = {0, 0}, units[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
    };
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!__all_sync(0xffffffffu, ok)) break;
      const PgSeg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      const int nx = g.region < 0 ? 2 : 1, reg0 = g.region < 0 ? 0 : g.region;
      auto issue_s = [&](int x, int it) {  // S_x = Q_x K^T; its columns held the P that O_x has taken in
        if (sc[x] > 0) wait(odone(x), sc[x] - 1);
        ++sc[x];
        tc_fence_after();
        if (ok) {
          const uint32_t q = sb + Lay::q + (reg0 + x) * Lay::kItem, kt = sb + Lay::kv + it % kSlots * Lay::kItem;
#pragma unroll
          for (int d = 0; d < D / 16; ++d)  // 16 dims per MMA: +32 B inside a 64-dim half, the next half after 4
            umma_bf16(tS(x), umma_desc_sw128(q + (d >> 2) * kPgBox + (d & 3) * 32),
                      umma_desc_sw128(kt + (d >> 2) * kPgBox + (d & 3) * 32), id_s, d > 0 ? 1u : 0u);
        }
        umma_commit(sfull(x));
      };
      auto issue_pv = [&](int x, int it, bool first) {  // O_x += P_x V
        if (first && units[x] > 0) wait(ofree(x), units[x] - 1);
        wait(pfull(x), pc[x]);
        ++pc[x];
        tc_fence_after();
        if (ok) {
          const uint32_t v = sb + Lay::kv + it % kSlots * Lay::kItem;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys per MMA: 8 columns of P pairs; V two 8-key atoms
            umma_bf16_ts(tO(x), tS(x) + 8 * kk, umma_desc_sw128(v + kk * 2048, kPgBox, 1024), id_o,
                         (first && kk == 0) ? 0u : 1u);
        }
        umma_commit(odone(x));
      };
      if (lane == 0) {
        for (int x = 0; x < nx; ++x) wait(qfull(reg0 + x), uses[reg0 + x]);
        wait(full(item % kSlots), item / kSlots);
        for (int x = 0; x < nx; ++x) issue_s(x, item);
        umma_commit(empty(item % kSlots));
        if (g.nb == 1)
          for (int x = 0; x < nx; ++x) umma_commit(qempty(reg0 + x));
      }
      for (int x = 0; x < nx; ++x) ++uses[reg0 + x];
      for (int j = 0; j < g.nb; ++j, item += 2) {
        const int vi = item + 1, ki = item + 2;
        const int rows = g.kv - (g.j0 + j) * kPgKeys;
        if (lane == 0) wait(full(vi % kSlots), vi / kSlots);
        __syncwarp();
        if (rows < kPgKeys) {  // V rows past the last key hold anything: zero them
          char* v = smem + Lay::kv + vi % kSlots * Lay::kItem;
          for (int c = max(rows, 0) * 8 + lane; c < kPgKeys * 8; c += 32)
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
              *reinterpret_cast<uint4*>(v + hf * kPgBox + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          for (int x = 0; x < nx; ++x) {
            issue_pv(x, vi, j == 0);
            if (x == nx - 1) umma_commit(empty(vi % kSlots));
            if (j + 1 < g.nb) {
              if (x == 0) wait(full(ki % kSlots), ki / kSlots);
              issue_s(x, ki);
              if (x == nx - 1) umma_commit(empty(ki % kSlots));
              if (j + 2 == g.nb) umma_commit(qempty(reg0 + x));
            }
          }
        }
        __syncwarp();
      }
      for (int x = 0; x < nx; ++x) ++units[x];
      if (!__all_sync(0xffffffffu, ok)) break;
    }
    if (lane == 0)  // no MMA may still run when its memory is given back
      for (int x = 0; x < 2; ++x)
        if (pc[x] > 0) mbar_wait(odone(x), (pc[x] - 1) & 1, a.b.err, kErrDrain);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPgSoftmaxRegs));
    // ------------------------------------------------------------ softmax and epilogue: warpgroup x = tile x
    const int x = warp >> 2, r = 32 * (warp & 3) + lane;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    int cnt = 0, meets = 0;
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto meet = [&]() {  // the four warps of this tile; bounded, unlike a named barrier
      __syncwarp();
      if (lane == 0) mbar_arrive(group(x));
      wait(group(x), meets++);
    };
    float4* const po = reinterpret_cast<float4*>(a.partials);
    float2* const pm = reinterpret_cast<float2*>(a.partials + (int64_t)2 * gridDim.x * 2 * D * 128);
    auto part_o = [&](int slot, int c4, int row) { return po + ((int64_t)(slot * 2 + x) * (D / 4) + c4) * 128 + row; };
    auto part_m = [&](int slot, int row) { return pm + (slot * 2 + x) * 128 + row; };
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!ok) break;
      const PgSeg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      if (x == 1 && g.region >= 0) continue;  // a single tile
      const int ntok = min(a.tpt, g.ntok - x * a.tpt), rows = ntok * a.group;
      const int my_tok = r / a.group, tok = g.row0 + x * a.tpt + my_tok;
      const int head = g.head * a.group + r - my_tok * a.group;
      // keys this row sees: up to its own position; none for the MMA rows past the last token
      const int lim = r < rows ? min(g.kv, g.pos0 + x * a.tpt + my_tok + 1) : 0;
      const bool idle = (r & ~31) >= rows;  // no row of this warp is a token's
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < g.nb; ++j, ++cnt) {
        wait(sfull(x), cnt);
        if (!ok) break;
        tc_fence_after();
        if (!idle) {
          uint32_t sv[128];
          tmem_ld64(tS(x) + lane_off, sv);
          tmem_ld64(tS(x) + lane_off + 64, sv + 64);
          const int left = lim - (g.j0 + j) * kPgKeys;
          if (__any_sync(0xffffffffu, left < kPgKeys)) {
#pragma unroll
            for (int e = 0; e < 128; ++e)
              if (e >= left) sv[e] = __float_as_uint(-INFINITY);
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 128; e += 8)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              m4[c] = pg_max3(m4[c], __uint_as_float(sv[e + 2 * c]), __uint_as_float(sv[e + 2 * c + 1]));
          const float m_new = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
          // warp-uniform (tensor-memory loads and stores are warp-collective); O_x holds every block before
          // this one: S_x was issued after their products had completed
          if (__any_sync(0xffffffffu, m_new > m_used + 8.f)) {
            const float m_to = fmaxf(m_used, m_new);
            const float alpha = m_to == -INFINITY ? 1.f : exp2f(m_used - m_to);
            if (j > 0) {
#pragma unroll 1
              for (int c4 = 0; c4 < D / 32; ++c4) {
                uint32_t o[32];
                tmem_ld32(tO(x) + lane_off + 32 * c4, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st32(tO(x) + lane_off + 32 * c4, o);
              }
            }
            l *= alpha;
            m_used = m_to;
          }
          const float nm = m_used == -INFINITY ? 0.f : -m_used;  // a row that has seen no key yet: P = 0
          float ls[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 64; ++c) {  // P pair c = keys 2c, 2c + 1, packed in place over the scores
            const float p0 = pg_ex2(fmaf(__uint_as_float(sv[2 * c]), a.scale_log2, nm));
            const float p1 = pg_ex2(fmaf(__uint_as_float(sv[2 * c + 1]), a.scale_log2, nm));
            ls[(2 * c) & 7] += p0;
            ls[(2 * c + 1) & 7] += p1;
            sv[c] = Elem<T>::pack(p0, p1);
          }
          l += ((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7]));
          tmem_st64(tS(x) + lane_off, sv);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull(x));
      }
      wait(odone(x), cnt - 1);
      if (!ok) break;
      tc_fence_after();
      T* const orow = reinterpret_cast<T*>(a.out) + tok * a.ldo + (int64_t)head * D;
      if (g.whole) {
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        if (!idle) {
#pragma unroll 1
          for (int c4 = 0; c4 < D / 32; ++c4) {
            uint32_t o[32];
            tmem_ld32(tO(x) + lane_off + 32 * c4, o);
            if (r < rows) {
              uint4* d4 = reinterpret_cast<uint4*>(orow + 32 * c4);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = Elem<T>::pack(__uint_as_float(o[8 * c + 2 * e]) * inv, __uint_as_float(o[8 * c + 2 * e + 1]) * inv);
                d4[c] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
          if (r < rows && a.lse)
            a.lse[tok * a.ld_lse + head] = l > 0.f ? (m_used + __log2f(l)) * 0.69314718055994531f : -INFINITY;
        }
      } else if (!idle) {
#pragma unroll 1
        for (int c4 = 0; c4 < D / 32; ++c4) {
          uint32_t o[32];
          tmem_ld32(tO(x) + lane_off + 32 * c4, o);
          if (r < rows)
#pragma unroll
            for (int c = 0; c < 8; ++c)
              __stcg(part_o(g.slot, 8 * c4 + c, r),
                     make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]), __uint_as_float(o[4 * c + 2]),
                                 __uint_as_float(o[4 * c + 3])));
        }
        if (r < rows) __stcg(part_m(g.slot, r), make_float2(m_used, l));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ofree(x));
      if (g.whole) continue;
      // ---- the unit is cut: whoever finishes last joins the pieces, in the order of their keys
      __threadfence();
      meet();
      if (!ok) break;
      if (r == 0) {
        const bool last = atom_add_acq_rel(a.tickets + 2 * g.c0 + x, 1) == g.nc - 1;
        if (last) a.tickets[2 * g.c0 + x] = 0;
        misc[10 + x] = last;
      }
      meet();
      if (!ok) break;
      if (!misc[10 + x]) continue;
      __threadfence();
      auto slot_of = [&](int q) { return 2 * (g.c0 + q) + (q == 0 ? 1 : 0); };
      for (int e = r; e < rows * (D / 4); e += 128) {
        const int row = e % rows, c4 = e / rows;
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q0 = 0; q0 < g.nc; q0 += 8) {
          float2 ml[8];
          float4 v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (q0 + q < g.nc) {
              ml[q] = __ldcg(part_m(slot_of(q0 + q), row));
              v[q] = __ldcg(part_o(slot_of(q0 + q), c4, row));
            }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (q0 + q < g.nc && ml[q].y > 0.f) {  // a piece in which the row saw no key counts for nothing
              const float mn = fmaxf(M, ml[q].x), fa = exp2f(M - mn), fb = exp2f(ml[q].x - mn);
              M = mn;
              L = L * fa + ml[q].y * fb;
              acc.x = acc.x * fa + v[q].x * fb;
              acc.y = acc.y * fa + v[q].y * fb;
              acc.z = acc.z * fa + v[q].z * fb;
              acc.w = acc.w * fa + v[q].w * fb;
            }
        }
        const float inv = L > 0.f ? 1.0f / L : 0.f;
        const int t2 = g.row0 + x * a.tpt + row / a.group, h2 = g.head * a.group + row % a.group;
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + t2 * a.ldo + (int64_t)h2 * D + 4 * c4) =
            make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
        if (c4 == 0 && a.lse)
          a.lse[t2 * a.ld_lse + h2] = L > 0.f ? (M + __log2f(L)) * 0.69314718055994531f : -INFINITY;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
  if (tid == 0) {  // no bulk copy may still be writing shared memory when the CTA exits
    const int n = misc[8];
    for (int it = max(n - kSlots, 0); it < n; ++it)
      if (!mbar_wait(full(it % kSlots), (it / kSlots) & 1, a.b.err, kErrDrain)) break;
    for (int x = 0; x < 2; ++x)
      if (misc[6 + x] > 0) mbar_wait(qfull(x), (misc[6 + x] - 1) & 1, a.b.err, kErrDrain);
  }
}

struct PagedAttnPlan {
  int64_t off_partials, bytes;
};
static PagedAttnPlan paged_attn_plan(int grid, int head_dim) {
  PagedAttnPlan p;
  p.off_partials = ((int64_t)grid * 2 * 4 + 255) / 256 * 256;  // the tickets first
  p.bytes = p.off_partials + (int64_t)2 * grid * 2 * 128 * (head_dim * 4 + 8);
  return p;
}

}  // namespace qd

using namespace qd;

extern "C" int qd_paged_attn_plan(int nq_heads, int nkv_heads, int head_dim, int grid_hint, int* grid,
                                  int64_t* scratch_bytes) {
  if (!grid || !scratch_bytes) return set_error(QD_ERR_ARG, "paged attention plan: null result");
  if (nkv_heads < 1 || nq_heads < nkv_heads || nq_heads % nkv_heads || nq_heads / nkv_heads > 128 ||
      (head_dim != 64 && head_dim != 128))
    return set_error(QD_ERR_UNSUPPORTED, "paged attention: %d query heads over %d KV heads of %d", nq_heads,
                     nkv_heads, head_dim);
  *grid = grid_hint > 0 ? grid_hint : host_sm_count();
  *scratch_bytes = paged_attn_plan(*grid, head_dim).bytes;
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
  const PagedAttnPlan plan = paged_attn_plan(grid < 1 ? 1 : grid, head_dim);
  if (grid < 1 || !scratch || scratch_bytes < plan.bytes || !aligned16(scratch))
    return set_error(QD_ERR_SCRATCH, "paged attention: grid %d needs %lld B of 16-byte aligned scratch (have %lld)", grid,
                     (long long)plan.bytes, (long long)scratch_bytes);
  if (tokens == 0) return QD_OK;
  const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (!encode) return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  a.group = nq_heads / nkv_heads;
  a.tpt = 128 / a.group;
  const CUtensorMapDataType type = dtype == QD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  auto map4 = [&](CUtensorMap* m, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
    return encode(m, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  {  // a tile's rows are token-major, its KV head's query heads inner
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)a.group, (cuuint64_t)nkv_heads, (cuuint64_t)tokens};
    const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)a.group * head_dim * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)a.group, 1, (cuuint32_t)a.tpt}, box1[4] = {64, (cuuint32_t)a.group, 1, 1};
    if (!map4(&a.tq, q, dims, strides, box) || !map4(&a.tq1, q, dims, strides, box1))
      return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for q");
  }
  {
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)page_size, (cuuint64_t)nkv_heads, (cuuint64_t)n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)ps_head * 2, (cuuint64_t)ps_page * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)page_size, 1, 1};
    if (!map4(&a.tk, k_pages, dims, strides, box) || !map4(&a.tv, v_pages, dims, strides, box))
      return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for the pools");
  }
  int g = 2 * a.tpt;  // gcd(2 tpt, 128): the power of two in 2 tpt, up to 128
  g = (g & -g) < kPgKeys ? (g & -g) : kPgKeys;
  a.period = kPgKeys / g;
  a.period_blocks = 2 * a.tpt / g;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.ldo = ldo;
  a.ld_lse = ld_lse;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.tickets = static_cast<int*>(scratch);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(scratch) + plan.off_partials);
  const void* fn = dtype == QD_BF16 ? (head_dim == 128 ? (const void*)paged_attn_kernel<__nv_bfloat16, 128>
                                                       : (const void*)paged_attn_kernel<__nv_bfloat16, 64>)
                                    : (head_dim == 128 ? (const void*)paged_attn_kernel<__half, 128>
                                                       : (const void*)paged_attn_kernel<__half, 64>);
  const int smem = head_dim == 128 ? PgLayout<128>::total : PgLayout<64>::total;
  const int rs = set_max_dynamic_smem(fn, smem);
  if (rs != QD_OK) return rs;
  return launch_kernel(fn, dim3((unsigned)grid), dim3(kPgThreads), smem, pdl, stream, &a);
}
