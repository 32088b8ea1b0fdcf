// Attention of a few query rows of each request over cache pages of 8 bits, on the tcgen05 tensor cores in 8 bits.
//
// A unit is a request's (at most 16) rows of one KV head: single tokens of a group of query heads, or a few tokens. The
// keys and values go to the tensor cores as they lie in the cache, so a key costs D + 1 bytes of memory and of shared
// memory for K and as many for V, and nothing is widened:
//   S^T = K Q^T   tcgen05.mma kind::f8f6f4, M = 128 keys, E4M3 x E4M3
//   O^T += V^T P^T   M = head_dim (V as an MN-major operand), E4M3 x E5M2
// Q and P have more bits than 8, so each goes in as a sum of terms, a column per row and term:
//   Q row = 2^e (t1 + t2 / 16 [+ t3 / 256]), E4M3: 4 bits a term, so two hold a BF16 and three an FP16 exactly, but for
//   elements 2^13 and more below the row's largest, which are off by 2^-22 of that;
//   P = t1 + t2 / 8 + t3 / 64 [+ t4 / 512], E5M2: 3 bits a term, 2^-9 of P in three (BF16) and 2^-12 in four (FP16), what
//   the 16-bit attention's rounding of P gives. E5M2 for its range: a thousand keys that each weigh 2^-20 of the largest
//   must not vanish, which E4M3's range would make them do.
// The products are exact, their sums fp32. A product of 128 x 16 x 32 takes the tensor core as long as one of
// 128 x 64 x 32, so the terms are free.
//
// A row's power of two is its thread's: thread r has key r of the block, so its score is S^T * 2^e_k, and 2^e_v is added
// to the exponent of the weight, P' = exp2(s log2 e + e_v - m), whose running maximum m is that of the weights of the
// codes. l sums P' / 2^e_v.
//
// The key blocks of all units form one line that is cut evenly over the CTAs, two to an SM: a warpgroup that turns scores
// into weights each, so that one CTA's start, unit ends and last block hide behind the other's stream of blocks. The
// scores of the next two blocks are always under way, across the units too. Pieces of a cut unit are left in the scratch
// and joined in the order of their keys by the CTA that ends last.
//
// Measured, 32 query and 8 KV heads of 128 in BF16: 8 single tokens over up to 41 k keys 94 to 98 us (6.0 to 6.2 TB/s,
// 0.92 to 0.95 of a copy's rate); 64 over 1 to 1.5 k keys 40 us (4.3 TB/s: start 4 us, unit ends and the pieces' joins 2 us
// each); one over 1 k keys 11.0 us in a graph. A block of 128 keys takes a CTA 0.8 us when its data is there, of which S, the
// maxima, P and the barriers between are a quarter each; two CTAs need one every 1.5 us.
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>

#include "qd_host.h"
#include "qd_paged_attn8.h"
#include "qd_paged_attn_dev.cuh"

namespace qd {

constexpr int kF8Threads = 256;  // warps 0-3 softmax, 4 producer, 5 MMA, 6 the line and the queries, 7 the scales
constexpr int kF8Scales = 8;     // blocks whose scales are in shared memory
constexpr int kF8Unit = 2;       // blocks' time that a unit's start and end take
constexpr int kF8Bias = 7;       // P' is up to 2^(8 + 7): the upper end of E5M2's range

template <typename T, int D>
struct F8Lay {
  static constexpr int kTQ = Elem<T>::kBf16 ? 2 : 3, kTP = Elem<T>::kBf16 ? 3 : 4;  // terms
  static constexpr int kItem = kPgKeys * D;         // a K or V block
  static constexpr int kQ = kFewRows * kTQ * D;     // a unit's queries
  static constexpr int kP = kFewRows * kTP * kPgKeys;
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int q = 0;                       // two units'
  static constexpr int p = q + 2 * kQ;              // two blocks'
  static constexpr int kv = p + 2 * kP;
  static constexpr int sc = kv + kSlots * kItem;    // [block][K, V][128 keys]
  static constexpr int bars = sc + kF8Scales * 2 * kPgKeys;
  // q8full[2], qempty[2], sfull[2], pfull[2], odone[2], group, segfull[4], segempty[4], then scfull[], scempty[], full[], empty[]
  static constexpr int nbars = 19 + 2 * kF8Scales + 2 * kSlots;
  static constexpr int seg = bars + (nbars * 8 + 63) / 64 * 64;
  static constexpr int qs = seg + 4 * 64;     // the queries' powers of two [2 units][16]
  static constexpr int misc = qs + 128;       // tmem, abort, line start, drain count, last flag; then the scan's totals
  static constexpr int sums = misc + 256;     // the warps' sums [16 rows][4 warps]
  static constexpr int mx = sums + 256;       // and maxima, of two blocks
  static constexpr int total = mx + 512;
  static_assert(kQ % 1024 == 0 && kP % 1024 == 0 && kItem % 1024 == 0, "operands start on 1 KiB");
  static_assert(kF8Resident * (total + 1024) <= 228 * 1024, "shared memory of an SM");
};

struct alignas(64) Few8Args {
  CUtensorMap tk, tv;
  PagedBatch b;
  const char* q;
  const uint8_t *k_scale, *v_scale;
  char* out;
  float* lse;
  int64_t ldq, ldo, ld_lse, ss_page, ss_head;
  PgShape s;
  int room;       // positions in a row of the page table, kPgMaxKeys at most
  int inv_group;  // row / group = row * inv_group >> 16
  int alone;      // no other kernel takes the requests of more tokens
  int beside;     // the kernel before is the one for those: nothing of it is waited for but its end
  float scale_log2;
  float* partials;  // [2 * grid slots][16 rows][D], then the rows' (m, l)
  int* tickets;     // [grid]
};

struct F8Seg {
  int row0, ntok, pos0, kv;  // first token row, tokens, the first's position, keys of the request
  int head, j0, nb, whole;   // KV head, first key block, blocks (0 ends the list), all of the unit's
  int slot, c0, nc;          // partial slot, first CTA and number of CTAs of the unit
  int request;
};
static_assert(sizeof(F8Seg) <= 64, "segment ring entry");

// 8-bit operands whose rows are D bytes, swizzled over 128 or 64 bytes
template <int D>
constexpr uint32_t f8_desc_hi() {
  return (8u * D >> 4) | (1u << 14) | ((D == 128 ? 2u : 4u) << 29);
}
template <uint32_t kHiA, uint32_t kHiB>
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %6};\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kHiA), "n"(kHiB)
      : "memory");
}
// E4M3 x E4M3 (or E5M2: b_e5m2) -> F32, M = 128, N = n; B K-major, A too unless a_mn
constexpr uint32_t f8_idesc(int n, bool a_mn, bool b_e5m2) {
  return (1u << 4) | ((b_e5m2 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// 16 columns of this thread's lane of tensor memory, waited for
__device__ __forceinline__ void f8_load(uint32_t taddr, uint32_t* r) {
  tmem_ld16_raw(taddr, r);
  tmem_wait_ld16(r);
}
constexpr int f8_cols(int n) { return (n + 15) / 16 * 16; }
// The sums of kC rows' terms, each `step` of the one before it: column c + t kC is row c's term t.
template <int kC, int kTerms>
__device__ __forceinline__ void f8_terms(uint32_t taddr, float step, float* v) {
  if constexpr (kC < 16) {  // all in one load
    uint32_t u[16];
    f8_load(taddr, u);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      v[c] = __uint_as_float(u[c + (kTerms - 1) * kC]);
#pragma unroll
      for (int t = kTerms - 2; t >= 0; --t) v[c] = fmaf(v[c], step, __uint_as_float(u[c + t * kC]));
    }
  } else {
#pragma unroll
    for (int t = kTerms - 1; t >= 0; --t) {
      uint32_t u[16];
      f8_load(taddr + t * kC, u);
#pragma unroll
      for (int c = 0; c < kC; ++c) v[c] = t == kTerms - 1 ? __uint_as_float(u[c]) : fmaf(v[c], step, __uint_as_float(u[c]));
    }
  }
}

// whether the phase with `parity` has completed, without waiting
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// one request's blocks in this kernel (0: not its)
__device__ __forceinline__ int f8_blocks(const PgShape& s, const PgReq& r) {
  return r.n > 0 && r.n <= s.tpf ? pg_max((pg_min(r.kv, r.pos0 + r.n) + kPgKeys - 1) / kPgKeys, 1) : 0;
}

// and places on the line for each KV head: the unit's own, then a block each
__device__ __forceinline__ int f8_places(int blocks) { return blocks ? blocks + kF8Unit : 0; }

// Joins a cut unit's pieces in the order of their keys: a row per D / 4 lanes of four warps, eight pieces in flight.
template <typename T, int D>
__device__ __forceinline__ void f8_join(const Few8Args& a, const F8Seg& g, int r, int rows) {
  constexpr int kLanes = D / 4, kAt = 128 / kLanes, kAhead = 8;
  const int c4 = r % kLanes;
  const float2* const pm = reinterpret_cast<const float2*>(a.partials + (int64_t)2 * gridDim.x * kFewRows * D);
#pragma unroll 1
  for (int row = r / kLanes; row < rows; row += kAt) {
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int q0 = 0; q0 < g.nc; q0 += kAhead) {
      float2 ml[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int qq = min(q0 + q, g.nc - 1);  // past the last piece: the last again, not counted
        const int64_t at = (int64_t)(2 * (g.c0 + qq) + (qq == 0 ? 1 : 0)) * kFewRows + row;
        ml[q] = __ldcg(pm + at);
        v[q] = __ldcg(reinterpret_cast<const float4*>(a.partials + at * D) + c4);
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        if (q0 + q < g.nc && ml[q].y != 0.f) {  // a piece in which the row saw no key counts for nothing
          const float mn = fmaxf(M, ml[q].x), fa = exp2f(M - mn), fb = exp2f(ml[q].x - mn);
          M = mn;
          L = L * fa + ml[q].y * fb;
          acc.x = acc.x * fa + v[q].x * fb;
          acc.y = acc.y * fa + v[q].y * fb;
          acc.z = acc.z * fa + v[q].z * fb;
          acc.w = acc.w * fa + v[q].w * fb;
        }
    }
    const float inv = pg_inverse(L);
    const int tok = (row * a.inv_group) >> 16, hq = g.head * a.s.group + row - tok * a.s.group;
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (g.row0 + tok) * a.ldo + (int64_t)hq * D + 4 * c4) =
        make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
    if (c4 == 0 && a.lse) a.lse[(g.row0 + tok) * a.ld_lse + hq] = pg_lse(M - kF8Bias, L);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kF8Threads, kF8Resident) paged_few8_kernel(const __grid_constant__ Few8Args a) {
  using Lay = F8Lay<T, D>;
  constexpr int kSlots = Lay::kSlots, kTQ = Lay::kTQ, kTP = Lay::kTP;
  extern __shared__ __align__(1024) char smem[];
  const uint32_t sb = smem_u32(smem), bars = sb + Lay::bars;
  auto q8full = [&](int s) { return bars + 8u * (s & 1); };
  auto qempty = [&](int s) { return bars + 16 + 8u * (s & 1); };
  auto sfull = [&](int x) { return bars + 32 + 8u * x; };
  // A barrier for each of two blocks: the softmax may be done with two before the first product, and two products may be
  // under way at a unit's end. A parity wait two phases behind a barrier never ends, and two ahead of it does not wait.
  auto pfull = [&](int x) { return bars + 48 + 8u * x; };
  auto odone = [&](int x) { return bars + 64 + 8u * x; };
  const uint32_t group = bars + 80;
  auto segfull = [&](int s) { return bars + 88 + 8u * (s & 3); };
  auto segempty = [&](int s) { return bars + 120 + 8u * (s & 3); };
  auto scfull = [&](int b) { return bars + 152 + 8u * (b & (kF8Scales - 1)); };
  auto scempty = [&](int b) { return bars + 152 + 8u * (kF8Scales + (b & (kF8Scales - 1))); };
  auto full = [&](int s) { return bars + 152 + 8u * (2 * kF8Scales + s); };
  auto empty = [&](int s) { return bars + 152 + 8u * (2 * kF8Scales + kSlots + s); };
  F8Seg* segs = reinterpret_cast<F8Seg*>(smem + Lay::seg);
  int* misc = reinterpret_cast<int*>(smem + Lay::misc);
  int* abort = misc + 1;
  int64_t* scan = reinterpret_cast<int64_t*>(misc + 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (sb & 1023u) {  // the swizzled operands need 1 KiB alignment, and there is no room to realign
    grid_dep_wait();
    if (tid == 0 && blockIdx.x == 0) flag_error(a.b.err, kErrSmem);
    return;
  }
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(q8full(x), 1);
      mbar_init(qempty(x), 5);  // the MMA's products and four softmax warps
      mbar_init(sfull(x), 1);
      mbar_init(pfull(x), 4);
      mbar_init(odone(x), 1);
    }
    mbar_init(group, 4);
    for (int k = 0; k < 4; ++k) {
      mbar_init(segfull(k), 1);
      mbar_init(segempty(k), 7);  // all warps but the one that walks the line
    }
    for (int k = 0; k < kF8Scales; ++k) {
      mbar_init(scfull(k), 1);
      mbar_init(scempty(k), 4);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_mbar_init();
    for (int m = 1; m < 16; ++m) misc[m] = 0;
  }
  if (warp == 5) tmem_alloc(smem_u32(misc), 256);
  // Beside the tiles' kernel nothing is waited for here: its CTAs had all waited for what came before both when they let
  // this one start, so those writes are in L2. What lies in an SM's L1 may be older (the queries of the call before, in
  // the same buffer), so all that is read ahead of the wait at the end bypasses L1: ld.cg, and copies, which do.
  if (!a.beside) grid_dep_wait();
  {  // the page table on its way to L2 while the lengths are read: a line per thread of the grid
    const int lines = (a.b.max_pages + 31) / 32;
    const int64_t at = (int64_t)blockIdx.x * kF8Threads + tid, row = at / lines;
    if (row < a.b.batch) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.b.table + row * a.b.ld_table + (at - row * lines) * 32));
  }

  // ---- this CTA's place on the line: a prefix sum over the requests, and a walk from the one it starts in
  const int per = (a.b.batch + kF8Threads - 1) / kF8Threads;
  const int i0 = min(tid * per, a.b.batch), i1 = min(i0 + per, a.b.batch);
  auto request = [&](int i) {
    return pg_make_request(a.s, ld_i32(a.b.cu + i), ld_i32(a.b.cu + i + 1), ld_i32(a.b.kv_len + i), (int)a.b.tokens, a.room);
  };
  PgReq r = {};
  int64_t mine = 0;
  int flags = 0;
  for (int i = i0; i < i1; ++i) {
    r = request(i);
    const int nb = f8_blocks(a.s, r);
    mine += (int64_t)a.b.nkv * f8_places(nb);
    if (nb && r.kv != r.pos0 + r.n) flags |= QD_DEVERR_PAGE;
    if (a.alone && r.n > a.s.tpf) flags |= QD_DEVERR_POS;
  }
  if (flags && blockIdx.x == 0) flag_error(a.b.err, flags);
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
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kF8Threads / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const PgLine line = pg_line(total, (int)gridDim.x, 1);
  const int cta = blockIdx.x;
  const int64_t begin = cta < line.ctas ? line.begin(cta) : 0, end = cta < line.ctas ? line.begin(cta + 1) : 0;
  if (begin < end && begin >= before && begin < before + mine) {
    int64_t w = begin - before;
    int i = i0;
    if (per > 1) {
      for (r = request(i);; r = request(++i)) {
        const int64_t c = (int64_t)a.b.nkv * f8_places(f8_blocks(a.s, r));
        if (w < c) break;
        w -= c;
      }
    }
    const int nb = f8_places(f8_blocks(a.s, r));
    misc[2] = i;
    misc[3] = (int)(w / nb);
    misc[4] = (int)(w % nb);
    *reinterpret_cast<PgReq*>(smem + Lay::mx) = r;
  }
  __syncthreads();
  const uint32_t tmem = (uint32_t)misc[0];
  auto tS = [&](int x) { return tmem + 64u * x; };
  const uint32_t tO = tmem + 128u;

  if (warp == 4) {
    // ------------------------------------------------------------ producer: a lane per page of a block
    const uint64_t pol = policy_evict_normal();
    const int boxes = kPgKeys >> a.b.page_shift, box_bytes = a.b.page_size * D;
    const int per_lot = 32 / boxes;  // blocks
    int items = 0, slot = 0, of_request = -1, first_lot = -2;
    uint32_t phase = 1;  // of empty(slot): a ring's first round passes at once
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity, int code) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, code, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
#pragma unroll 1
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2, kErrWaitFull);
      if (!ok) break;
      const F8Seg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      // The request's page entries, 32 at a time (aligned, so that a block's lie in one lot), a lot ahead: a block's
      // copies take less time than a load of their entries. The first lot stays for the request's other heads.
      auto lot = [&](int n) {
        const int entry = 32 * n + lane;
        return (int64_t)entry << a.b.page_shift < g.kv ? ld_i32(a.b.table + g.request * a.b.ld_table + entry) : -2;
      };
      if (g.request != of_request) first_lot = lot(0);
      of_request = g.request;
      int n_lot = g.j0 / per_lot, entries = n_lot ? lot(n_lot) : first_lot, ahead = lot(n_lot + 1);
      for (int j = g.j0; j < g.j0 + g.nb && ok; ++j) {
        if (j / per_lot != n_lot) {
          entries = ahead;
          ahead = lot(++n_lot + 1);
        }
        int page = __shfl_sync(0xffffffffu, entries, (j % per_lot) * boxes + (lane & (boxes - 1)));
        const bool need = lane < boxes && ((int64_t)j * kPgKeys + (lane << a.b.page_shift)) < g.kv;
        if (need && (page < 0 || page >= a.b.n_pages)) {
          flag_error(a.b.err, QD_DEVERR_PAGE);
          page = -1;  // outside the tensor map: the copy fills zeros
        }
        const int n_need = __popc(__ballot_sync(0xffffffffu, need));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          wait(empty(slot), phase, kErrWaitEmpty);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(full(slot), n_need * box_bytes);
            misc[8] = ++items;
          }
          __syncwarp();
          if (need)
            pg_tma_4d(sb + Lay::kv + slot * Lay::kItem + lane * box_bytes, kv ? &a.tv : &a.tk, 0, 0, g.head, page, full(slot), pol);
          if (++slot == kSlots) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) break;
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ MMA: one elected lane, whatever is ready first
    constexpr uint32_t hi = f8_desc_hi<D>(), hi_p = f8_desc_hi<128>(), kItem16 = Lay::kItem >> 4;
    if (elect_one()) {
      const uint32_t d_q = umma_desc_lo(sb + Lay::q), d_k = umma_desc_lo(sb + Lay::kv), d_p = umma_desc_lo(sb + Lay::p);
      // heads of 64: the 64 upper rows of O^T repeat the lower ones (block stride 0)
      const uint32_t d_v = umma_desc_lo(sb + Lay::kv, 0);
      struct Side {  // of the next scores, and of the next product with V: segment, blocks left of it, block, its slot
        int seg, left, blk, slot;
        uint32_t phase, id;
      };
      Side s = {0, 0, 0, 0, 0, 0}, v = {0, 0, 0, 1, 0, 0};
      auto step = [&](Side& x) {
        ++x.blk;
        x.slot += 2;
        if (x.slot >= kSlots) {
          x.slot -= kSlots;
          x.phase ^= 1;
        }
      };
      bool s_end = false, first = false, ok = true;
      uint64_t t0 = globaltimer();
      for (uint32_t idle = 0; ok; ++idle) {
        if (v.left == 0 && (v.blk < s.blk || s_end)) {  // (its segment is known: the scores are ahead)
          const F8Seg& g = segs[v.seg & 3];
          v.left = g.nb;
          if (v.left == 0) break;
          v.id = g.ntok * a.s.group <= 4 ? f8_idesc(f8_cols(4 * kTP), true, true) : f8_idesc(kFewRows * kTP, true, true);
          first = true;
        }
        if (v.blk < s.blk && mbar_test(pfull(v.blk & 1), (v.blk >> 1) & 1) && mbar_test(full(v.slot), v.phase)) {
          tc_fence_after();
          const uint32_t vt = d_v + v.slot * kItem16, pt = d_p + (v.blk & 1) * (Lay::kP >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 keys per MMA: four groups of 8 rows of V
            umma_f8<hi, hi_p>(tO, vt + k * (32 * D >> 4), pt + 2 * k, v.id, k || !first ? 1u : 0u);
          first = false;
          umma_commit(odone(v.blk & 1));
          umma_commit(empty(v.slot));
          step(v);
          if (--v.left == 0) mbar_arrive(segempty(v.seg++));
          idle = 0;
        }
        if (s.left == 0 && !s_end && mbar_test(segfull(s.seg), (s.seg >> 2) & 1)) {
          const F8Seg& g = segs[s.seg & 3];
          s.left = g.nb;
          s_end = s.left == 0;
          s.id = g.ntok * a.s.group <= 4 ? f8_idesc(f8_cols(4 * kTQ), false, false) : f8_idesc(kFewRows * kTQ, false, false);
        }
        if (s.left > 0 && s.blk < v.blk + 2 && mbar_test(q8full(s.seg), (s.seg >> 1) & 1) && mbar_test(full(s.slot), s.phase)) {
          tc_fence_after();
          const uint32_t qt = d_q + (s.seg & 1) * (Lay::kQ >> 4), kt = d_k + s.slot * kItem16;
#pragma unroll
          for (int d = 0; d < D / 32; ++d) umma_f8<hi, hi>(tS(s.blk & 1), kt + 2 * d, qt + 2 * d, s.id, d > 0 ? 1u : 0u);
          umma_commit(sfull(s.blk & 1));
          umma_commit(empty(s.slot));
          step(s);
          if (--s.left == 0) umma_commit(qempty(s.seg++));
          idle = 0;
        }
        if (idle == 0) t0 = globaltimer();
        if ((idle & 63u) == 63u) {  // bounded, as every wait
          if (*reinterpret_cast<volatile int*>(abort)) ok = false;
          if (globaltimer() - t0 > kWaitLimitNs) {
            if (a.b.err) atomicOr(a.b.err, kErrWaitFull);
            atomicExch(abort, 1);
            ok = false;
          }
        }
      }
      // no MMA may still run when its memory is given back
      if (s.blk > 0) mbar_wait(sfull((s.blk - 1) & 1), ((s.blk - 1) >> 1) & 1, a.b.err, kErrDrain);
      if (v.blk > 0) mbar_wait(odone((v.blk - 1) & 1), ((v.blk - 1) >> 1) & 1, a.b.err, kErrDrain);
    }
    __syncwarp();
  } else if (warp == 7) {
    // ------------------------------------------------------------ the rows' powers of two, four keys a lane
    constexpr int kAhead = 4;  // blocks whose loads are in flight (entries, then scales: two waits for memory)
    bool ok = true;
    int blk = 0;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
#pragma unroll 1
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!ok) break;
      const F8Seg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      const int32_t* const table = a.b.table + g.request * a.b.ld_table;
#pragma unroll 1
      for (int j0 = 0; j0 < g.nb && ok; j0 += kAhead) {
        int page[kAhead];
        uint32_t ks[kAhead], vs[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int key = (g.j0 + j0 + j) * kPgKeys + 4 * lane;
          page[j] = j0 + j < g.nb && key < g.kv ? ld_i32(table + (key >> a.b.page_shift)) : -1;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {  // keys of no page: 1
          const int64_t at = page[j] * a.ss_page + g.head * a.ss_head + (((g.j0 + j0 + j) * kPgKeys + 4 * lane) & (a.b.page_size - 1));
          const bool in = page[j] >= 0 && page[j] < a.b.n_pages;
          ks[j] = in ? __ldcg(reinterpret_cast<const uint32_t*>(a.k_scale + at)) : 0x7f7f7f7fu;
          vs[j] = in ? __ldcg(reinterpret_cast<const uint32_t*>(a.v_scale + at)) : 0x7f7f7f7fu;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (j0 + j >= g.nb) break;
          wait(scempty(blk), (blk / kF8Scales) + 1);  // (a ring's first round passes at once)
          if (!ok) break;
          uint32_t* const to = reinterpret_cast<uint32_t*>(smem + Lay::sc + (blk & (kF8Scales - 1)) * 2 * kPgKeys);
          to[lane] = ks[j];
          to[lane + 32] = vs[j];
          __syncwarp();
          if (lane == 0) mbar_arrive(scfull(blk));
          ++blk;
        }
      }
      if (!ok) break;
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------ walks the line, and makes the queries' terms
    constexpr int kLanes = D / 8, kAt = 32 / kLanes, kAhead = 2;  // lanes of a row, rows at a time, loads in flight
    const int sub = lane % kLanes;
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity, int code) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, code, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    int64_t at = begin;
    int i = misc[2], h = misc[3], o = misc[4];
    r = *reinterpret_cast<const PgReq*>(smem + Lay::mx);
    __syncwarp();
    // Names the next piece of the line, or its end (0 blocks). The others then know of it while the one before is under
    // way, and have its page entries, scales and queries at hand when they come to it.
    auto publish = [&](int seg) {
      if (seg >= 4) wait(segempty(seg), (seg >> 2) - 1, kErrWaitEmpty);
      if (!ok) return;
      F8Seg g = {};
      while (at < end && g.nb == 0) {  // (a CTA whose share ends in a unit's own places has no block of it)
        const int nblk = f8_blocks(a.s, r), take = (int)min(end - at, (int64_t)(f8_places(nblk) - o));
        const int64_t first = at - o + kF8Unit;  // place of the unit's first block
        g.row0 = r.row0;
        g.ntok = r.n;
        g.pos0 = r.pos0;
        g.kv = r.kv;
        g.head = h;
        g.j0 = max(o - kF8Unit, 0);
        g.nb = max(o + take - kF8Unit, 0) - g.j0;
        g.whole = g.nb == nblk;
        g.slot = 2 * cta + (g.j0 > 0 ? 0 : 1);
        g.c0 = line.owner(first);
        g.nc = line.owner(first + nblk - 1) - g.c0 + 1;
        g.request = i;
        at += take;
        o = 0;
        if (at < end && ++h == a.b.nkv) {
          h = 0;
          do r = request(++i);
          while (f8_blocks(a.s, r) == 0);
        }
      }
      if (lane == 0) {
        segs[seg & 3] = g;
        mbar_arrive(segfull(seg));
      }
      __syncwarp();
    };
    publish(0);
#pragma unroll 1
    for (int seg = 0; ok; ++seg) {
      const F8Seg g = segs[seg & 3];
      if (g.nb == 0) break;
      publish(seg + 1);
      if (seg >= 2) wait(qempty(seg), (seg >> 1) - 1, kErrWaitEmpty);
      if (!ok) break;
      const int rows = g.ntok * a.s.group, step = rows <= 4 ? 4 : kFewRows;
      char* const to = smem + Lay::q + (seg & 1) * Lay::kQ;
#pragma unroll 1
      for (int c0 = 0; c0 < rows; c0 += kAhead * kAt) {
        uint4 u[kAhead];
#pragma unroll
        for (int y = 0; y < kAhead; ++y) {
          const int c = min(c0 + y * kAt + lane / kLanes, rows - 1);  // (past the last row: that one again)
          const int tok = (c * a.inv_group) >> 16, hq = g.head * a.s.group + c - tok * a.s.group;
          u[y] = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (g.row0 + tok) * a.ldq + (int64_t)hq * D + 8 * sub));
        }
#pragma unroll
        for (int y = 0; y < kAhead; ++y) {
          const int c = min(c0 + y * kAt + lane / kLanes, rows - 1);
          float x[8], most = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = Elem<T>::unpack((&u[y].x)[k]);
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[k]) <= FLT_MAX ? fabsf(x[k]) : 0.f);
#pragma unroll
          for (int n = kLanes / 2; n > 0; n >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, n));
          // the row's largest comes to (224, 448] (or less, where it is below 2^-100); what is not finite is NaN
          const int e = max((int)(__float_as_uint(most) >> 23) - 127 - 8 + ((__float_as_uint(most) & 0x7fffffu) > 0x600000u ? 1 : 0), -110);
          const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = fabsf(x[k]) <= FLT_MAX ? x[k] * inv : __uint_as_float(0x7fffffffu);
#pragma unroll
          for (int t = 0; t < kTQ; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * k], x[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
              const __half2_raw f2 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w[k], __NV_E4M3);
              const float2 f = __half22float2(__half2(f2));
              x[2 * k] = (x[2 * k] - f.x) * 16.f;
              x[2 * k + 1] = (x[2 * k + 1] - f.y) * 16.f;
            }
            const int n = t * step + c, sw = D == 128 ? n & 7 : (n >> 1) & 3;
            *reinterpret_cast<uint2*>(to + n * D + (((sub >> 1) ^ sw) << 4) + (sub & 1) * 8) =
                make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
          }
          if (sub == 0) reinterpret_cast<float*>(smem + Lay::qs)[(seg & 1) * kFewRows + c] = __uint_as_float((uint32_t)(127 + e) << 23);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q8full(seg));
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue
    const int r = tid, wg = warp;  // r: the key, or the dim of O^T
    const uint32_t lane_off = (uint32_t)(32 * wg) << 16;
    int b = 0, meets = 0;  // blocks of all units so far
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto meet = [&]() {  // the four warps; bounded, unlike a named barrier
      __syncwarp();
      if (lane == 0) mbar_arrive(group);
      wait(group, meets++);
    };
    float2* const pm = reinterpret_cast<float2*>(a.partials + (int64_t)2 * gridDim.x * kFewRows * D);
    float4* const sums = reinterpret_cast<float4*>(smem + Lay::sums);
    auto unit = [&](auto cols, const F8Seg& g, int seg) __attribute__((always_inline)) {
      constexpr int kC = decltype(cols)::value;
      const int rows = g.ntok * a.s.group;
      wait(q8full(seg), seg >> 1);
      if (!ok) return;
      const float sc = lane < rows ? reinterpret_cast<const float*>(smem + Lay::qs)[(seg & 1) * kFewRows + lane] * a.scale_log2 : 0.f;
      __syncwarp();
      if (lane == 0) mbar_arrive(qempty(seg));
      float m = -INFINITY;  // of row `lane`, the same in all four warps
      float l[kC];          // of every row, this thread's keys
#pragma unroll
      for (int c = 0; c < kC; ++c) l[c] = 0.f;
#pragma unroll 1
      for (int j = 0; j < g.nb; ++j, ++b) {
        wait(scfull(b), b / kF8Scales);
        if (!ok) return;
        const uint8_t* const two = reinterpret_cast<const uint8_t*>(smem) + Lay::sc + (b & (kF8Scales - 1)) * 2 * kPgKeys;
        const float ks = __uint_as_float((uint32_t)two[r] << 23), ev = (float)two[kPgKeys + r] - 127.f;
        __syncwarp();
        if (lane == 0) mbar_arrive(scempty(b));
        wait(sfull(b & 1), b >> 1);
        if (!ok) return;
        tc_fence_after();
        float t[kC];  // the weights' exponents, in twos
        {
          f8_terms<kC, kTQ>(tS(b & 1) + lane_off, 0.0625f, t);
#pragma unroll
          for (int c = 0; c < kC; ++c) t[c] = fmaf(t[c] * ks, __shfl_sync(0xffffffffu, sc, c), ev);
        }
        const int key0 = (g.j0 + j) * kPgKeys;
        if (key0 + kPgKeys > min(g.kv, g.pos0 + 1)) {  // some row sees only a part of this block
          const int key = key0 + r;
          int lim = g.pos0 + 1, next = a.s.group;  // of the row's token
#pragma unroll
          for (int c = 0; c < kC; ++c) {
            if (c == next) {
              ++lim;
              next += a.s.group;
            }
            if (key >= min(lim, g.kv)) t[c] = -INFINITY;
          }
          if (key0 + kPgKeys > g.kv) {  // V rows past the last key hold anything: zeroed, since 0 x NaN is NaN
            const int item = 2 * b + 1, slot = item % kSlots;
            wait(full(slot), item / kSlots);
            if (!ok) return;
            if (key >= g.kv) {
              char* const row = smem + Lay::kv + slot * Lay::kItem + r * D;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) *reinterpret_cast<uint4*>(row + ((i ^ (r & (D / 16 - 1))) << 4)) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float v = redux_max(t[c]);
          top = lane == c ? v : top;
        }
        // (a warp may write the next block's before the others have read this one's)
        float4* const mx = reinterpret_cast<float4*>(smem + Lay::mx) + (b & 1) * kFewRows;
        if (lane < rows) reinterpret_cast<float*>(mx + lane)[wg] = top;
        meet();
        if (!ok) return;
        float mn = -INFINITY;
        if (lane < rows) {
          const float4 v = mx[lane];
          mn = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        }
        if (__any_sync(0xffffffffu, mn > m + 8.f)) {  // the same in every warp
          const float m_to = fmaxf(m, mn), alpha = m_to == -INFINITY ? 1.f : exp2f(m - m_to);
          m = m_to;
          if (j > 0) {
            wait(odone((b - 1) & 1), (b - 1) >> 1);  // the sums with every block before this one
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kC; ++c) l[c] *= __shfl_sync(0xffffffffu, alpha, c);
#pragma unroll 1
            for (int i = 0; i < f8_cols(kC * kTP); i += 16) {
              uint32_t o[16];
              f8_load(tO + lane_off + i, o);
#pragma unroll
              for (int c = 0; c < 16; ++c)
                o[c] = __float_as_uint(__uint_as_float(o[c]) * __shfl_sync(0xffffffffu, alpha, c & (kC - 1)));
              tmem_st16(tO + lane_off + i, o);
            }
          }
        }
        const float nm = m == -INFINITY ? (float)kF8Bias : kF8Bias - m, per_code = exp2f(-ev);
        char* const p_to = smem + Lay::p + (b & 1) * Lay::kP + (r & 15);  // (the product of two blocks ago has been done)
#pragma unroll
        for (int c = 0; c < kC; c += 2) {
          float2 p;
          p.x = pg_ex2(t[c] + __shfl_sync(0xffffffffu, nm, c));
          p.y = pg_ex2(t[c + 1] + __shfl_sync(0xffffffffu, nm, c + 1));
          l[c] = fmaf(p.x, per_code, l[c]);
          l[c + 1] = fmaf(p.y, per_code, l[c + 1]);
#pragma unroll
          for (int q = 0; q < kTP; ++q) {
            const uint32_t w = __nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, __NV_E5M2);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const int n = c + d + q * kC;
              p_to[n * kPgKeys + (((r >> 4) ^ (n & 7)) << 4)] = (char)(w >> (8 * d));
            }
            const uint32_t h = __byte_perm(w, 0, 0x1404);  // an E5M2 is the upper half of an FP16
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            p.x = (p.x - f.x) * 8.f;
            p.y = (p.y - f.y) * 8.f;
          }
        }
        tc_fence_before();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull(b & 1));
      }
      {  // the warps' sums of every row, side by side
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int c = 0; c < kC; ++c) l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
        float mine = 0.f;
#pragma unroll
        for (int c = 0; c < kC; ++c) mine = lane == c ? l[c] : mine;
        if (lane < rows) reinterpret_cast<float*>(sums + lane)[wg] = mine;
      }
      meet();
      wait(odone((b - 1) & 1), (b - 1) >> 1);
      if (!ok) return;
      tc_fence_after();
      float ov[kC];
      f8_terms<kC, kTP>(tO + lane_off, 0.125f, ov);
      tc_fence_before();
      float inv = 1.f;
      int64_t row_at = 0;  // of row `lane`, in elements
      if (lane < rows) {
        const float4 s = sums[lane];
        const float L = (s.x + s.y) + (s.z + s.w);
        const int tok = (lane * a.inv_group) >> 16, hq = g.head * a.s.group + lane - tok * a.s.group;
        row_at = (g.row0 + tok) * a.ldo + (int64_t)hq * D;
        if (g.whole) {
          inv = pg_inverse(L);
          if (wg == 0 && a.lse) a.lse[(g.row0 + tok) * a.ld_lse + hq] = pg_lse(m - kF8Bias, L);
        } else if (wg == 0) {
          __stcg(pm + (int64_t)g.slot * kFewRows + lane, make_float2(m, L));
        }
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const float v = ov[c] * __shfl_sync(0xffffffffu, inv, c);
        const int64_t to = __shfl_sync(0xffffffffu, row_at, c);
        if (c < rows && r < D) {
          if (g.whole)
            reinterpret_cast<uint16_t*>(a.out)[to + r] = (uint16_t)Elem<T>::pack(v, 0.f);
          else
            __stcg(a.partials + ((int64_t)g.slot * kFewRows + c) * D + r, v);
        }
      }
      if (g.whole) return;
      // a cut unit: whoever finishes last joins the pieces. Their stores are made visible by the barrier and the
      // ticket (release is cumulative)
      meet();
      if (!ok) return;
      if (r == 0) {
        const bool last = atom_add_acq_rel(a.tickets + g.c0, 1) == g.nc - 1;
        if (last) a.tickets[g.c0] = 0;
        misc[10] = last;
      }
      meet();
      if (ok && misc[10]) f8_join<T, D>(a, g, r, rows);
    };
#pragma unroll 1
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!ok) break;
      const F8Seg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      if (g.ntok * a.s.group <= 4)
        unit(Const<4>(), g, seg);
      else
        unit(Const<kFewRows>(), g, seg);
      if (!ok) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (a.beside) grid_dep_wait();  // whoever waits for this kernel waits for both
  if (warp == 5) tmem_dealloc(tmem, 256);
  if (tid == 0) {  // no copy may still be writing shared memory when the CTA exits
    const int n = misc[8];
    for (int it = max(n - kSlots, 0); it < n; ++it)
      if (!mbar_wait(full(it % kSlots), (it / kSlots) & 1, a.b.err, kErrDrain)) break;
  }
}

int map_pools8(const Paged8Call& c, PFN_cuTensorMapEncodeTiled_v12000 encode, int row, CUtensorMap* tk, CUtensorMap* tv) {
  const int D = c.head_dim;
  const PagedBatch& b = c.b;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)b.page_size, (cuuint64_t)b.nkv, (cuuint64_t)b.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)D, (cuuint64_t)b.ps_head, (cuuint64_t)b.ps_page};
  const cuuint32_t box[4] = {(cuuint32_t)row, (cuuint32_t)b.page_size, 1, 1}, one[4] = {1, 1, 1, 1};
  for (int v = 0; v < 2; ++v)
    if (encode(v ? tv : tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(v ? c.v_pages : c.k_pages), dims, strides,
               box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for the pools");
  return QD_OK;
}

int launch_few8(const Paged8Call& c, bool beside) {
  const PagedBatch& b = c.b;
  Few8Args a = {};
  a.b = b;
  a.s = pg_shape(b.nq, b.nkv);
  const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (!encode) return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int D = c.head_dim;
  const int rp = map_pools8(c, encode, c.head_dim, &a.tk, &a.tv);
  if (rp != QD_OK) return rp;
  a.q = static_cast<const char*>(c.q);
  a.k_scale = static_cast<const uint8_t*>(c.k_scale);
  a.v_scale = static_cast<const uint8_t*>(c.v_scale);
  a.out = static_cast<char*>(c.out);
  a.lse = c.lse;
  a.ldq = c.ldq;
  a.ldo = c.ldo;
  a.ld_lse = c.ld_lse;
  a.ss_page = c.ss_page;
  a.ss_head = c.ss_head;
  a.room = (int)std::min((int64_t)b.max_pages * b.page_size, (int64_t)kPgMaxKeys);
  a.inv_group = 65536 / a.s.group + 1;
  a.alone = !beside;
  a.beside = beside;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  const Paged8Plan plan = paged8_plan(c.grid, c.head_dim);
  a.tickets = reinterpret_cast<int*>(static_cast<char*>(c.scratch) + plan.off_few_tickets);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(c.scratch) + plan.off_few);
  const bool bf = c.dtype == QD_BF16;
  const void* fn = bf ? (D == 128 ? (const void*)paged_few8_kernel<__nv_bfloat16, 128> : (const void*)paged_few8_kernel<__nv_bfloat16, 64>)
                      : (D == 128 ? (const void*)paged_few8_kernel<__half, 128> : (const void*)paged_few8_kernel<__half, 64>);
  const int smem = bf ? (D == 128 ? F8Lay<__nv_bfloat16, 128>::total : F8Lay<__nv_bfloat16, 64>::total)
                      : (D == 128 ? F8Lay<__half, 128>::total : F8Lay<__half, 64>::total);
  const int rc = set_max_dynamic_smem(fn, smem);
  if (rc != QD_OK) return rc;
  return launch_kernel(fn, dim3((unsigned)(kF8Resident * c.grid)), dim3(kF8Threads), smem, c.pdl, c.stream, &a);
}

}  // namespace qd
