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
// The key blocks of all units form one line that is cut evenly over the CTAs; blocks alternate between two warpgroups,
// across the units too, and the scores of the next two blocks are always under way. Pieces of a cut unit are left in the
// scratch and joined in the order of their keys by the CTA that ends last.
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>

#include "qd_host.h"
#include "qd_paged_attn8.h"
#include "qd_paged_attn_dev.cuh"

namespace qd {

constexpr int kF8Threads = 384;  // warps 0-3 softmax A, 4-7 softmax B, 8 producer, 9 MMA, 10-11 the queries' terms
constexpr int kF8Scales = 8;     // blocks whose scales are in shared memory
constexpr int kF8Bias = 7;       // P' is up to 2^(8 + 7): the upper end of E5M2's range

template <typename T, int D>
struct F8Lay {
  static constexpr int kTQ = Elem<T>::kBf16 ? 2 : 3, kTP = Elem<T>::kBf16 ? 3 : 4;  // terms
  static constexpr int kItem = kPgKeys * D;         // a K or V block
  static constexpr int kQ = kFewRows * kTQ * D;     // a unit's queries
  static constexpr int kP = kFewRows * kTP * kPgKeys;
  static constexpr int kSlots = D == 128 ? 11 : 20;
  static constexpr int q = 0;                       // two units'
  static constexpr int p = q + 2 * kQ;              // the two warpgroups'
  static constexpr int kv = p + 2 * kP;
  static constexpr int sc = kv + kSlots * kItem;    // [block][K, V][128 keys]
  static constexpr int bars = sc + kF8Scales * 2 * kPgKeys;
  // q8full[2], qempty[2], sfull[2], pfull[2], odone[2], ofree[2], group[2], segfull[4], segempty[4], join, then
  // scfull[], scempty[], full[], empty[]
  static constexpr int nbars = 23 + 2 * kF8Scales + 2 * kSlots;
  static constexpr int seg = bars + (nbars * 8 + 63) / 64 * 64;
  static constexpr int qs = seg + 4 * 64;     // the queries' powers of two [2 units][16]
  static constexpr int misc = qs + 128;       // tmem, abort, line start, last flags, drain counts; then the scan's totals
  static constexpr int sums = misc + 256;     // the warps' sums [2 groups][16 rows][4 warps]
  static constexpr int mx = sums + 512;       // and maxima
  static constexpr int mb = mx + 512;         // warpgroup B's maxima [16]
  static constexpr int total = mb + 64;
  static_assert(kQ % 1024 == 0 && kP % 1024 == 0 && kItem % 1024 == 0, "operands start on 1 KiB");
  static_assert(total <= 227 * 1024, "shared memory of an SM");
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
  float scale_log2;
  float* partials;  // [2 * grid slots][16 rows][D], then the rows' (m, l)
  int* tickets;     // [grid][2], of which the first
};

struct F8Seg {
  int row0, ntok, pos0, kv;  // first token row, tokens, the first's position, keys of the request
  int head, j0, nb, whole;   // KV head, first key block, blocks (0 ends the list), all of the unit's
  int slot, c0, nc;          // partial slot, first CTA and number of CTAs of the unit
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
// N columns of this thread's lane of tensor memory, in steps of 16, waited for
template <int N>
__device__ __forceinline__ void f8_load(uint32_t taddr, uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; i += 16) tmem_ld16_raw(taddr + i, r + i);
#pragma unroll
  for (int i = 0; i < N; i += 16) tmem_wait_ld16(r + i);
}
constexpr int f8_cols(int n) { return (n + 15) / 16 * 16; }

// one request's blocks in this kernel (0: not its)
__device__ __forceinline__ int f8_blocks(const PgShape& s, const PgReq& r) {
  return r.n > 0 && r.n <= s.tpf ? pg_max((pg_min(r.kv, r.pos0 + r.n) + kPgKeys - 1) / kPgKeys, 1) : 0;
}

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
__global__ void __launch_bounds__(kF8Threads, 1) paged_few8_kernel(const __grid_constant__ Few8Args a) {
  using Lay = F8Lay<T, D>;
  constexpr int kSlots = Lay::kSlots, kTQ = Lay::kTQ, kTP = Lay::kTP;
  extern __shared__ __align__(1024) char smem[];
  const uint32_t sb = smem_u32(smem), bars = sb + Lay::bars;
  auto q8full = [&](int s) { return bars + 8u * (s & 1); };
  auto qempty = [&](int s) { return bars + 16 + 8u * (s & 1); };
  auto sfull = [&](int x) { return bars + 32 + 8u * x; };
  auto pfull = [&](int x) { return bars + 48 + 8u * x; };
  auto odone = [&](int x) { return bars + 64 + 8u * x; };
  auto ofree = [&](int x) { return bars + 80 + 8u * x; };
  auto group = [&](int x) { return bars + 96 + 8u * x; };
  auto segfull = [&](int s) { return bars + 112 + 8u * (s & 3); };
  auto segempty = [&](int s) { return bars + 144 + 8u * (s & 3); };
  const uint32_t join = bars + 176;
  auto scfull = [&](int b) { return bars + 184 + 8u * (b & (kF8Scales - 1)); };
  auto scempty = [&](int b) { return bars + 184 + 8u * (kF8Scales + (b & (kF8Scales - 1))); };
  auto full = [&](int s) { return bars + 184 + 8u * (2 * kF8Scales + s); };
  auto empty = [&](int s) { return bars + 184 + 8u * (2 * kF8Scales + kSlots + s); };
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
      mbar_init(q8full(x), 2);
      mbar_init(qempty(x), 9);  // the MMA's products and eight softmax warps
      mbar_init(sfull(x), 1);
      mbar_init(pfull(x), 4);
      mbar_init(odone(x), 1);
      mbar_init(ofree(x), 4);
      mbar_init(group(x), 4);
    }
    for (int k = 0; k < 4; ++k) {
      mbar_init(segfull(k), 1);
      mbar_init(segempty(k), 11);  // the MMA warp, eight softmax warps, two for the queries
    }
    mbar_init(join, 4);
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
  if (warp == 9) tmem_alloc(smem_u32(misc), 256);
  grid_dep_wait();

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
    mine += (int64_t)a.b.nkv * nb;
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
        const int64_t c = (int64_t)a.b.nkv * f8_blocks(a.s, r);
        if (w < c) break;
        w -= c;
      }
    }
    const int nb = f8_blocks(a.s, r);
    misc[2] = i;
    misc[3] = (int)(w / nb);
    misc[4] = (int)(w % nb);
    *reinterpret_cast<PgReq*>(smem + Lay::mx) = r;
  }
  __syncthreads();
  const uint32_t tmem = (uint32_t)misc[0];
  auto tS = [&](int x) { return tmem + 64u * x; };
  auto tO = [&](int x) { return tmem + 128u + 64u * x; };

  if (warp == 8) {
    // ------------------------------------------------------------ producer: all lanes walk the line
    const uint64_t pol = policy_evict_normal();
    int64_t at = begin;
    int i = misc[2], h = misc[3], o = misc[4];
    const int boxes = kPgKeys >> a.b.page_shift, box_bytes = a.b.page_size * D;
    int seg = 0, blk = 0, slot = 0;
    uint32_t phase = 1;  // of empty(slot): a ring's first round passes at once
    bool ok = true;
    r = *reinterpret_cast<const PgReq*>(smem + Lay::mx);
    __syncwarp();
    // this lane's page of block j of the current request; -2: none (past the last key)
    auto page_of = [&](int j) {
      const int key = j * kPgKeys + (lane << a.b.page_shift);
      if (lane >= boxes || key >= r.kv) return -2;
      return max(ld_i32(a.b.table + i * a.b.ld_table + (key >> a.b.page_shift)), -1);
    };
    while (at < end && ok) {
      const int nblk = f8_blocks(a.s, r), take = (int)min(end - at, (int64_t)(nblk - o));
      const int j0 = o, j1 = o + take;
      int page = page_of(j0);
      if (seg >= 4) ok = mbar_wait_abort(segempty(seg), ((seg >> 2) - 1) & 1, a.b.err, kErrWaitEmpty, abort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        const int64_t first = at - o;
        const int c0 = line.owner(first), c1 = line.owner(first + nblk - 1);
        F8Seg* s = segs + (seg & 3);
        s->row0 = r.row0;
        s->ntok = r.n;
        s->pos0 = r.pos0;
        s->kv = r.kv;
        s->head = h;
        s->j0 = j0;
        s->nb = take;
        s->whole = take == nblk;
        s->slot = 2 * cta + (j0 > 0 ? 0 : 1);
        s->c0 = c0;
        s->nc = c1 - c0 + 1;
        mbar_arrive(segfull(seg));
      }
      ++seg;
      for (int j = j0; j < j1 && ok; ++j, ++blk) {
        const int next = j + 1 < j1 ? page_of(j + 1) : -2;
        const bool need = page != -2;
        bool in = need;
        if (need && (page < 0 || page >= a.b.n_pages)) {
          flag_error(a.b.err, QD_DEVERR_PAGE);
          page = -1;  // outside the tensor map: the copy fills zeros
          in = false;
        }
        const int n_need = __popc(__ballot_sync(0xffffffffu, need)), n_in = __popc(__ballot_sync(0xffffffffu, in));
        {  // the rows' powers of two
          const bool got = mbar_wait_abort(scempty(blk), ((blk / kF8Scales) & 1) ^ 1, a.b.err, kErrWaitEmpty, abort);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
          const int at_scale = Lay::sc + (blk & (kF8Scales - 1)) * 2 * kPgKeys + (lane << a.b.page_shift);
          if (need && !in) {
            for (int c = 0; c < a.b.page_size; c += 16) {
              *reinterpret_cast<uint4*>(smem + at_scale + c) = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
              *reinterpret_cast<uint4*>(smem + at_scale + kPgKeys + c) = make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
            }
            fence_proxy_async_smem();  // a later block's come by copies
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_expect_tx(scfull(blk), n_in * a.b.page_size * 2);
            misc[9] = blk + 1;
          }
          __syncwarp();
          if (in) {
            const int64_t from = page * a.ss_page + h * a.ss_head;
            bulk_g2s(sb + at_scale, a.k_scale + from, a.b.page_size, scfull(blk), pol);
            bulk_g2s(sb + at_scale + kPgKeys, a.v_scale + from, a.b.page_size, scfull(blk), pol);
          }
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const bool got = mbar_wait_abort(empty(slot), phase, a.b.err, kErrWaitEmpty, abort);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(full(slot), n_need * box_bytes);
            misc[8] = 2 * blk + kv + 1;
          }
          __syncwarp();
          if (need)
            pg_tma_4d(sb + Lay::kv + slot * Lay::kItem + lane * box_bytes, kv ? &a.tv : &a.tk, 0, 0, h, page, full(slot), pol);
          if (++slot == kSlots) {
            slot = 0;
            phase ^= 1;
          }
        }
        page = next;
      }
      at += take;
      o = 0;
      if (at < end && ++h == a.b.nkv) {
        h = 0;
        do r = request(++i);
        while (f8_blocks(a.s, r) == 0);
      }
    }
    // the end of the list: a segment without blocks
    if (ok && seg >= 4) ok = mbar_wait_abort(segempty(seg), ((seg >> 2) - 1) & 1, a.b.err, kErrWaitEmpty, abort);
    if (ok && lane == 0) {
      segs[seg & 3].nb = 0;
      mbar_arrive(segfull(seg));
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA: one elected lane waits and issues
    constexpr uint32_t hi = f8_desc_hi<D>(), hi_p = f8_desc_hi<128>(), kItem16 = Lay::kItem >> 4;
    const uint32_t d_q = umma_desc_lo(sb + Lay::q), d_k = umma_desc_lo(sb + Lay::kv), d_p = umma_desc_lo(sb + Lay::p);
    // heads of 64: the 64 upper rows of O^T repeat the lower ones (block stride 0)
    const uint32_t d_v = umma_desc_lo(sb + Lay::kv, 0);
    int slot = 0, pc[2] = {0, 0}, units[2] = {0, 0};  // slot: of the next V product's K block
    uint32_t phase = 0;
    int s_seg = 0, s_left = 0, s_blk = 0, s_slot = 0;  // of the next scores
    uint32_t s_phase = 0, s_id = 0;
    bool s_end = false, ok = true;
    const bool leader = elect_one();
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
    };
    // the scores of the next block on the line, whichever unit's it is
    auto next_scores = [&]() {
      if (s_end || !ok) return;
      if (s_left == 0) {
        wait(segfull(s_seg), s_seg >> 2);
        if (!ok) return;
        const F8Seg& g = segs[s_seg & 3];
        s_left = g.nb;
        if (s_left == 0) {
          s_end = true;
          return;
        }
        s_id = g.ntok * a.s.group <= 4 ? f8_idesc(f8_cols(4 * kTQ), false, false) : f8_idesc(kFewRows * kTQ, false, false);
        wait(q8full(s_seg), s_seg >> 1);
      }
      const int x = s_blk & 1;
      wait(full(s_slot), s_phase);
      tc_fence_after();
      if (ok) {
        const uint32_t qt = d_q + (s_seg & 1) * (Lay::kQ >> 4), kt = d_k + s_slot * kItem16;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) umma_f8<hi, hi>(tS(x), kt + 2 * d, qt + 2 * d, s_id, d > 0 ? 1u : 0u);
      }
      umma_commit(sfull(x));
      umma_commit(empty(s_slot));
      ++s_blk;
      s_slot += 2;
      if (s_slot >= kSlots) {
        s_slot -= kSlots;
        s_phase ^= 1;
      }
      if (--s_left == 0) umma_commit(qempty(s_seg++));
    };
    // `rows` of V are keys; the ones past them hold anything and are zeroed (the whole warp comes here)
    auto zero_v = [&](int rows, int s, uint32_t ph) {
      if (leader) wait(full(s), ph);
      __syncwarp();
      char* const vt = smem + Lay::kv + s * Lay::kItem;
#pragma unroll 1
      for (int c = max(rows, 0) * (D / 16) + lane; c < kPgKeys * (D / 16); c += 32)
        *reinterpret_cast<uint4*>(vt + 16 * c) = make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_smem();
      __syncwarp();
    };
    if (leader) {
      next_scores();
      next_scores();
    }
    __syncwarp();
    int b = 0;
#pragma unroll 1
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int nb = segs[seg & 3].nb, keys = segs[seg & 3].kv - segs[seg & 3].j0 * kPgKeys;
      const bool four = segs[seg & 3].ntok * a.s.group <= 4;
      __syncwarp();
      if (nb == 0) break;
      const uint32_t id = four ? f8_idesc(f8_cols(4 * kTP), true, true) : f8_idesc(kFewRows * kTP, true, true);
#pragma unroll 1
      for (int j = 0; j < nb; ++j, ++b) {
        const int x = b & 1, v = slot + 1 == kSlots ? 0 : slot + 1;
        const uint32_t v_phase = slot + 1 == kSlots ? phase ^ 1u : phase;
        const int rows = keys - j * kPgKeys;
        if (rows < kPgKeys) zero_v(rows, v, v_phase);
        if (leader) {
          wait(full(v), v_phase);
          if (j < 2 && units[x] > 0) wait(ofree(x), units[x] - 1);
          wait(pfull(x), pc[x]);
          tc_fence_after();
          if (ok) {
            const uint32_t vt = d_v + v * kItem16, pt = d_p + x * (Lay::kP >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 32 keys per MMA: four groups of 8 rows of V
              umma_f8<hi, hi_p>(tO(x), vt + k * (32 * D >> 4), pt + 2 * k, id, k ? 1u : j < 2 ? 0u : 1u);
          }
          ++pc[x];
          umma_commit(odone(x));
          umma_commit(empty(v));
          next_scores();
        }
        if (j < 2) ++units[x];
        slot += 2;
        if (slot >= kSlots) {
          slot -= kSlots;
          phase ^= 1;
        }
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(segempty(seg));  // (the scores are at most two blocks ahead, in a ring of four)
    }
    if (leader)  // no MMA may still run when its memory is given back
      for (int x = 0; x < 2; ++x)
        if (pc[x] > 0) mbar_wait(odone(x), (pc[x] - 1) & 1, a.b.err, kErrDrain);
  } else if (warp >= 10) {
    // ------------------------------------------------------------ the queries' terms, a unit ahead
    constexpr int kLanes = D / 8, kAt = 32 / kLanes;  // lanes of a row, rows at a time
    const int sub = lane % kLanes;
    bool ok = true;
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
      if (seg >= 2) wait(qempty(seg), (seg >> 1) - 1);
      if (!ok) break;
      const int rows = g.ntok * a.s.group, step = rows <= 4 ? 4 : kFewRows;
      char* const to = smem + Lay::q + (seg & 1) * Lay::kQ;
#pragma unroll 1
      for (int c0 = (warp - 10) * kAt; c0 < rows; c0 += 2 * kAt) {
        const int c = min(c0 + lane / kLanes, rows - 1);  // (past the last row: that one again)
        const int tok = (c * a.inv_group) >> 16, hq = g.head * a.s.group + c - tok * a.s.group;
        const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (g.row0 + tok) * a.ldq +
                                                        (int64_t)hq * D + 8 * sub);
        float x[8], most = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Elem<T>::unpack((&u.x)[k]);
          x[2 * k] = f.x;
          x[2 * k + 1] = f.y;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[k]) <= FLT_MAX ? fabsf(x[k]) : 0.f);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
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
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w[k], __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * k] = (x[2 * k] - f.x) * 16.f;
            x[2 * k + 1] = (x[2 * k + 1] - f.y) * 16.f;
          }
          const int n = t * step + c, sw = D == 128 ? n & 7 : (n >> 1) & 3;
          *reinterpret_cast<uint2*>(to + n * D + (((sub >> 1) ^ sw) << 4) + (sub & 1) * 8) =
              make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
        }
        if (sub == 0) reinterpret_cast<float*>(smem + Lay::qs)[(seg & 1) * kFewRows + c] = __uint_as_float((uint32_t)(127 + e) << 23);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q8full(seg));
    }
  } else {
    // ------------------------------------------------------------ softmax and epilogue: every second block
    const int x = warp >> 2, r = 32 * (warp & 3) + lane, wg = warp & 3;  // (r: the key, or the dim of O^T)
    const uint32_t lane_off = (uint32_t)(32 * wg) << 16;
    int cnt = 0, b0 = 0, meets = 0, joins = 0;  // blocks of this group, of all units so far
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto meet = [&]() {  // the four warps of this group; bounded, unlike a named barrier
      __syncwarp();
      if (lane == 0) mbar_arrive(group(x));
      wait(group(x), meets++);
    };
    float2* const pm = reinterpret_cast<float2*>(a.partials + (int64_t)2 * gridDim.x * kFewRows * D);
    float4* const mx = reinterpret_cast<float4*>(smem + Lay::mx) + x * kFewRows;
    float4* const sums = reinterpret_cast<float4*>(smem + Lay::sums);
    float* const mb = reinterpret_cast<float*>(smem + Lay::mb);
    char* const p_to = smem + Lay::p + x * Lay::kP + (r & 15);
    auto unit = [&](auto cols, const F8Seg& g, int seg) __attribute__((always_inline)) {
      constexpr int kC = decltype(cols)::value, kSc = f8_cols(kC * kTQ), kOc = f8_cols(kC * kTP);
      const int rows = g.ntok * a.s.group, jf = (b0 ^ x) & 1;  // this group's first block
      const bool joined = g.nb > 1;
      wait(q8full(seg), seg >> 1);
      if (!ok) return;
      const float sc = lane < rows ? reinterpret_cast<const float*>(smem + Lay::qs)[(seg & 1) * kFewRows + lane] * a.scale_log2 : 0.f;
      __syncwarp();
      if (lane == 0) mbar_arrive(qempty(seg));
      if (jf >= g.nb) return;
      float m = -INFINITY;  // of row `lane`
      float l[kC];          // of every row, this thread's keys
#pragma unroll
      for (int c = 0; c < kC; ++c) l[c] = 0.f;
#pragma unroll 1
      for (int j = jf; j < g.nb; j += 2, ++cnt) {
        const int b = b0 + j;
        wait(scfull(b), b / kF8Scales);
        if (!ok) return;
        const uint8_t* const two = reinterpret_cast<const uint8_t*>(smem) + Lay::sc + (b & (kF8Scales - 1)) * 2 * kPgKeys;
        const float ks = __uint_as_float((uint32_t)two[r] << 23), ev = (float)two[kPgKeys + r] - 127.f;
        __syncwarp();
        if (lane == 0) mbar_arrive(scempty(b));
        wait(sfull(x), cnt);
        if (!ok) return;
        tc_fence_after();
        float t[kC];  // the weights' exponents, in twos
        {
          uint32_t sv[kSc];
          f8_load<kSc>(tS(x) + lane_off, sv);
#pragma unroll
          for (int c = 0; c < kC; ++c) {
            float s = __uint_as_float(sv[c + (kTQ - 1) * kC]);
#pragma unroll
            for (int q = kTQ - 2; q >= 0; --q) s = fmaf(s, 0.0625f, __uint_as_float(sv[c + q * kC]));
            t[c] = fmaf(s * ks, __shfl_sync(0xffffffffu, sc, c), ev);
          }
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
        }
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float v = redux_max(t[c]);
          top = lane == c ? v : top;
        }
        if (lane < rows) reinterpret_cast<float*>(mx + lane)[wg] = top;
        meet();
        if (!ok) return;
        float mn = -INFINITY;
        if (lane < rows) {
          const float4 v = mx[lane];
          mn = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
        }
        if (__any_sync(0xffffffffu, mn > m + 8.f)) {  // the same in every warp of the group
          const float m_to = fmaxf(m, mn), alpha = m_to == -INFINITY ? 1.f : exp2f(m - m_to);
          m = m_to;
          if (j > jf) {
            uint32_t o[kOc];
            f8_load<kOc>(tO(x) + lane_off, o);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
              const float f = __shfl_sync(0xffffffffu, alpha, c);
#pragma unroll
              for (int q = 0; q < kTP; ++q) o[c + q * kC] = __float_as_uint(__uint_as_float(o[c + q * kC]) * f);
              l[c] *= f;
            }
#pragma unroll
            for (int i = 0; i < kOc; i += 16) tmem_st16(tO(x) + lane_off + i, o + i);
          }
        }
        const float nm = m == -INFINITY ? (float)kF8Bias : kF8Bias - m, per_code = exp2f(-ev);
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
        if (lane == 0) mbar_arrive(pfull(x));
      }
      wait(odone(x), cnt - 1);
      if (!ok) return;
      tc_fence_after();
      {  // the warps' sums of every row, side by side
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int c = 0; c < kC; ++c) l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
        float mine = 0.f;
#pragma unroll
        for (int c = 0; c < kC; ++c) mine = lane == c ? l[c] : mine;
        if (lane < rows) reinterpret_cast<float*>(sums + x * kFewRows + lane)[wg] = mine;
      }
      if (x == 1 && joined) {  // A's warps (same lanes of tensor memory) take O_B from here
        if (wg == 0 && lane < rows) mb[lane] = m;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(join);
        return;
      }
      meet();
      if (ok && joined) wait(join, joins++);
      if (!ok) return;
      tc_fence_after();
      float ov[kC], ob[kC];
      auto load_o = [&](int y, float* v) {
        uint32_t o[kOc];
        f8_load<kOc>(tO(y) + lane_off, o);
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          v[c] = __uint_as_float(o[c + (kTP - 1) * kC]);
#pragma unroll
          for (int q = kTP - 2; q >= 0; --q) v[c] = fmaf(v[c], 0.125f, __uint_as_float(o[c + q * kC]));
        }
      };
      load_o(x, ov);
      if (joined) load_o(1, ob);
      float fa = 1.f, fb = 0.f;
      int64_t row_at = 0;  // of row `lane`, in elements
      if (lane < rows) {
        const float4 s = sums[x * kFewRows + lane];
        float L = (s.x + s.y) + (s.z + s.w), M = m;
        if (joined) {
          const float4 s2 = sums[kFewRows + lane];
          const float m2 = mb[lane], mn = fmaxf(M, m2);
          fa = mn == -INFINITY ? 1.f : exp2f(M - mn);
          fb = mn == -INFINITY ? 0.f : exp2f(m2 - mn);
          L = L * fa + ((s2.x + s2.y) + (s2.z + s2.w)) * fb;
          M = mn;
        }
        const int tok = (lane * a.inv_group) >> 16, hq = g.head * a.s.group + lane - tok * a.s.group;
        row_at = (g.row0 + tok) * a.ldo + (int64_t)hq * D;
        if (g.whole) {
          const float inv = pg_inverse(L);
          fa *= inv;
          fb *= inv;
          if (wg == 0 && a.lse) a.lse[(g.row0 + tok) * a.ld_lse + hq] = pg_lse(M - kF8Bias, L);
        } else if (wg == 0) {
          __stcg(pm + (int64_t)g.slot * kFewRows + lane, make_float2(M, L));
        }
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        float v = ov[c] * __shfl_sync(0xffffffffu, fa, c);
        const float f = __shfl_sync(0xffffffffu, fb, c);
        const int64_t to = __shfl_sync(0xffffffffu, row_at, c);
        if (joined) v = fmaf(ob[c], f, v);
        if (c < rows && r < D) {
          if (g.whole)
            reinterpret_cast<uint16_t*>(a.out)[to + r] = (uint16_t)Elem<T>::pack(v, 0.f);
          else
            __stcg(a.partials + ((int64_t)g.slot * kFewRows + c) * D + r, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ofree(x));
        if (joined) mbar_arrive(ofree(1));
      }
      if (g.whole) return;
      // a cut unit: whoever finishes last joins the pieces. Their stores are made visible by the barrier and the
      // ticket (release is cumulative)
      meet();
      if (!ok) return;
      if (r == 0) {
        const bool last = atom_add_acq_rel(a.tickets + 2 * g.c0, 1) == g.nc - 1;
        if (last) a.tickets[2 * g.c0] = 0;
        misc[10 + x] = last;
      }
      meet();
      if (ok && misc[10 + x]) f8_join<T, D>(a, g, r, rows);
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
      b0 += g.nb;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 256);
  if (tid == 0) {  // no copy may still be writing shared memory when the CTA exits
    const int n = misc[8], k = misc[9];
    for (int it = max(n - kSlots, 0); it < n; ++it)
      if (!mbar_wait(full(it % kSlots), (it / kSlots) & 1, a.b.err, kErrDrain)) break;
    for (int it = max(k - kF8Scales, 0); it < k; ++it)
      if (!mbar_wait(scfull(it), (it / kF8Scales) & 1, a.b.err, kErrDrain)) break;
  }
}

int launch_few8(const Paged8Call& c, bool alone) {
  const PagedBatch& b = c.b;
  Few8Args a = {};
  a.b = b;
  a.s = pg_shape(b.nq, b.nkv);
  const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (!encode) return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int D = c.head_dim;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)b.page_size, (cuuint64_t)b.nkv, (cuuint64_t)b.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)D, (cuuint64_t)b.ps_head, (cuuint64_t)b.ps_page};
  const cuuint32_t box[4] = {(cuuint32_t)D, (cuuint32_t)b.page_size, 1, 1}, one[4] = {1, 1, 1, 1};
  for (int v = 0; v < 2; ++v)
    if (encode(v ? &a.tv : &a.tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(v ? c.v_pages : c.k_pages), dims, strides,
               box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for the pools");
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
  a.alone = alone;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.tickets = static_cast<int*>(c.scratch);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(c.scratch) + paged_attn_plan(c.grid, D).off_partials);
  const bool bf = c.dtype == QD_BF16;
  const void* fn = bf ? (D == 128 ? (const void*)paged_few8_kernel<__nv_bfloat16, 128> : (const void*)paged_few8_kernel<__nv_bfloat16, 64>)
                      : (D == 128 ? (const void*)paged_few8_kernel<__half, 128> : (const void*)paged_few8_kernel<__half, 64>);
  const int smem = bf ? (D == 128 ? F8Lay<__nv_bfloat16, 128>::total : F8Lay<__nv_bfloat16, 64>::total)
                      : (D == 128 ? F8Lay<__half, 128>::total : F8Lay<__half, 64>::total);
  const int rc = set_max_dynamic_smem(fn, smem);
  if (rc != QD_OK) return rc;
  return launch_kernel(fn, dim3((unsigned)c.grid), dim3(kF8Threads), smem, c.pdl, c.stream, &a);
}

}  // namespace qd
