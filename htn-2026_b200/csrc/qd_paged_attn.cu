// Causal grouped-query attention of a ragged batch's new tokens over cache pages, on the tcgen05 tensor cores.
//
// Rows. The query heads of one KV head share its keys, so a tile of 128 MMA rows holds tpt = 128 / group
// tokens x group heads (row = token * group + head), and a work unit is (request, tile pair, KV head): up to
// two such tiles (A, B) that read the same key blocks. Per block of 128 keys, for each tile x:
//   S_x = Q_x K^T   tcgen05.mma M = 128 rows, N = 128 keys, fp32 in tensor memory
//   softmax         a warpgroup per tile, thread = row: running maximum and sum in fp32,
//                   P = exp2(s * scale * log2 e - m) written over S_x as 16-bit pairs
//   O_x += P_x V    M = 128 rows, N = head_dim, P from tensor memory, V an MN-major operand
// While one warpgroup turns its S into P the tensor cores run the other tile's products. A unit of one tile
// keeps both busy too: A takes its even blocks, B its odd ones, and A's warps add O_B to O_A at the end, each
// with its own maximum. The maximum only moves when a row's grows by more than 2^8 (then the warp rescales
// O_x in tensor memory): O / l does not depend on which maximum is used, and 2^8 leaves the fp32 sums and the
// 16-bit P far from overflow. P is rounded to the 16-bit element type because a 16-bit product of the tensor cores
// takes both operands in it; l sums the unrounded P. Against 64 bits the results are off by 0.0017 to 0.0024 of
// their size in BF16 and 0.00028 in FP16, where their own last rounding alone gives 0.0017 and 0.00021.
//
// Few rows. With at most 16 rows (a single token of up to 16 heads a group, or a few tokens) most of a
// 128-row tile would be exponentials of nothing, so the products are turned round: S^T = K Q^T (M = 128
// keys, N = 16 rows) puts a key in every thread, which has one score per row to deal with; the rows' maxima
// are reduced over the warpgroup, P goes to shared memory as the K-major operand of O^T += V^T P^T (M =
// head_dim, N = 16 rows). Even and odd blocks alternate between the warpgroups as above.
//
// Keys and values come page by page: a copy (TMA, 128-byte swizzle) per page and half of 64 dims (or per page),
// issued by a lane of the producer warp each, into a ring of slots that K and V blocks take in turn. Rows
// past the request's last key hold anything, NaN included: their scores are replaced by -inf before any
// arithmetic, and the MMA warp zeroes their V rows in shared memory (0 x NaN would be NaN).
//
// Split. The key blocks of all units form one line, cut evenly over the CTAs (one per SM) wherever the cuts
// fall: single tokens over long caches, whole prompts and mixtures of them balance alike. A unit that is cut
// leaves fp32 partials (O, m, l) in the scratch, and the CTA that finishes last (a ticket per cut unit)
// joins them in the order of the keys, so results repeat bit for bit. Every CTA finds its place on the line
// from cu_tokens and kv_len itself: no planning launch, and no length is needed on the host.
//
// Measured, 32 query and 8 KV heads of 128 in BF16: 8 single tokens over up to 41 k keys 183 us (HBM: 6.3 TB/s); 64
// single tokens over 1 to 1.5 k keys 72 us (4.7 TB/s: each CTA's start and end); one token over 1 k keys 12.3 us in a
// graph, 14.5 with the keys not in L2 (latency; a call takes the host 11.9); 2048 tokens after 8192 keys 340 to 368 us
// (0.50 to 0.54 of the BF16 peak: a pair's block of 128 keys takes some 4000 cycles, 2048 of them products, since each
// tile's softmax and products wait for one another). Heads of 64 in FP16, 14 over 2: the 64 single tokens 33 us, the 8
// long ones 51. At 168 registers a thread the instances spill: 168 bytes stored and 456 loaded in the code of a
// thread with heads of 128 (156 and 428 with pages of 16 rows), 120 and 356 with heads of 64.
#include <algorithm>
#include <climits>

#include "qd_host.h"
#include "qd_paged_dev.cuh"
#include "qd_paged_line.h"
#include "qd_umma.cuh"

namespace qd {

constexpr int kPgThreads = 384;  // warps 0-3 softmax A, 4-7 softmax B, 8 producer, 9 MMA, 10-11 only start up
// registers per thread after the start: 2 * 224 + 56 = 3 * 168, what the launch gave the three warpgroups
constexpr int kPgSoftmaxRegs = 224, kPgOtherRegs = 56;
constexpr int kPgBox = 128 * 128;  // [128 rows][64 dims] of 16 bits
constexpr int kFewP = 2 * kFewRows * 128;  // its P: 2 halves of 64 keys x 16 rows of 128 B
constexpr int kPgManyUnits = 1 << 20;  // above any grid (whose scratch would be 280 GB); 384 of them fit 32 bits
constexpr int kPgWhole = 8;   // key blocks up to which units of tiles are left whole, when there are CTAs for all

struct alignas(64) PagedAttnArgs {
  CUtensorMap tq, tqf, tq1, tk, tv;  // q boxes: a whole tile's tokens, as many as make 16 rows, one
  PagedBatch b;
  char* out;
  float* lse;
  int64_t ldo, ld_lse;
  PgShape s;
  int room;         // positions in a row of the page table, kPgMaxKeys at most
  int head_groups;  // groups of 8 rows from a KV head of a page to the next
  int inv_group;    // row / group = row * inv_group >> 16 for the rows of a tile
  float scale_log2;
  // [2 * grid slots][2 tiles] of 128 x D floats ([D / 4][128 rows][4], few-row units [rows][D]), then the rows'
  // (m, l) [slots][2][128]
  float* partials;
  int* tickets;     // [grid][2]
};

template <int D>
struct PgLayout {
  static constexpr int kItem = D / 64 * kPgBox;  // a K or V block, and a Q tile
  static constexpr int kSlots = D == 128 ? 5 : 10;
  static constexpr int q = 0;
  static constexpr int kv = q + 2 * kItem;
  static constexpr int p = kv + kSlots * kItem;  // P of few-row units (head_dim 128: in their Q region)
  static constexpr int bars = p + (D == 64 ? 2 * kFewP : 0);
  // qfull[2], qempty[2], sfull[2], pfull[2], odone[2], ofree[2], group[2], segfull[4], segempty[4], join,
  // sload A odd, A even, B, full[slots], empty[slots]
  static constexpr int nbars = 26 + 2 * kSlots;
  static constexpr int seg = bars + nbars * 8;  // segment ring
  static constexpr int misc = seg + 4 * 64;     // tmem slot, abort, line start, flags, drain counts
  static constexpr int ml = misc + 192;         // at a unit's end: (m, l) of the odd blocks' rows [128], or the
                                                // warps' sums of few-row units [2 groups][16 rows][4 warps]
  static constexpr int mx = ml + 1024;          // the warps' maxima of few-row units [2 groups][16][4]
  static constexpr int mb = mx + 1024;          // the odd blocks' maxima of few-row units [16]
  static constexpr int total = mb + 128;
  // where warpgroup x's P of a few-row unit in Q region `reg` is: Q takes the first 4 KiB of each 64-dim half
  static __device__ __forceinline__ int few_p(int reg, int x) {
    return D == 128 ? q + reg * kItem + 4096 + x * kPgBox : p + x * kFewP;
  }
};

// A CTA's piece of a unit: what every warp needs to know of it.
struct PgSeg {
  int row0, ntok, pos0, kv;  // first token row, tokens, the first's position, keys of the request
  int head, j0, nb;          // KV head, first key block, blocks; nb = 0 ends the CTA's list
  int whole;                 // this piece is the whole unit (no partials)
  int few;                   // one tile of at most 16 rows
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
__device__ __forceinline__ void pg_tma_5d(uint32_t dst, const CUtensorMap* map, int z, int w, int v, uint32_t bar,
                                          uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(z), "r"(w), "r"(v), "r"(bar), "l"(policy)
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

// A row's end: 1 / sum of its exponentials, and its log-sum-exp. A sum of 0 is a row that saw no key; a sum that is
// not a number stays one.
__device__ __forceinline__ float pg_inverse(float l) { return l == 0.f ? 0.f : 1.0f / l; }
__device__ __forceinline__ float pg_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

template <int N>
struct Const {
  static constexpr int value = N;
};

// maximum over the warp (NaN where a lane has one only if all have)
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void tmem_ld4_wait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};\n"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};\n"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 64 consecutive columns of this thread's lane, not waited for; and the wait, which ties the registers
__device__ __forceinline__ void tmem_ld64_raw(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld64(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]), "+r"(r[32]), "+r"(r[33]), "+r"(r[34]), "+r"(r[35]), "+r"(r[36]), "+r"(r[37]), "+r"(r[38]), "+r"(r[39]), "+r"(r[40]), "+r"(r[41]), "+r"(r[42]), "+r"(r[43]), "+r"(r[44]), "+r"(r[45]), "+r"(r[46]), "+r"(r[47]), "+r"(r[48]), "+r"(r[49]), "+r"(r[50]), "+r"(r[51]), "+r"(r[52]), "+r"(r[53]), "+r"(r[54]), "+r"(r[55]), "+r"(r[56]), "+r"(r[57]), "+r"(r[58]), "+r"(r[59]), "+r"(r[60]), "+r"(r[61]), "+r"(r[62]), "+r"(r[63])::"memory");
}
__device__ __forceinline__ PgReq pg_request(const PagedAttnArgs& a, int i) {
  return pg_make_request(a.s, ld_i32(a.b.cu + i), ld_i32(a.b.cu + i + 1), ld_i32(a.b.kv_len + i), (int)a.b.tokens, a.room);
}

// Joins a cut few-row unit's pieces (rows of D floats) in the order of their keys: four warps, a row per D / 4
// lanes, kRows such rows at a time with kPieces pieces' loads in flight for each.
template <typename T, int D, int kRows, int kPieces>
__device__ __forceinline__ void pg_join_few(const PagedAttnArgs& a, const PgSeg& g, int r, int rows) {
  constexpr int kAt = 128 / (D / 4);  // rows under way per step of kRows
  const int c4 = r % (D / 4), first = r / (D / 4);
  const float2* const pm = reinterpret_cast<const float2*>(a.partials + (int64_t)2 * gridDim.x * 2 * 128 * D);
#pragma unroll 1
  for (int r0 = first; r0 < rows; r0 += kAt * kRows) {
    float M[kRows], L[kRows];
    float4 acc[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      M[i] = -INFINITY;
      L[i] = 0.f;
      acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll 1
    for (int q0 = 0; q0 < g.nc; q0 += kPieces) {
      float2 ml[kPieces][kRows];
      float4 v[kPieces][kRows];
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int qq = min(q0 + q, g.nc - 1);  // past the last piece: the last again, not counted
        const int64_t at = ((2 * (g.c0 + qq) + (qq == 0 ? 1 : 0)) * 2) * 128;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int64_t row = at + min(r0 + kAt * i, rows - 1);
          ml[q][i] = __ldcg(pm + row);
          v[q][i] = __ldcg(reinterpret_cast<const float4*>(a.partials + row * D) + c4);
        }
      }
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (q0 + q < g.nc && ml[q][i].y != 0.f) {  // a piece in which the row saw no key counts for nothing
            const float mn = fmaxf(M[i], ml[q][i].x), fa = exp2f(M[i] - mn), fb = exp2f(ml[q][i].x - mn);
            M[i] = mn;
            L[i] = L[i] * fa + ml[q][i].y * fb;
            acc[i].x = acc[i].x * fa + v[q][i].x * fb;
            acc[i].y = acc[i].y * fa + v[q][i].y * fb;
            acc[i].z = acc[i].z * fa + v[q][i].z * fb;
            acc[i].w = acc[i].w * fa + v[q][i].w * fb;
          }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = r0 + kAt * i;
      if (row < rows) {
        const float inv = pg_inverse(L[i]);
        const int tok = (row * a.inv_group) >> 16, t2 = g.row0 + tok, h2 = g.head * a.s.group + row - tok * a.s.group;
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + t2 * a.ldo + (int64_t)h2 * D + 4 * c4) =
            make_uint2(Elem<T>::pack(acc[i].x * inv, acc[i].y * inv), Elem<T>::pack(acc[i].z * inv, acc[i].w * inv));
        if (c4 == 0 && a.lse)
          a.lse[t2 * a.ld_lse + h2] = pg_lse(M[i], L[i]);
      }
    }
  }
}

// A K or V block in shared memory: the halves of 64 dims, in each the rows of 128 bytes, 8 to a group; or, merged,
// the groups and in each the halves, so that a page's whole rows are one box of a copy.
template <typename T, int D, bool kMerged>
__global__ void __launch_bounds__(kPgThreads, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  using Lay = PgLayout<D>;
  constexpr int kHalves = D / 64, kSlots = Lay::kSlots;
  constexpr uint32_t kGroup = kMerged ? 2048 : 1024, kHalf = kMerged ? 1024 : kPgBox;  // bytes from one to the next
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
  const uint32_t join = bars + 176;
  // S_A's loads alternate between two barriers: B waits for one that may be two phases away from the last it
  // knows of, and a parity wait two phases ahead (or behind) of a barrier answers wrongly
  auto sload_a = [&](int n) { return bars + ((n & 1) ? 184 : 192); };
  const uint32_t sload_b = bars + 200;
  auto full = [&](int s) { return bars + 208 + 8u * s; };
  auto empty = [&](int s) { return bars + 208 + 8u * (kSlots + s); };
  PgSeg* segs = reinterpret_cast<PgSeg*>(smem + Lay::seg);
  int* misc = reinterpret_cast<int*>(smem + Lay::misc);
  int* abort = misc + 1;
  int64_t* scan = reinterpret_cast<int64_t*>(misc + 12);  // the warps' totals: places, and units
  int* scan_u = misc + 36;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(qfull(x), 1);
      mbar_init(qempty(x), 1);
      mbar_init(sfull(x), 1);
      mbar_init(pfull(x), 4);
      mbar_init(odone(x), 1);
      mbar_init(ofree(x), 4);
      mbar_init(group(x), 4);
      mbar_init(x ? sload_b : sload_a(0), 4);
    }
    mbar_init(join, 4);
    mbar_init(sload_a(1), 4);
    for (int k = 0; k < 4; ++k) {
      mbar_init(segfull(k), 1);
      mbar_init(segempty(k), 9);  // the MMA warp and eight softmax warps
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    fence_mbar_init();
    for (int m = 1; m < 12; ++m) misc[m] = 0;  // (the scan comes after them)
  }
  if (warp == 9) tmem_alloc(smem_u32(misc), 512);

  // ---- this CTA's place on the line: a prefix sum over the requests, and a walk from the one it starts in
  int64_t mine = 0;  // places
  int mine_u = 0;    // and units, of which no more are counted than make the sum larger than any grid
  const int per = (a.b.batch + kPgThreads - 1) / kPgThreads;
  const int i0 = min(tid * per, a.b.batch), i1 = min(i0 + per, a.b.batch);
  PgReq r = {};
  bool cut = false, tiles = false, longer = false;
  for (int i = i0; i < i1; ++i) {
    r = pg_request(a, i);
    tiles |= r.n > a.s.tpf;
    cut |= r.kv != r.pos0 + r.n && r.n > 0;
    mine += a.b.nkv * pg_sum_cost(a.s, r);
    mine_u = (int)min(mine_u + (int64_t)a.b.nkv * r.pairs, (int64_t)kPgManyUnits);
    longer |= r.pairs && pg_blocks(a.s, r, r.pairs - 1) > kPgWhole;
  }
  if (cut && blockIdx.x == 0) flag_error(a.b.err, QD_DEVERR_PAGE);
  int64_t incl = mine;
  int incl_u = mine_u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    const int u = __shfl_up_sync(0xffffffffu, incl_u, o);
    if (lane >= o) {
      incl += v;
      incl_u += u;
    }
  }
  if (lane == 31) {
    scan[warp] = incl;
    scan_u[warp] = incl_u;
  }
  tc_fence_before();
  tiles = __syncthreads_or(tiles);
  longer = __syncthreads_or(longer);
  tc_fence_after();
  grid_dep_launch();
  int units = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 32; ++w) units += scan_u[w];
  // Units of tiles that are few and short are not cut: a place each, and a CTA each
  const bool whole = tiles && !longer && units <= (int)gridDim.x;
  if (whole) {
    mine = mine_u;
    incl = incl_u;
  }
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kPgThreads / 32; ++w) {
    const int64_t v = whole ? scan_u[w] : scan[w];
    if (w < warp) before += v;
    total += v;
  }
  // With little work the first CTAs take kPgPiece places each (a block, if all units have few rows), the rest
  // nothing: joining the pieces of a tile of 128 rows costs about as much as some blocks of keys. No CTA takes
  // less than a block, so that every one between the first and the last of a cut unit has some of it.
  const PgLine line = pg_line(total, (int)gridDim.x, whole ? 1 : tiles ? kPgPiece : kPgBlockCost);
  const int cta = blockIdx.x;
  const int64_t begin = cta < line.ctas ? line.begin(cta) : 0, end = cta < line.ctas ? line.begin(cta + 1) : 0;
  if (begin < end && begin >= before && begin < before + mine) {
    int64_t w = begin - before;
    int i = i0;
    if (per > 1) {
      for (r = pg_request(a, i);; r = pg_request(a, ++i)) {
        const int64_t c = a.b.nkv * (whole ? r.pairs : pg_sum_cost(a.s, r));
        if (w < c) break;
        w -= c;
      }
    }
    const PgPlace at = pg_place(a.s, r, w, whole);
    misc[2] = i;
    misc[3] = at.k;
    misc[4] = at.h;
    misc[5] = at.o;
    *reinterpret_cast<PgReq*>(smem + Lay::mx) = r;
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
    // a lane's copy: a page of the block, and a half of its dims unless they are merged
    constexpr int copies = kMerged ? 1 : kHalves;
    const int boxes = (kPgKeys >> a.b.page_shift) * copies;
    const int box_bytes = a.b.page_size * (D * 2) / copies, my_page = lane / copies, my_half = lane % copies;
    int seg = 0, items = 0, slot = 0, next_region = 0, qfills[2] = {0, 0};
    uint32_t phase = 1;  // of empty(slot): a ring's first round passes at once
    bool ok = true;
    r = *reinterpret_cast<const PgReq*>(smem + Lay::mx);
    __syncwarp();
    // this lane's page of block j of the current request; -2: no box (past the last key)
    auto page_of = [&](int j) {
      const int key = j * kPgKeys + (my_page << a.b.page_shift);
      if (lane >= boxes || key >= r.kv) return -2;
      return max(ld_i32(a.b.table + i * a.b.ld_table + (key >> a.b.page_shift)), -1);
    };
    while (at < end && ok) {
      const int nblk = pg_blocks(a.s, r, k), wt = pg_weight(a.s, r, k), fixed = pg_fixed(a.s, r, k);
      const int len = whole ? 1 : fixed + wt * nblk;
      const int take = (int)min(end - at, (int64_t)(len - o));
      // the blocks whose first places are among these
      const int j0 = whole ? 0 : (max(o - fixed, 0) + wt - 1) / wt;
      const int j1 = whole ? nblk : (max(o + take - fixed, 0) + wt - 1) / wt;
      if (j1 > j0) {
        int page = page_of(j0);
        const int64_t first = at - o + fixed;  // place of the unit's first block
        const int t0 = k * 2 * a.s.tpt, ntok = min(2 * a.s.tpt, r.n - t0);
        const bool two = ntok > a.s.tpt, few = ntok <= a.s.tpf;
        const int ra = two ? 0 : next_region;
        // Q: the regions this unit takes, once their last users are done
        for (int x = 0; x <= (two ? 1 : 0) && ok; ++x) {
          const int reg = two ? x : ra;
          if (qfills[reg] > 0 && !mbar_wait_abort(qempty(reg), (qfills[reg] - 1) & 1, a.b.err, kErrWaitEmpty, abort))
            ok = false;
        }
        if (ok && seg >= 4) ok = mbar_wait_abort(segempty(seg), ((seg >> 2) - 1) & 1, a.b.err, kErrWaitEmpty, abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          for (int x = 0; x <= (two ? 1 : 0); ++x) {
            const int reg = two ? x : ra;
            const bool one = ntok - x * a.s.tpt == 1;
            const CUtensorMap* map = one ? &a.tq1 : few ? &a.tqf : &a.tq;
            mbar_arrive_expect_tx(qfull(reg), kHalves * a.s.group * (one ? 1 : few ? a.s.tpf : a.s.tpt) * 128);
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
              pg_tma_4d(sb + Lay::q + reg * Lay::kItem + hf * kPgBox, map, 64 * hf, 0, h, r.row0 + t0 + x * a.s.tpt,
                        qfull(reg), pol);
            misc[6 + reg] = qfills[reg] + 1;
          }
          const int c0 = whole ? cta : line.owner(first), c1 = whole ? cta : line.owner(first + wt * (nblk - 1));
          PgSeg* s = segs + (seg & 3);
          s->row0 = r.row0 + t0;
          s->ntok = ntok;
          s->pos0 = r.pos0 + t0;
          s->kv = r.kv;
          s->head = h;
          s->j0 = j0;
          s->nb = j1 - j0;
          s->whole = j0 == 0 && j1 == nblk;
          s->few = few;
          s->slot = 2 * cta + (j0 > 0 ? 0 : 1);
          s->c0 = c0;
          s->nc = c1 - c0 + 1;
          s->region = two ? -1 : ra;
          mbar_arrive(segfull(seg));
        }
        for (int x = 0; x <= (two ? 1 : 0); ++x) ++qfills[two ? x : ra];
        next_region = two ? 0 : 1 - ra;
        ++seg;
        // K and V blocks in turn
        for (int j = j0; j < j1 && ok; ++j) {
          const int next = j + 1 < j1 ? page_of(j + 1) : -2;
          const bool need = page != -2;
          const int n_need = __popc(__ballot_sync(0xffffffffu, need));
          if (need && (page < 0 || page >= a.b.n_pages)) {
            flag_error(a.b.err, QD_DEVERR_PAGE);
            page = -1;  // outside the tensor map: the copy fills zeros
          }
          const uint32_t at_page = sb + Lay::kv + my_half * kPgBox + my_page * box_bytes;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const bool got = mbar_wait_abort(empty(slot), phase, a.b.err, kErrWaitEmpty, abort);
            if (!__all_sync(0xffffffffu, got)) {
              ok = false;
              break;
            }
            if (lane == 0) {
              mbar_arrive_expect_tx(full(slot), n_need * box_bytes);
              misc[8] = ++items;
            }
            __syncwarp();
            if (need)
              pg_tma_5d(at_page + slot * Lay::kItem, kv ? &a.tv : &a.tk, my_half, h * a.head_groups, page, full(slot), pol);
            if (++slot == kSlots) {
              slot = 0;
              phase ^= 1;
            }
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
    // ------------------------------------------------------------ MMA: one elected lane waits and issues
    constexpr uint32_t kTypes = (7u << 7) | (7u << 10), kind = Elem<T>::kBf16 ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t id_s = (umma_idesc_bf16(kPgKeys) & ~kTypes) | kind;
    constexpr uint32_t id_o = (umma_idesc_bf16(D, false, true) & ~kTypes) | kind;
    constexpr uint32_t id_sf = (umma_idesc_bf16(kFewRows) & ~kTypes) | kind;
    constexpr uint32_t id_of = (umma_idesc_bf16(kFewRows, true, false) & ~kTypes) | kind;
    // low words of the operand descriptors: a start address in units of 16 B, so steps are plain additions
    const uint32_t d_q = umma_desc_lo(sb + Lay::q), d_k = umma_desc_lo(sb + Lay::kv);
    const uint32_t d_v = umma_desc_lo(sb + Lay::kv, kHalf);
    // few rows, head_dim 64: the 64 upper rows of O^T repeat the lower ones (block stride 0)
    const uint32_t d_vf = umma_desc_lo(sb + Lay::kv, D == 128 ? kHalf : 0);
    constexpr uint32_t kItem16 = Lay::kItem >> 4;
    int slot = 0, pc[2] = {0, 0}, units[2] = {0, 0};
    uint32_t phase = 0, quse = 0;  // of full(slot); bit r: the phase of qfull(r)
    int pairs = 0;                 // blocks of units of two tiles so far
    const bool leader = elect_one();
    bool ok = true;
    auto wait = [&](uint32_t bar, int parity) {
      if (ok) ok = mbar_wait_abort(bar, parity & 1, a.b.err, kErrWaitFull, abort);
    };
    struct Ring {
      int slot;
      uint32_t phase;
    };
    auto ahead = [&](int n) {  // the item n places on
      const int t = slot + n;
      return t >= kSlots ? Ring{t - kSlots, phase ^ 1u} : Ring{t, phase};
    };
    auto advance = [&](int n) {
      const Ring t = ahead(n);
      slot = t.slot;
      phase = t.phase;
    };
    // every product that reads P has been done
    auto wait_pv = [&](int x) {
      if (pc[x] > 0) wait(odone(x), pc[x] - 1);
    };
    // S_x = Q K^T
    auto issue_s = [&](auto xc, auto fewc, int reg, Ring k) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value;
      constexpr bool few = decltype(fewc)::value != 0;
      wait(full(k.slot), k.phase);
      tc_fence_after();
      if (ok) {
        const uint32_t q = d_q + reg * kItem16, kt = d_k + k.slot * kItem16;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {  // 16 dims per MMA: +32 B inside a 64-dim half, the next half after 4
          const uint32_t q_d = q + (((d >> 2) * kPgBox + (d & 3) * 32) >> 4), k_d = kt + (((d >> 2) * kHalf + (d & 3) * 32) >> 4);
          if constexpr (few)
            umma_f16<kGroup, 1024>(tS(x), k_d, q_d, id_sf, d > 0 ? 1u : 0u);
          else
            umma_f16<1024, kGroup>(tS(x), q_d, k_d, id_s, d > 0 ? 1u : 0u);
        }
      }
      umma_commit(sfull(x));
    };
    // O_x += P_x V
    auto issue_pv = [&](auto xc, auto modec, int reg, Ring v, bool first) __attribute__((always_inline)) {
      constexpr int x = decltype(xc)::value;
      constexpr bool few = decltype(modec)::value == 1, pair = decltype(modec)::value == 2;
      if (first && units[x] > 0) wait(ofree(x), units[x] - 1);
      const uint32_t vt = (few ? d_vf : d_v) + v.slot * kItem16;
      const uint32_t pt = umma_desc_lo(sb + Lay::few_p(reg, x));
      wait(pfull(x), pc[x]);
      tc_fence_after();
      if (ok) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {  // 16 keys per MMA: 8 columns of P pairs; V two 8-key atoms
          const uint32_t acc = kk ? 1u : first ? 0u : 1u;
          const uint32_t v_k = vt + kk * (2 * kGroup >> 4);
          if constexpr (few)
            umma_f16<kGroup, 1024>(tO(x), v_k, pt + (((kk >> 2) * (kFewP / 2) + (kk & 3) * 32) >> 4), id_of, acc);
          else
            umma_f16_ts<kGroup>(tO(x), tS(pair ? 1 - x : x) + 8 * kk, v_k, id_o, acc);
        }
      }
      ++pc[x];
      umma_commit(odone(x));
    };
    // `rows` of V are keys; the ones past them hold anything and are zeroed (the whole warp comes here)
    auto zero_v = [&](int rows, Ring v) {
      if (leader) wait(full(v.slot), v.phase);
      __syncwarp();
      char* const vt = smem + Lay::kv + v.slot * Lay::kItem;
#pragma unroll 1
      for (int c = max(rows, 0) * 8 + lane; c < kPgKeys * 8; c += 32)
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf)
          *reinterpret_cast<uint4*>(vt + (c >> 6) * kGroup + hf * kHalf + (c & 63) * 16) = make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_smem();
      __syncwarp();
    };
    const Const<0> c0;
    const Const<1> c1;
    const Const<2> c2;
    // Two tiles over the same blocks. Each tile's P goes over the other's S, which that has long loaded: so the
    // next S of a tile does not wait for its own P to be used up, and S_A runs a block ahead:
    //   S_A 0, S_B 0, S_A 1;  PV_A j, S_B j+1, PV_B j, S_A j+2
    auto pair_unit = [&](const PgSeg& g) {
      if (leader) {
        wait(qfull(0), quse);
        wait(qfull(1), quse >> 1);
        wait_pv(0);
        wait_pv(1);
        issue_s(c0, c0, 0, ahead(0));
        issue_s(c1, c0, 1, ahead(0));
        if (g.nb > 1) {
          umma_commit(empty(slot));
          wait(sload_a(pairs), pairs >> 1);
          issue_s(c0, c0, 0, ahead(2));
        } else {
          umma_commit(qempty(0));
          umma_commit(qempty(1));
        }
      }
#pragma unroll 1
      for (int j = 0; j < g.nb; ++j) {
        const Ring v = ahead(1), k1 = ahead(2), k2 = ahead(4);
        const int rows = g.kv - (g.j0 + j) * kPgKeys;
        if (rows < kPgKeys) zero_v(rows, v);
        if (leader) {
          wait(full(v.slot), v.phase);
          issue_pv(c0, c2, 0, v, j == 0);
          if (j + 1 < g.nb) {
            wait_pv(0);  // S_B's columns hold P_A
            issue_s(c1, c0, 1, k1);
            if (j + 2 == g.nb) {
              umma_commit(qempty(0));
              umma_commit(qempty(1));
            } else {
              umma_commit(empty(k1.slot));
            }
          }
          issue_pv(c1, c2, 0, v, j == 0);
          if (j + 1 < g.nb) umma_commit(empty(v.slot));  // the last K and V slots: the softmax warps' to give back
          if (j + 2 < g.nb) {
            wait_pv(1);
            issue_s(c0, c0, 0, k2);
          }
        }
        advance(2);
        __syncwarp();
      }
      quse ^= 3;
      pairs += g.nb;
      ++units[0];
      ++units[1];
    };
    // one tile: its even blocks in S_A, O_A, its odd ones in S_B, O_B; K_j+2 is asked for after V_j
    auto single_unit = [&](const PgSeg& g, auto fewc) {
      constexpr bool few = decltype(fewc)::value != 0;
      const int reg = g.region;
      if (leader) {
        wait(qfull(reg), quse >> reg);
        wait_pv(0);
        wait_pv(1);
        issue_s(c0, fewc, reg, ahead(0));
        umma_commit(empty(slot));
        if (g.nb > 1) {
          issue_s(c1, fewc, reg, ahead(2));
          umma_commit(empty(ahead(2).slot));
        }
      }
      auto block = [&](auto xc, int j) __attribute__((always_inline)) {
        const Ring v = ahead(1), k = ahead(4);
        const int rows = g.kv - (g.j0 + j) * kPgKeys;
        if (rows < kPgKeys) zero_v(rows, v);
        if (leader) {
          wait(full(v.slot), v.phase);
          issue_pv(xc, fewc, reg, v, j < 2);
          if (few || j + 1 < g.nb) umma_commit(empty(v.slot));  // else the softmax warps' to give back
          if (j + 2 < g.nb) {
            wait_pv(decltype(xc)::value);
            issue_s(xc, fewc, reg, k);
            umma_commit(empty(k.slot));
          }
          // the region is free after the last S products; a few-row unit's P is in it too
          if (few ? j + 1 == g.nb : (j + 3 == g.nb || (g.nb < 3 && j == 0))) umma_commit(qempty(reg));
        }
        advance(2);
        __syncwarp();
      };
#pragma unroll 1
      for (int j = 0; j < g.nb; j += 2) {
        block(c0, j);
        if (j + 1 < g.nb) block(c1, j + 1);
      }
      quse ^= 1u << reg;
      ++units[0];
      if (g.nb > 1) ++units[1];
    };
#pragma unroll 1
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!__all_sync(0xffffffffu, ok)) break;
      const PgSeg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      if (g.region < 0)
        pair_unit(g);
      else if (g.few)
        single_unit(g, c1);
      else
        single_unit(g, c0);
      if (!__all_sync(0xffffffffu, ok)) break;
    }
    if (leader)  // no MMA may still run when its memory is given back
      for (int x = 0; x < 2; ++x)
        if (pc[x] > 0) mbar_wait(odone(x), (pc[x] - 1) & 1, a.b.err, kErrDrain);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPgSoftmaxRegs));
    // ------------------------------------------------------------ softmax and epilogue: warpgroup x = tile x
    const int x = warp >> 2, r = 32 * (warp & 3) + lane;  // (r: the row, no longer the request)
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    int cnt = 0, pairs = 0, blocks = 0, meets = 0, joins = 0;  // blocks: of all units so far
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
    float2* const pm = reinterpret_cast<float2*>(a.partials + (int64_t)2 * gridDim.x * 2 * 128 * D);
    // a few-row piece's row, and four dims of a tile's rows
    auto part_o = [&](int slot, int row) { return a.partials + ((int64_t)slot * 2 * 128 + row) * D; };
    auto part_c = [&](int slot, int c4) {
      return reinterpret_cast<float4*>(a.partials) + ((int64_t)(slot * 2 + x) * (D / 4) + c4) * 128;
    };
    auto part_m = [&](int slot, int row) { return pm + (slot * 2 + x) * 128 + row; };
    // A cut unit: whoever finishes last (true) joins the pieces. Their stores are made visible by the barrier
    // and the ticket (release is cumulative).
    auto is_last = [&](const PgSeg& g) {
      meet();
      if (!ok) return false;
      if (r == 0) {
        const bool last = atom_add_acq_rel(a.tickets + 2 * g.c0 + x, 1) == g.nc - 1;
        if (last) a.tickets[2 * g.c0 + x] = 0;
        misc[10 + x] = last;
      }
      meet();
      return ok && misc[10 + x] != 0;
    };
    // A unit of at most kC rows on this warpgroup's blocks: thread r has key r of the block (and, of O^T, dim r);
    // what there is one of per row (maximum, factors) is lane c's for row c, the same in all four warps.
    auto few_rows = [&](auto cols, const PgSeg& g, int rows, bool joined) __attribute__((always_inline)) {
      constexpr int kC = decltype(cols)::value;
      auto load_cols = [&](uint32_t taddr, uint32_t* v) {
        if constexpr (kC == 4)
          tmem_ld4_wait(taddr, v);
        else {
          tmem_ld16_raw(taddr, v);
          tmem_wait_ld16(v);
        }
      };
      float4* const mx = reinterpret_cast<float4*>(smem + Lay::mx) + x * kFewRows;
      float4* const sums = reinterpret_cast<float4*>(smem + Lay::ml);
      float* const mb = reinterpret_cast<float*>(smem + Lay::mb);
      char* const p_row = smem + Lay::few_p(g.region, x) + (r >> 6) * (kFewP / 2) + (r & 7) * 2;
      const int chunk = (r & 63) >> 3, wg = warp & 3;
      float m = -INFINITY;  // of row `lane`
      float l[kC];          // of every row, this thread's keys
#pragma unroll
      for (int c = 0; c < kC; ++c) l[c] = 0.f;
#pragma unroll 1
      for (int j = x; j < g.nb; j += 2, ++cnt) {
        wait(sfull(x), cnt);
        if (!ok) return;
        tc_fence_after();
        uint32_t sv[kC];
        load_cols(tS(x) + lane_off, sv);
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
            if (key >= min(lim, g.kv)) sv[c] = __float_as_uint(-INFINITY);
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float v = redux_max(__uint_as_float(sv[c]));
          top = lane == c ? v : top;
        }
        if (lane < rows) reinterpret_cast<float*>(mx + lane)[wg] = top;
        meet();
        if (!ok) return;
        float mn = -INFINITY;
        if (lane < rows) {
          const float4 v = mx[lane];
          mn = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) * a.scale_log2;
        }
        if (__any_sync(0xffffffffu, mn > m + 8.f)) {  // the same in every warp of the group
          const float m_to = fmaxf(m, mn), alpha = m_to == -INFINITY ? 1.f : exp2f(m - m_to);
          m = m_to;
          if (j > x) {
            uint32_t o[kC];
            load_cols(tO(x) + lane_off, o);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
              const float f = __shfl_sync(0xffffffffu, alpha, c);
              o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              l[c] *= f;
            }
            if constexpr (kC == 4)
              tmem_st4(tO(x) + lane_off, o);
            else
              tmem_st16(tO(x) + lane_off, o);
          }
        }
        const float nm = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float p = pg_ex2(fmaf(__uint_as_float(sv[c]), a.scale_log2, __shfl_sync(0xffffffffu, nm, c)));
          l[c] += p;
          const uint32_t w = Elem<T>::pack(p, 0.f);  // rounded: the operand's type
          *reinterpret_cast<uint16_t*>(p_row + c * 128 + ((chunk ^ (c & 7)) << 4)) = (uint16_t)w;
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
      if (x == 1) {  // tile A's warps (same lanes of tensor memory) take O_B from here
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
      uint32_t o[kC], ob[kC];
      load_cols(tO(0) + lane_off, o);
      if (joined) load_cols(tO(1) + lane_off, ob);
      float fa = 1.f, fb = 0.f;
      int64_t row_at = 0;  // of row `lane`, in elements
      if (lane < rows) {
        const float4 s = sums[lane];
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
          if (wg == 0 && a.lse)
            a.lse[(g.row0 + tok) * a.ld_lse + hq] = pg_lse(M, L);
        } else if (wg == 0) {
          __stcg(part_m(g.slot, lane), make_float2(M, L));
        }
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        float v = __uint_as_float(o[c]) * __shfl_sync(0xffffffffu, fa, c);
        const float f = __shfl_sync(0xffffffffu, fb, c);
        const int64_t to = __shfl_sync(0xffffffffu, row_at, c);
        if (joined) v = fmaf(__uint_as_float(ob[c]), f, v);
        if (c < rows && r < D) {
          if (g.whole)
            reinterpret_cast<uint16_t*>(a.out)[to + r] = (uint16_t)Elem<T>::pack(v, 0.f);
          else
            __stcg(part_o(g.slot, c) + r, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ofree(0));
        if (joined) mbar_arrive(ofree(1));
      }
    };
    for (int seg = 0;; ++seg) {
      wait(segfull(seg), seg >> 2);
      if (!ok) break;
      const PgSeg g = segs[seg & 3];
      __syncwarp();
      if (lane == 0) mbar_arrive(segempty(seg));
      if (g.nb == 0) break;
      blocks += g.nb;
      const bool two = g.region < 0, joined = !two && g.nb > 1;
      if (x == 1 && !two && !joined) continue;  // one tile, one block
      const int t0 = two ? x * a.s.tpt : 0;       // this tile's first token
      const int ntok = min(a.s.tpt, g.ntok - t0), rows = ntok * a.s.group;
      const int my_tok = (r * a.inv_group) >> 16, tok = g.row0 + t0 + my_tok;
      const int head = g.head * a.s.group + r - my_tok * a.s.group;
      // keys this row sees: up to its own position (MMA rows past the last token hold anything)
      const int lim = r < rows ? min(g.kv, g.pos0 + t0 + my_tok + 1) : INT_MAX;
      const bool idle = (r & ~31) >= rows;  // no row of this warp is a token's
      float m_used = -INFINITY, l = 0.f;
      const int jf = two ? 0 : x;
      if (g.few) {
        if (rows <= 4)
          few_rows(Const<4>(), g, rows, joined);
        else
          few_rows(Const<kFewRows>(), g, rows, joined);
        if (!ok) break;
        if (x == 1 || g.whole) continue;
        if (is_last(g)) {
          if (rows <= 4)
            pg_join_few<T, D, 1, 4>(a, g, r, rows);
          else
            pg_join_few<T, D, 2, 2>(a, g, r, rows);
        }
        if (!ok) break;
        continue;
      }
      const int step = two ? 1 : 2;  // one tile: the even blocks, or the odd ones
      for (int j = jf; j < g.nb; j += step, ++cnt) {
        wait(sfull(x), cnt);
        if (!ok) break;
        tc_fence_after();
        uint32_t sv[128];
        if (!idle) {
          tmem_ld64(tS(x) + lane_off, sv);
          tmem_ld64_raw(tS(x) + lane_off + 64, sv + 64);
        }
        const int left = lim - (g.j0 + j) * kPgKeys;
        float m_new = -INFINITY;
        if (!idle) {
          const bool part = __any_sync(0xffffffffu, left < kPgKeys);
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t* const v = sv + 64 * hf;
            if (hf) tmem_wait_ld64(v);
            if (part) {
#pragma unroll
              for (int e = 0; e < 64; ++e)
                if (64 * hf + e >= left) v[e] = __float_as_uint(-INFINITY);
            }
#pragma unroll
            for (int e = 0; e < 64; e += 8)
#pragma unroll
              for (int c = 0; c < 4; ++c)
                m4[c] = pg_max3(m4[c], __uint_as_float(v[e + 2 * c]), __uint_as_float(v[e + 2 * c + 1]));
          }
          m_new = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
          if (r >= rows) m_new = -INFINITY;  // what a row holds that is no token's must not move its warp's maxima
        }
        if (two) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(x ? sload_b : sload_a(pairs + j));
        }
        if (!idle) {
          // warp-uniform (tensor-memory loads and stores are warp-collective)
          if (__any_sync(0xffffffffu, m_new > m_used + 8.f)) {
            const float m_to = fmaxf(m_used, m_new);
            const float alpha = m_to == -INFINITY ? 1.f : exp2f(m_used - m_to);
            if (j > jf) {
              wait(odone(x), cnt - 1);  // O_x with every block before this one
              tc_fence_after();
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
        }
        if (!idle) {
          const float nm = m_used == -INFINITY ? 0.f : -m_used;  // a row that has seen no key yet: P = 0
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 64; ++c) {  // P pair c = keys 2c, 2c + 1, rounded (the operand's type), over the scores
            const float p0 = pg_ex2(fmaf(__uint_as_float(sv[2 * c]), a.scale_log2, nm));
            const float p1 = pg_ex2(fmaf(__uint_as_float(sv[2 * c + 1]), a.scale_log2, nm));
            ls[(2 * c) & 3] += p0;
            ls[(2 * c + 1) & 3] += p1;
            sv[c] = Elem<T>::pack(p0, p1);
          }
          l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
          if (two) {  // over the other tile's S, once that has loaded it (B: the one A is ahead with, whose
                      // products were issued after B's last P was used up)
            const int n = pairs + min(j + 1, g.nb - 1);  // the S_A that A has by now
            if (x == 0)
              wait(sload_b, pairs + j);
            else if (j == 0 || j + 1 < g.nb)
              wait(sload_a(n), n >> 1);
            else  // no S_A comes after B's last P but one, which has to be used up before the last
              wait(odone(1), cnt - 1);
            tc_fence_after();
          }
          tmem_st64(tS(two ? 1 - x : x) + lane_off, sv);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull(x));
        // the next S may come before this P is complete: a warp without rows must not arrive twice for it
        if (idle && two) wait(pfull(x), cnt);
      }
      if (two) pairs += g.nb;
      wait(odone(x), cnt - 1);
      if (!ok) break;
      tc_fence_after();
      float2* const ml = reinterpret_cast<float2*>(smem + Lay::ml);
      if (joined && x == 1) {  // the odd blocks: tile A's warps (same lanes of tensor memory) take O_B from here
        ml[r] = make_float2(m_used, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(join);
        continue;
      }
      float fa = 1.f, fb = 0.f;
      if (joined) {
        wait(join, joins++);
        if (!ok) break;
        tc_fence_after();
        const float2 o = ml[r];
        const float m = fmaxf(m_used, o.x);
        if (m != -INFINITY) {
          fa = exp2f(m_used - m);
          fb = exp2f(o.x - m);
        }
        l = l * fa + o.y * fb;
        m_used = m;
      }
      // Rows go out through the shared memory of the unit's last V block (of two tiles, A: its last K block, whose
      // products were issued before those that this warpgroup has waited for; V is B's, which comes last): thread
      // r lays down row r, 16-byte chunks swizzled by row, and whole rows are stored from there (row by row from
      // the registers would be partial sectors, 32 lines an instruction: 7 k cycles).
      const int it = 2 * blocks - 1 - (two ? 1 - x : 0), slot = it % kSlots;
      char* const stage = smem + Lay::kv + slot * Lay::kItem;
      auto lay_down = [&](int c, const uint32_t* w) {  // dims 8 c .. 8 c + 7, packed
        *reinterpret_cast<uint4*>(stage + r * (2 * D) + ((c ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      auto store_rows = [&]() {
        meet();
#pragma unroll 1
        for (int i = r; i < rows * (D / 8); i += 128) {
          const int row = i / (D / 8), c = i % (D / 8), rt = (row * a.inv_group) >> 16;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + row * (2 * D) + ((c ^ (row & 7)) << 4));
          T* const to = reinterpret_cast<T*>(a.out) + (g.row0 + t0 + rt) * a.ldo +
                        (int64_t)(g.head * a.s.group + row - rt * a.s.group) * D + 8 * c;
          *reinterpret_cast<uint4*>(to) = v;
        }
      };
      const float norm = !g.whole ? 1.f : pg_inverse(l);  // a piece's rows stay as they are
      fa *= norm;
      fb *= norm;
      if (!idle) {
#pragma unroll 1
        for (int c4 = 0; c4 < D / 32; ++c4) {
          uint32_t o[32];
          tmem_ld32(tO(x) + lane_off + 32 * c4, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fa);
          if (joined) {
            uint32_t ob[32];
            tmem_ld32(tO(1) + lane_off + 32 * c4, ob);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = __float_as_uint(fmaf(__uint_as_float(ob[e]), fb, __uint_as_float(o[e])));
          }
          if (g.whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = Elem<T>::pack(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
#pragma unroll
            for (int c = 0; c < 4; ++c) lay_down(4 * c4 + c, o + 4 * c);
          } else if (r < rows) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              __stcg(part_c(g.slot, 8 * c4 + c) + r, make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]),
                                                                 __uint_as_float(o[4 * c + 2]), __uint_as_float(o[4 * c + 3])));
          }
        }
        if (r < rows && !g.whole) __stcg(part_m(g.slot, r), make_float2(m_used, l));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ofree(x));
        if (joined) mbar_arrive(ofree(1));
      }
      bool out_rows = g.whole;
      if (!g.whole && is_last(g)) {  // join the pieces in the order of their keys
        out_rows = true;
        // kP pieces of 4 / kP times 8 dims of a row at a time: 8 loads in flight, none twice where a unit is cut once
        // (16 in flight spill)
        auto join_pieces = [&](auto pieces) __attribute__((always_inline)) {
          constexpr int kP = decltype(pieces)::value, kI = 4 / kP;
          const int items = rows * (D / 8);
#pragma unroll 1
          for (int e0 = r; e0 < items; e0 += 128 * kI) {
            float M[kI], L[kI], acc[kI][8];
            int c8[kI], row[kI];
#pragma unroll
            for (int i = 0; i < kI; ++i) {
              const int e = min(e0 + 128 * i, items - 1);
              c8[i] = e / rows;
              row[i] = e - c8[i] * rows;
              M[i] = -INFINITY;
              L[i] = 0.f;
#pragma unroll
              for (int d = 0; d < 8; ++d) acc[i][d] = 0.f;
            }
#pragma unroll 1
            for (int q0 = 0; q0 < g.nc; q0 += kP) {
              float2 p[kI][kP];
              float4 v[kI][kP][2];
#pragma unroll
              for (int i = 0; i < kI; ++i)
#pragma unroll
                for (int q = 0; q < kP; ++q) {
                  const int qq = min(q0 + q, g.nc - 1), slot_q = 2 * (g.c0 + qq) + (qq == 0 ? 1 : 0);
                  p[i][q] = __ldcg(part_m(slot_q, row[i]));
                  v[i][q][0] = __ldcg(part_c(slot_q, 2 * c8[i]) + row[i]);
                  v[i][q][1] = __ldcg(part_c(slot_q, 2 * c8[i] + 1) + row[i]);
                }
#pragma unroll
              for (int i = 0; i < kI; ++i)
#pragma unroll
                for (int q = 0; q < kP; ++q)
                  if (q0 + q < g.nc && p[i][q].y != 0.f) {  // a piece in which the row saw no key counts for nothing
                    const float mn = fmaxf(M[i], p[i][q].x), wa = exp2f(M[i] - mn), wb = exp2f(p[i][q].x - mn);
                    M[i] = mn;
                    L[i] = L[i] * wa + p[i][q].y * wb;
                    const float4 lo = v[i][q][0], hi = v[i][q][1];
                    const float u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[i][d] = acc[i][d] * wa + u[d] * wb;
                  }
            }
#pragma unroll
            for (int i = 0; i < kI; ++i) {
              if (e0 + 128 * i >= items) break;
              const float inv = pg_inverse(L[i]);
              uint32_t w[4];
#pragma unroll
              for (int d = 0; d < 4; ++d) w[d] = Elem<T>::pack(acc[i][2 * d] * inv, acc[i][2 * d + 1] * inv);
              *reinterpret_cast<uint4*>(stage + row[i] * (2 * D) + ((c8[i] ^ (row[i] & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
              if (c8[i] == 0 && a.lse) {
                const int rt = (row[i] * a.inv_group) >> 16;
                a.lse[(g.row0 + t0 + rt) * a.ld_lse + g.head * a.s.group + row[i] - rt * a.s.group] =
                    pg_lse(M[i], L[i]);
              }
            }
          }
        };
        if (g.nc == 2)
          join_pieces(Const<2>());
        else
          join_pieces(Const<4>());
      }
      if (!ok) break;
      if (out_rows) {
        store_rows();
        if (!ok) break;
        if (g.whole && r < rows && a.lse)
          a.lse[tok * a.ld_lse + head] = pg_lse(m_used, l);
      }
      fence_proxy_async_smem();  // the slot's next contents come by TMA
      meet();
      if (!ok) break;
      if (r == 0) mbar_arrive(empty(slot));
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

template <typename T>
static const void* attn_kernel(int head_dim, bool merged) {
  return head_dim == 64 ? (const void*)paged_attn_kernel<T, 64, false>
         : merged       ? (const void*)paged_attn_kernel<T, 128, true>
                        : (const void*)paged_attn_kernel<T, 128, false>;
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
  if ((tokens > 0 && (!q || !out)) || !aligned16(q) || !aligned16(out) || ldq % 8 || ldo % 8 || ldq < (int64_t)nq_heads * head_dim ||
      ldo < (int64_t)nq_heads * head_dim || (lse && ld_lse < nq_heads) || !(scale > 0.f))
    return set_error(QD_ERR_ARG, "paged attention: q / out / lse null, misaligned or with a bad stride (%lld, %lld, %lld), or scale %g",
                     (long long)ldq, (long long)ldo, (long long)ld_lse, (double)scale);
  const PagedAttnPlan plan = paged_attn_plan(grid < 1 ? 1 : grid, head_dim);
  if (grid < 1 || !scratch || scratch_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(scratch) & 31))
    return set_error(QD_ERR_SCRATCH, "paged attention: grid %d needs %lld B of 32-byte aligned scratch (have %lld)", grid,
                     (long long)plan.bytes, (long long)scratch_bytes);
  if (ps_head % (8 * head_dim))
    return set_error(QD_ERR_ARG, "paged attention: head stride %lld (whole groups of 8 rows)", (long long)ps_head);
  if (tokens == 0) return QD_OK;
  const PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
  if (!encode) return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  a.s = pg_shape(nq_heads, nkv_heads);
  a.room = (int)std::min((int64_t)max_pages * page_size, (int64_t)kPgMaxKeys);
  a.inv_group = 65536 / a.s.group + 1;  // exact: the excess is below 128 / 65536, a fraction's distance to 1 at least 1 / 128
  const CUtensorMapDataType type = dtype == QD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  auto map4 = [&](CUtensorMap* m, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
    return encode(m, type, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  {  // a tile's rows are token-major, its KV head's query heads inner
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)a.s.group, (cuuint64_t)nkv_heads, (cuuint64_t)tokens};
    const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)a.s.group * head_dim * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)a.s.group, 1, (cuuint32_t)a.s.tpt}, box1[4] = {64, (cuuint32_t)a.s.group, 1, 1};
    const cuuint32_t boxf[4] = {64, (cuuint32_t)a.s.group, 1, (cuuint32_t)(a.s.tpf > 0 ? a.s.tpf : 1)};
    if (!map4(&a.tq, q, dims, strides, box) || !map4(&a.tqf, q, dims, strides, boxf) || !map4(&a.tq1, q, dims, strides, box1))
      return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for q");
  }
  // Pages of 16 rows are merged: half the copies (64 decoding requests 71 us, 84 apart). Larger pages are not: the
  // products read the interleaved rows slower (a chunk of 2048 after 8192 keys 349 us, 341 apart).
  const bool merged = page_size == 16 && head_dim == 128;
  {  // a page of a KV head: 64 dims x 8 rows x halves x groups of 8 rows, in that order; heads are whole groups apart
    const int64_t group = 8 * (int64_t)head_dim;
    a.head_groups = (int)(ps_head / group);
    const cuuint64_t dims[5] = {64, 8, (cuuint64_t)head_dim / 64, (cuuint64_t)((nkv_heads - 1) * (ps_head / group) + page_size / 8),
                                (cuuint64_t)n_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)head_dim * 2, 128, (cuuint64_t)group * 2, (cuuint64_t)ps_page * 2};
    const cuuint32_t box[5] = {64, 8, merged ? (cuuint32_t)head_dim / 64 : 1, (cuuint32_t)page_size / 8, 1}, one[5] = {1, 1, 1, 1, 1};
    for (int v = 0; v < 2; ++v)
      if (encode(v ? &a.tv : &a.tk, type, 5, const_cast<void*>(v ? v_pages : k_pages), dims, strides, box, one,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return set_error(QD_ERR_CUDA, "cuTensorMapEncodeTiled failed for the pools");
  }
  a.out = static_cast<char*>(out);
  a.lse = lse;
  a.ldo = ldo;
  a.ld_lse = ld_lse;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.tickets = static_cast<int*>(scratch);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(scratch) + plan.off_partials);
  const void* fn = dtype == QD_BF16 ? attn_kernel<__nv_bfloat16>(head_dim, merged) : attn_kernel<__half>(head_dim, merged);
  const int smem = head_dim == 128 ? PgLayout<128>::total : PgLayout<64>::total;
  const int rs = set_max_dynamic_smem(fn, smem);
  if (rs != QD_OK) return rs;
  return launch_kernel(fn, dim3((unsigned)grid), dim3(kPgThreads), smem, pdl, stream, &a);
}
