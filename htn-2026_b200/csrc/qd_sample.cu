// A token per row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number.
//
// The weights are whole multiples of 2^-40 of the row's largest, so every sum is an exact 64-bit integer
// and the kept set and the token do not depend on how the additions are split. With the logits as
// order-preserving 32-bit keys the kept set is a prefix of the tokens ordered by (key descending, index):
// all keys above a threshold, and of the keys equal to it the first few by index.
//
// The logits are read from memory once: a cluster of up to 8 CTAs holds a row in shared memory (38 KB a CTA
// for 151,936 BF16 logits), each CTA a contiguous part and each of its warps a contiguous part of that, so
// sums by warp are sums in index order. Values that all CTAs need go to every CTA's memory (distributed
// shared memory) behind a cluster barrier.
//   1  load, largest logit
//   2  (top-k or top-p) a histogram over up to 2048 equal steps of d down to the weights that round to 0, summed
//      over the cluster by shares of bins: the bin in which the prefix ends, by weight sometimes two. A bin holds
//      its number of tokens and bounds of its weight; the exact weight of all is added up beside it
//   3  one pass for the exact weight above that bracket, and its tokens, a few hundred, gathered by CTA. Every
//      CTA takes all of them, ranks them and finds the last one kept. A bracket of more than 1024 (many ties, a
//      high temperature) is cut again, by key, first
//   4  the kept weight of every warp (known from 3, unless min-p cuts off more), the warp in which u falls, and
//      the walk through its tokens by all warps of its CTA
// Without top-k and top-p only 1 and 4 are left, and the weights are computed once.
//
// Measured with 151,936 BF16 logits a row: one row 8 us unfiltered, 17 us with top-k, 21 us with top-p; 64 rows
// 18, 31 and 50 us; 256 rows 65 us (1.2 TB/s), 113 and 160 us; 256 unfiltered FP32 rows 101 us. A row's chain
// bounds it: some 20 barriers of the CTA or the cluster (1000 to 1500 cycles each for the cluster's) with two CTAs
// an SM to fill them, and for many filtered rows the instructions and shared-memory additions of 2 and 3 (20,000
// and 11,000 of 58,000 cycles of a row with top-p).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qd_common.cuh"
#include "qd_host.h"

namespace qd {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 1024;               // tokens that are sorted, kSampleOwn a thread
constexpr int kSampleOwn = kSampleList / kSampleThreads;
constexpr float kSampleOne = 1099511627776.0f;  // 2^40
constexpr float kSampleDeep = 28.5f;            // e^-28.42 = 2^-41: beyond, weights round to 0
constexpr int64_t kSampleMaxVocab = 1 << 18;    // 2^18 weights of 2^40 stay below 2^63
constexpr int kSampleMaxCluster = 8;

struct SampleArgs {
  const void* logits;
  int64_t ld, vocab;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *u;
  int64_t* tok;
  float* logprob;
  int per_warp;  // logits per warp, a multiple of 8
  int wide;      // rows are 16-byte aligned
};

// a 16-byte vector of logits, as floats
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ uint32_t lowest() { return 0xff800000u; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf_lo(w[i]);
      x[2 * i + 1] = bf_hi(w[i]);
    }
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ uint32_t lowest() { return 0xff80ff80u; }
};
template <>
struct Vec<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
  static __device__ __forceinline__ uint32_t lowest() { return 0xfc00fc00u; }
};

// larger logit = larger key; -0 and +0 are the same key, NaN the key of -inf
__device__ __forceinline__ uint32_t logit_key(float l) {
  if (l != l) l = -INFINITY;
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// d = (l - m) / temperature of the definition, for a finite m (NaN for a NaN logit: below every bound)
__device__ __forceinline__ float logit_depth(float l, float m, float inv_t) { return __fmul_rn(__fsub_rn(l, m), inv_t); }
// w = expf(d) <= 1 as a whole number of 2^-40: hi = floor(w 2^20) and lo = the rest, rounded to even, each in
// the low bits of a float of 2^23 (adding 2^23 rounds to a whole number). Six instructions and no carry where
// a 64-bit conversion and addition take some twenty; the bits above are taken off once per sum.
constexpr uint32_t kHalfBits = 0x4b000000u;
__device__ __forceinline__ void weight_halves(float w, uint32_t& hi, uint32_t& lo) {
  const float h = __fmaf_rd(w, 1048576.0f, 8388608.0f);
  const float rest = __fmaf_rn(w, 1048576.0f, -(h - 8388608.0f));
  hi = __float_as_uint(h);
  lo = __float_as_uint(__fmaf_rn(rest, 1048576.0f, 8388608.0f));
}
__device__ __forceinline__ uint64_t depth_weight(float d) {
  uint32_t hi, lo;
  weight_halves(expf(d), hi, lo);
  return ((uint64_t)(hi - kHalfBits) << 20) + (lo - kHalfBits);
}
// d in 256ths of the steps into which 0 to -kSampleDeep is cut, rounded down (a larger number for what is deeper,
// -inf or NaN). An addition of 2^23 here too: a conversion to int would take the exponentials' pipe.
__device__ __forceinline__ uint32_t depth_place(float d, float per_d256) {
  return __float_as_uint(__fmaf_rd(-d, per_d256, 8388608.0f)) - kHalfBits;
}

// 64-bit sum over the warp by 16-bit pieces: four reduction instructions in place of ten dependent shuffles
__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    s += (uint64_t)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> (16 * i)) & 0xffffu) << (16 * i);
  return s;
}
__device__ __forceinline__ uint64_t warp_scan64(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  return v;
}

struct Trio64 {
  uint64_t a, b, c;
};
// Where a prefix ends: in the bins `bin` to `last`, which hold `n` tokens, after `count` tokens of `weight`.
struct Bracket {
  uint64_t count, weight;
  int bin, last, n;
};
// The bin of which this thread has the cluster's sums (none: 0), and the sums before it.
struct BinSums {
  uint32_t n;
  uint64_t w, count, weight, total_count, total_weight;
  bool complete;  // the words' numbers add up to the tokens counted (they are never more)
};

struct SampleShared {
  union {
    struct {
      uint64_t weight[kSampleBins];  // of the bins by key
      uint32_t cnt[kSampleBins];     // this CTA's histogram
    };
    struct {  // once all have read that, the bracket's tokens: this CTA's, all, and the weights up to each
      uint64_t list[kSampleList], sorted[kSampleList], sums[kSampleList];
    };
  };
  Trio64 xch[2][kSampleMaxCluster];  // values of every CTA, two exchanges in turn
  uint64_t warp_a[kSampleWarps], warp_b[kSampleWarps];
  Bracket found;
  int found_last;
  uint64_t found_after;       // tokens up to the bracket's end
  uint64_t cut_weight, cut;   // weight of the prefix, its last token
  unsigned long long part_w[kSampleWarps];  // per warp: weight of all, then of the tokens above the bracket or kept
  uint32_t part_eq[kSampleWarps];           // and its ties
  unsigned long long above[2];  // weight of this CTA's tokens above the bracket, by top-k and by top-p
  int list_n[2];              // this CTA's tokens in the bracket, by top-k and by top-p
  uint32_t key_min, key_max, counted;
};
constexpr int kSampleShared = (sizeof(SampleShared) + 15) / 16 * 16;

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int kVec = Vec<T>::n;
  extern __shared__ __align__(16) char smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  uint4* const part = reinterpret_cast<uint4*>(smem_raw + kSampleShared);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / C;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;");  // waited for before the first store to another CTA
  grid_dep_wait();
  grid_dep_launch();

  // ---- 1: this warp's logits into shared memory (past the row's end: -inf), and the largest
  const int n = (int)a.vocab, vecs = a.per_warp / kVec;
  const int first = (rank * kSampleWarps + warp) * a.per_warp;  // index of this warp's first logit
  uint4* const mine = part + warp * vecs;
  const T* const x = static_cast<const T*>(a.logits) + row * a.ld + first;
  // the row's parameters come with the logits
  const float temp = a.temperature ? a.temperature[row] : 1.f, p = a.top_p ? a.top_p[row] : 1.f;
  const float mp = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
  const int k = a.top_k ? a.top_k[row] : 0;
  uint64_t best = 0;  // (key, ~index): the lowest index among equals
  {
    constexpr int kAhead = 4;  // vectors in flight per lane
    float top = -INFINITY;
    int top_i = 0;  // the first vector that has it
    for (int v0 = lane; v0 < vecs; v0 += 32 * kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = v0 + 32 * k;
        const int left = n - first - i * kVec;
        v[k] = make_uint4(Vec<T>::lowest(), Vec<T>::lowest(), Vec<T>::lowest(), Vec<T>::lowest());
        if (i < vecs && left >= kVec && a.wide) {
          v[k] = __ldcs(reinterpret_cast<const uint4*>(x) + i);
        } else if (i < vecs) {
          T* e = reinterpret_cast<T*>(&v[k]);
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (j < left) e[j] = x[(int64_t)i * kVec + j];
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = v0 + 32 * k;
        if (i >= vecs) break;
        mine[i] = v[k];
        float f[kVec];
        Vec<T>::get(v[k], f);
        float most = f[0];
#pragma unroll
        for (int j = 1; j < kVec; ++j) most = fmaxf(most, f[j]);
        if (most > top) {  // this lane's indices ascend, so the first of equals stays
          top = most;
          top_i = i;
        }
      }
    }
    if (top > -INFINITY) {
      float f[kVec];
      Vec<T>::get(mine[top_i], f);
      int at = 0;
#pragma unroll
      for (int j = kVec - 1; j >= 0; --j) at = f[j] == top ? j : at;
      best = ((uint64_t)logit_key(top) << 32) | (uint32_t)~(first + top_i * kVec + at);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) sh.warp_a[warp] = best;
  if (tid == 0) {
    sh.list_n[0] = sh.list_n[1] = 0;
    sh.above[0] = sh.above[1] = 0;
    sh.counted = 0;
  }
  __syncthreads();
  // a CTA's shared memory may be written to from outside only once the CTA runs: all have, long before this
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  int turn = 0;
  // (va, vb, vc), known to warp 0, to every CTA of the cluster; all threads pass the barrier
  auto exchange = [&](uint64_t va, uint64_t vb, uint64_t vc) {
    if (tid < C) *cluster.map_shared_rank(&sh.xch[turn][rank], tid) = Trio64{va, vb, vc};
    cluster.sync();
    const Trio64* r = sh.xch[turn];
    turn ^= 1;
    return r;
  };
  if (warp == 0) {
    best = lane < kSampleWarps ? sh.warp_a[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
      best = c > best ? c : best;
    }
  }
  {
    const Trio64* r = exchange(best, 0, 0);
    best = 0;
    for (int c = 0; c < C; ++c) best = r[c].a > best ? r[c].a : best;
  }
  const float m = best ? key_logit((uint32_t)(best >> 32)) : -INFINITY;
  if (m == -INFINITY || !(temp >= 1e-5f)) {
    if (rank == 0 && tid == 0) {
      a.tok[row] = m == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
      if (a.logprob) a.logprob[row] = m == -INFINITY ? m : 0.f;
    }
    return;  // (nothing of a CTA's memory is used by others after its last barrier)
  }
  // +inf logits share everything at any temperature: ties at the top, of which the filters keep the first
  const bool top_inf = m == INFINITY;
  // (an infinite temperature's 1 / T = 0 would make NaN of masked logits: any d that rounds to weight 1 will do)
  const float inv_t = fmaxf(__fdiv_rn(1.f, temp), 1e-38f);

  // f(kVec logits, index of the first) over this warp's vectors
  auto each = [&](auto f) {
#pragma unroll 1
    for (int i = lane; i < vecs; i += 32) {
      float v[kVec];
      Vec<T>::get(mine[i], v);
      f(v, first + i * kVec);
    }
  };

  const bool cut_k = k > 0 && k < n, cut_p = p < 1.f;
  float thr = top_inf ? INFINITY : -INFINITY;  // kept: logits above it ...
  uint64_t take = 0;                           // ... and this many of those equal to it
  bool summed = false;                         // the kept weights are already in part_w, part_eq

  if ((cut_k || cut_p) && !top_inf) {
    const int bins = min(kSampleBins, kSampleThreads * C), share = bins / C;  // a CTA's share: a bin a thread
    const float width = kSampleDeep / bins, per_d256 = 256.f / width;
    bool packed = cut_p;  // a bin's word: tokens << 20 | their 256ths; or, where that may not fit, tokens
    uint64_t weight = 0;  // of all tokens, then of the prefix
    // the cluster's histograms added up, each CTA a share of the bins, and the sums before this thread's; `vc`
    // (known to warp 0) is added up over the CTAs as the total weight
    auto sum_bins = [&](auto bin_sums, uint64_t vc) {
      BinSums s;
      s.n = 0;
      s.w = 0;
      if (tid < share) bin_sums(rank * share + tid, s.n, s.w);
      const uint64_t ci = warp_scan64(s.n, lane), wi = warp_scan64(s.w, lane);
      if (lane == 31) {
        sh.warp_a[warp] = ci;
        sh.warp_b[warp] = wi;
      }
      __syncthreads();
      s.count = ci - s.n;
      s.weight = wi - s.w;
      uint64_t ct = lane < kSampleWarps ? sh.warp_a[lane] : 0, wt = lane < kSampleWarps ? sh.warp_b[lane] : 0;
      s.count += warp_sum64(lane < warp ? ct : 0);
      s.weight += warp_sum64(lane < warp ? wt : 0);
      ct = warp_sum64(ct);
      wt = warp_sum64(wt);
      const Trio64* r = exchange(ct | (uint64_t)sh.counted << 32, wt, vc);
      s.total_count = s.total_weight = 0;
      uint64_t counted = 0;
      for (int q = 0; q < C; ++q) {
        if (q < rank) {
          s.count += (uint32_t)r[q].a;
          s.weight += r[q].b;
        }
        s.total_count += (uint32_t)r[q].a;
        s.total_weight += r[q].c;
        counted += r[q].a >> 32;
      }
      s.complete = s.total_count == counted;
      return s;
    };
    // the bins in which the prefix of `want` tokens (of weight `want`) ends, given what lies above all bins. The
    // weights may be lower bounds: what they are of is then at most w (1 + eps) + 3 per token.
    auto find = [&](const BinSums& s, uint64_t want, bool by_weight, uint64_t count0, uint64_t weight0, float eps) {
      const uint64_t c = count0 + s.count, w = weight0 + s.weight;
      auto most = [&](uint64_t x, uint64_t n) {
        return eps > 0.f ? x + (uint64_t)((double)(int64_t)x * eps) + 3 * n : x;
      };
      const uint64_t low = by_weight ? w : c, low_end = by_weight ? w + s.w : c + s.n;
      const uint64_t top = by_weight ? most(w, c) : c, top_end = by_weight ? most(w + s.w, c + s.n) : c + s.n;
      const int bin = rank * share + tid;
      if (top < want && want <= top_end)
        for (int q = 0; q < C; ++q) {
          Bracket* const to = cluster.map_shared_rank(&sh.found, q);
          to->count = c;
          to->weight = w;
          to->bin = bin;
        }
      if ((low < want && want <= low_end) || (bin == bins - 1 && tid < share && low_end < want))
        for (int q = 0; q < C; ++q) {
          *cluster.map_shared_rank(&sh.found_last, q) = bin;
          *cluster.map_shared_rank(&sh.found_after, q) = c + s.n;
        }
      cluster.sync();
      Bracket br = sh.found;
      br.last = sh.found_last;
      br.n = (int)(sh.found_after - br.count);
      return br;
    };
    // cuts the prefix: thr, take; returns the prefix's weight (if there is top-p)
    auto cut = [&](const BinSums& s0, uint64_t want, bool by_weight) {
      // what bin_sums below leaves open, relative to a weight of at least 1 - width
      const float eps = packed ? 1.1f * (width * width / 8 + width / 256) + 4e-5f : 1.05f * width + 4e-5f;
      Bracket br = find(s0, want, by_weight, 0, 0, eps);
      const uint32_t from_q = (uint32_t)br.bin << 8, end_q = (uint32_t)(br.last + 1) << 8;
      // logits below this are below the bracket, by more than the roundings of d (2^-20 of it and of l, m); a
      // temperature that has no such bound in fp32 gets none
      const float l_low = temp < 1e30f && br.last < bins - 1
                              ? m - (br.last + 1) * width * temp - 1e-5f * (fabsf(m) + kSampleDeep * temp)
                              : -INFINITY;
      // the weight of this CTA's tokens above the bracket, and f(logits, index, mask) of the bracket's
      auto pass = [&](auto f) {
        uint32_t hi = 0, lo = 0;
        each([&](const float* v, int i) {
          float most = v[0];
#pragma unroll
          for (int j = 1; j < kVec; ++j) most = fmaxf(most, v[j]);
          if (!(most >= l_low)) return;
          unsigned in = 0;
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const float d = logit_depth(v[j], m, inv_t);
            const uint32_t at = depth_place(d, per_d256);
            in |= (unsigned)(at >= from_q && at < end_q) << j;
            uint32_t h, l;
            weight_halves(expf(at < from_q ? d : -100.f), h, l);
            hi += h - kHalfBits;
            lo += l - kHalfBits;
          }
          if (in) f(v, i, in);
        });
        const uint64_t w = warp_sum64(((uint64_t)hi << 20) + lo);
        if (lane == 0) {
          atomicAdd(&sh.above[by_weight], (unsigned long long)w);
          sh.part_w[warp] = w;
          sh.part_eq[warp] = 0;
        }
      };
      uint32_t k_lo = 0, k_hi = 0;
      const bool by_key = br.n > kSampleList;  // too many to sort: cut by key first
      if (by_key) {
        if (tid == 0) {
          sh.key_min = 0xffffffffu;
          sh.key_max = 0;
        }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        pass([&](const float* v, int, unsigned in) {
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (in >> j & 1u) {
              lo = min(lo, logit_key(v[j]));
              hi = max(hi, logit_key(v[j]));
            }
        });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) {
          atomicMin(&sh.key_min, lo);
          atomicMax(&sh.key_max, hi);
        }
        __syncthreads();
        const Trio64* r = exchange(sh.key_min, sh.key_max, sh.above[by_weight]);
        k_lo = 0xffffffffu;
        br.weight = 0;
        for (int q = 0; q < C; ++q) {
          k_lo = min(k_lo, (uint32_t)r[q].a);
          k_hi = max(k_hi, (uint32_t)r[q].b);
          br.weight += r[q].c;
        }
      }
      // f(logit, its key, index) of the tokens from k_lo to k_hi
      auto each_key = [&](auto f) {
        each([&](const float* v, int i) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const uint32_t key = logit_key(v[j]);
            if (key >= k_lo && key <= k_hi) f(v[j], key, i + j);
          }
        });
      };
      // a round leaves a 512th or less of the keys' range: 32 bits take four; equal logits are arithmetic
      for (int round = 0; round < 4 && br.n > kSampleList && k_lo != k_hi; ++round) {
        int shift = 0;
        while (((k_hi - k_lo) >> shift) >= (uint32_t)bins) ++shift;
        for (int i = tid; i < bins; i += kSampleThreads) {
          sh.cnt[i] = 0;
          sh.weight[i] = 0;
        }
        __syncthreads();
        each_key([&](float l, uint32_t key, int) {
          const uint32_t bin = (k_hi - key) >> shift;
          atomicAdd(&sh.cnt[bin], 1u);
          if (cut_p) {  // 64 bits by two words, with the carry of the lower one
            uint32_t* const words = reinterpret_cast<uint32_t*>(&sh.weight[bin]);
            const uint64_t w = depth_weight(logit_depth(l, m, inv_t));
            const uint32_t old = atomicAdd(words, (uint32_t)w);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + (uint32_t)w < old ? 1u : 0u);
            if (hi) atomicAdd(words + 1, hi);
          }
        });
        cluster.sync();
        const BinSums s = sum_bins(
            [&](int bin, uint32_t& n, uint64_t& w) {
              for (int q = 0; q < C; ++q) {
                n += *cluster.map_shared_rank(&sh.cnt[bin], q);
                w += *cluster.map_shared_rank(&sh.weight[bin], q);
              }
            },
            0);
        br = find(s, want, by_weight, br.count, br.weight, 0.f);
        k_hi -= (uint32_t)br.bin << shift;
        k_lo = max(k_lo, k_hi - ((1u << shift) - 1u));
      }
      if (br.n > kSampleList) {
        thr = key_logit(k_lo);
        const uint64_t w1 = depth_weight(logit_depth(thr, m, inv_t));
        take = by_weight ? (want - br.weight + w1 - 1) / w1 : want - br.count;
        summed = false;
        return br.weight + take * w1;
      }
      // the bracket's tokens into this CTA's list, in any order; then every CTA takes all of them
      int* const list_n = &sh.list_n[by_weight];
      if (by_key)
        each_key([&](float, uint32_t key, int i) { sh.list[atomicAdd(list_n, 1)] = ((uint64_t)key << 32) | (uint32_t)~i; });
      else
        pass([&](const float* v, int i, unsigned in) {
          int to = atomicAdd(list_n, __popc(in));
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (in >> j & 1u) sh.list[to++] = ((uint64_t)logit_key(v[j]) << 32) | (uint32_t)~(i + j);
        });
      cluster.sync();
      uint64_t me[kSampleOwn], w[kSampleOwn] = {};
      auto own = [](const uint64_t* v, int o) {
        uint64_t x = v[0];
#pragma unroll
        for (int i = 1; i < kSampleOwn; ++i) x = i == o ? v[i] : x;
        return x;
      };
      {
        const int in_q = lane < C ? *cluster.map_shared_rank(list_n, lane) : 0;
        if (!by_key) br.weight = warp_sum64(lane < C ? *cluster.map_shared_rank(&sh.above[by_weight], lane) : 0);
#pragma unroll
        for (int o = 0; o < kSampleOwn; ++o) {
          const int t = tid + o * kSampleThreads;
          int q = -1, at = 0;
          for (int c = 0, before = 0; c < C; ++c) {
            const int in_c = __shfl_sync(0xffffffffu, in_q, c);
            if (t >= before && t < before + in_c) {
              q = c;
              at = t - before;
            }
            before += in_c;
          }
          me[o] = q >= 0 ? *cluster.map_shared_rank(&sh.list[at], q) : 0;
        }
      }
      // sorted downwards within the warp; a token's place and the weight up to it are then sums over the lots of
      // 32 of what is above it in each, found by halving
#pragma unroll 1
      for (int o = 0; o < kSampleOwn && o * kSampleThreads < br.n; ++o) {
        uint64_t x = own(me, o);
#pragma unroll
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll
          for (int step = size / 2; step > 0; step /= 2) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, x, step);
            const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
            x = (x > other) == keep_max ? x : other;
          }
        const uint64_t wx = x ? depth_weight(logit_depth(key_logit((uint32_t)(x >> 32)), m, inv_t)) : 0;
        sh.sorted[tid + o * kSampleThreads] = x;
        sh.sums[tid + o * kSampleThreads] = warp_scan64(wx, lane);
#pragma unroll
        for (int i = 0; i < kSampleOwn; ++i)
          if (i == o) {
            me[i] = x;
            w[i] = wx;
          }
      }
      __syncthreads();
#pragma unroll 1
      for (int o = 0; o < kSampleOwn && o * kSampleThreads < br.n; ++o) {
        const uint64_t x = own(me, o), wx = own(w, o);
        if (!x) continue;
        int place = 0;
        uint64_t upto = br.weight;
#pragma unroll 2
        for (int at = 0; at < br.n; at += 32) {
          int above = 0;  // of these 32 tokens, those not below this one
#pragma unroll
          for (int half = 16; half > 0; half /= 2) above += sh.sorted[at + above + half - 1] >= x ? half : 0;
          above += sh.sorted[at + above] >= x;
          place += above;
          upto += above ? sh.sums[at + above - 1] : 0;
        }
        if (by_weight ? upto - wx < want && want <= upto : br.count + place == want) {
          sh.cut_weight = upto;
          sh.cut = x;
        }
      }
      __syncthreads();
      const uint64_t last = sh.cut;
      thr = key_logit((uint32_t)(last >> 32));
      take = 0;
#pragma unroll
      for (int o = 0; o < kSampleOwn; ++o) {
        const bool tie = (me[o] >> 32) == (last >> 32);
        take += __syncthreads_count(tie && me[o] >= last);
        // what is kept of these, and the ties, to the sums of the warps whose tokens they are
        const int of_warp = (int)((~(uint32_t)me[o] - rank * kSampleWarps * a.per_warp) / (uint32_t)a.per_warp);
        if (!by_key && me[o] && of_warp >= 0 && of_warp < kSampleWarps) {
          if (tie)
            atomicAdd(&sh.part_eq[of_warp], 1u);
          else if (me[o] > last)
            atomicAdd(&sh.part_w[of_warp], (unsigned long long)w[o]);
        }
      }
      summed = !by_key;
      return sh.cut_weight;
    };

    // ---- 2: the histogram over steps of d, and the exact weight of all. One addition to shared memory per logit
    // (they fall into banks at random, 3.5 to one at the worst of 32): the number of a bin's tokens and the sum of
    // their 256ths of a step bound its weight to 2^-13. What is too deep to weigh anything is not counted.
    auto count = [&](bool weigh) {
      for (int i = tid; i < bins; i += kSampleThreads) sh.cnt[i] = 0;
      __syncthreads();
      uint32_t hi = 0, lo = 0, n_in = 0;
      const uint32_t end_q = (uint32_t)bins << 8;
      each([&](const float* v, int) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float d = logit_depth(v[j], m, inv_t);
          const uint32_t at = depth_place(d, per_d256);
          if (at < end_q) atomicAdd(&sh.cnt[at >> 8], packed ? (1u << 20) + (at & 255u) : 1u);
          n_in += at < end_q;
          if (weigh) {
            uint32_t h, l;
            weight_halves(expf(fmaxf(d, -100.f)), h, l);
            hi += h - kHalfBits;
            lo += l - kHalfBits;
          }
        }
      });
      const uint64_t w = warp_sum64(((uint64_t)hi << 20) + lo);
      n_in = __reduce_add_sync(0xffffffffu, n_in);
      if (lane == 0) {
        sh.part_w[warp] = w;
        atomicAdd(&sh.counted, n_in);
      }
      cluster.sync();
    };
    auto bin_sums = [&](int bin, uint32_t& n, uint64_t& w) {
      uint32_t f = 0;
      for (int q = 0; q < C; ++q) {
        const uint32_t word = *cluster.map_shared_rank(&sh.cnt[bin], q);
        n += packed ? word >> 20 : word;
        f += packed ? word & 0xfffffu : 0u;
      }
      // Lower bound of the weight: e^-x lies under its chord over the step, by width^2 / 8 at most, and a
      // place is a 256th deeper at most; 1e-5 for the roundings, and a weight is rounded by 1/2 itself.
      const float top = expf(-bin * width) * (kSampleOne * (1.f - 1e-5f)), slope = 1.f - expf(-width);
      const float part = packed ? n - (f + n) * (slope / 256) - n * (width * width / 8) : n * (1.f - slope);
      w = cut_p && n ? (uint64_t)fmaxf(top * part - n, 0.f) : 0;
    };
    auto all_weights = [&]() { return warp_sum64(warp == 0 && lane < kSampleWarps ? sh.part_w[lane] : 0); };
    count(cut_p && !cut_k);  // (top-k gives the prefix's weight itself)
    BinSums s = sum_bins(bin_sums, all_weights());
    // more than 4095 tokens of a bin in a CTA leave the word's upper 12 bits; and a top-k that reaches the tokens
    // that are not counted cuts nothing
    const bool whole = cut_p && cut_k && (uint64_t)k >= s.total_count;
    if ((packed && !s.complete) || whole) {
      packed = packed && s.complete;
      if (tid == 0) sh.counted = 0;  // (count() has a barrier before it adds to it)
      count(cut_p);
      s = sum_bins(bin_sums, all_weights());
    }
    // ---- 3: the cuts. A prefix that would reach the tokens that are not counted needs none.
    weight = s.total_weight;
    if (cut_k && (uint64_t)k < s.total_count) weight = cut(s, (uint64_t)k, false);
    if (cut_p) {
      const double want = ceil((double)p * (double)(int64_t)weight);
      cut(s, want >= 1. ? (uint64_t)want : 1u, true);
    }
  }

  // ---- 4: the kept weights, ties counted apart (they all weigh the same)
  const float floor_d = mp > 0.f ? logf(fminf(mp, 1.f)) : -INFINITY;
  const bool tied = top_inf || (thr > -INFINITY && logit_depth(thr, m, inv_t) >= floor_d);
  const uint64_t w1 = top_inf ? (uint64_t)1 << 40 : tied ? depth_weight(logit_depth(thr, m, inv_t)) : 0;
  auto taken = [&](uint64_t before, uint64_t here) {  // the weight of `here` ties that come after `before` others
    return before >= take ? (uint64_t)0 : min(here, take - before) * w1;
  };
  // logits below it are not kept: of the floor, by more than the roundings of d (a NaN bound leaves the threshold)
  const float low = temp < 1e30f ? fmaxf(thr, m + floor_d * temp - 1e-5f * (fabsf(m) - floor_d * temp)) : thr;
  // d of a kept logit above the threshold; of others one whose weight is 0 (of NaN too)
  auto kept = [&](float l) {
    const float d = logit_depth(l, m, inv_t);
    return l > thr && d >= floor_d ? d : -100.f;
  };
  // adds a vector's kept weights in halves, and its ties
  auto add_kept = [&](const float* v, uint32_t& hi, uint32_t& lo, uint32_t& eq) {
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kVec; ++j) most = fmaxf(most, v[j]);
    if (!(most >= low)) return;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      uint32_t h, l;
      weight_halves(expf(kept(v[j])), h, l);
      hi += h - kHalfBits;
      lo += l - kHalfBits;
      eq += v[j] == thr;
    }
  };
  if (summed && tied) {  // (a floor below the threshold cuts nothing)
    __syncthreads();
    if (tid < kSampleWarps) {
      sh.warp_a[tid] = sh.part_w[tid];
      sh.warp_b[tid] = tied ? sh.part_eq[tid] : 0;
    }
  } else {
    // halves of up to 2^20 a logit: 32 bits hold the sums of a lane's 16 vectors (at most 512 a warp, see the
    // cluster's choice), 2^27, and 64 the warp's
    uint32_t hi = 0, lo = 0, eq = 0;
    if (thr == -INFINITY && floor_d == -INFINITY)  // every token that is not masked
      each([&](const float* v, int) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          // the bound turns NaN and -inf into weight 0, as it is for all that deep
          uint32_t h, l;
          weight_halves(expf(fmaxf(logit_depth(v[j], m, inv_t), -100.f)), h, l);
          hi += h - kHalfBits;
          lo += l - kHalfBits;
        }
      });
    else
      each([&](const float* v, int) { add_kept(v, hi, lo, eq); });
    const uint64_t w = warp_sum64(((uint64_t)hi << 20) + lo);
    eq = tied ? __reduce_add_sync(0xffffffffu, eq) : 0;
    if (lane == 0) {
      sh.warp_a[warp] = w;
      sh.warp_b[warp] = eq;
    }
  }
  __syncthreads();
  uint64_t sum_w = 0, sum_eq = 0;
  if (warp == 0) {
    sum_w = warp_sum64(lane < kSampleWarps ? sh.warp_a[lane] : 0);
    sum_eq = __reduce_add_sync(0xffffffffu, lane < kSampleWarps ? (uint32_t)sh.warp_b[lane] : 0u);
  }
  const Trio64* r = exchange(sum_w, sum_eq, 0);
  if (top_inf) {
    for (int c = 0; c < C; ++c) take += r[c].b;
    if (cut_k) take = min(take, (uint64_t)k);
    if (cut_p) {
      const double want = ceil((double)p * (double)(int64_t)(take * w1));
      take = want > (double)w1 ? ((uint64_t)want + w1 - 1) / w1 : 1;
    }
  }
  uint64_t total = 0, seen = 0, run = 0, seen0 = 0, here = 0;  // run, seen0: before this CTA; here: its weight
  for (int c = 0; c < C; ++c) {
    const uint64_t w = r[c].a + (tied ? taken(seen, r[c].b) : 0);
    if (c == rank) {
      run = total;
      seen0 = seen;
      here = w;
    }
    total += w;
    seen += r[c].b;
  }
  const double at_d = floor((double)u * (double)(int64_t)total);
  uint64_t at = at_d >= 1. ? (uint64_t)at_d : 0;  // NaN and negative numbers count as 0
  if (at >= total) at = total - 1;
  if (run <= at && at < run + here) {  // this CTA has it
    // the warp's part in which the running sum passes `at`: lane q looks at part q
    uint64_t eq = lane < kSampleWarps ? sh.warp_b[lane] : 0, w = lane < kSampleWarps ? sh.warp_a[lane] : 0;
    uint64_t eq_before = seen0 + warp_scan64(eq, lane) - eq;
    if (tied) w += taken(eq_before, eq);
    uint64_t incl = run + warp_scan64(w, lane);
    const int q = __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1;
    run = __shfl_sync(0xffffffffu, incl - w, q);
    seen = __shfl_sync(0xffffffffu, eq_before, q);
    const uint4* const from = part + q * vecs;
    const int base = (rank * kSampleWarps + q) * a.per_warp;
    // its vectors, 32 to a warp (at most 512), then the warp in whose vectors the sum passes, its lane, and that
    // lane's logits
    const int i = warp * 32 + lane;
    uint32_t hi = 0, lo = 0, el = 0;
    if (i < vecs) {
      float v[kVec];
      Vec<T>::get(from[i], v);
      add_kept(v, hi, lo, el);
    }
    if (!tied) el = 0;
    const uint64_t wl = ((uint64_t)hi << 20) + lo;
    const uint32_t el_all = __reduce_add_sync(0xffffffffu, el);
    {
      const uint64_t sum = warp_sum64(wl);
      __syncthreads();  // all have read the sums of the parts
      if (lane == 0) {
        sh.warp_a[warp] = sum;
        sh.warp_b[warp] = el_all;
      }
      __syncthreads();
      eq = lane < kSampleWarps ? sh.warp_b[lane] : 0;
      w = lane < kSampleWarps ? sh.warp_a[lane] : 0;
      eq_before = seen + warp_scan64(eq, lane) - eq;
      if (tied) w += taken(eq_before, eq);
      incl = run + warp_scan64(w, lane);
    }
    if (warp == __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1) {
      run = __shfl_sync(0xffffffffu, incl - w, warp);
      seen = __shfl_sync(0xffffffffu, eq_before, warp);
      uint64_t e_before = seen;
      if (el_all) e_before += warp_scan64(el, lane) - el;
      const uint64_t wt = wl + (el_all ? taken(e_before, el) : 0), upto = run + warp_scan64(wt, lane);
      const int at_lane = __ffs(__ballot_sync(0xffffffffu, upto > at)) - 1;
      run = __shfl_sync(0xffffffffu, upto - wt, at_lane);
      seen = __shfl_sync(0xffffffffu, e_before, at_lane);
      const int iv = warp * 32 + at_lane;  // the vector; lane j takes its logit j
      const float l = lane < kVec ? Vec<T>::one(reinterpret_cast<const T*>(from + iv)[lane]) : -INFINITY;
      const bool tie = tied && l == thr;
      const unsigned ties = __ballot_sync(0xffffffffu, tie);
      uint32_t wh, wo;
      weight_halves(expf(kept(l)), wh, wo);
      const uint64_t wj = tie ? taken(seen + __popc(ties & ((1u << lane) - 1u)), 1)
                              : ((uint64_t)(wh - kHalfBits) << 20) + (wo - kHalfBits);
      const unsigned past = __ballot_sync(0xffffffffu, run + warp_scan64(wj, lane) > at);
      if (lane == __ffs(past) - 1) {
        a.tok[row] = base + iv * kVec + lane;
        if (a.logprob) a.logprob[row] = (top_inf ? 0.f : logit_depth(l, m, inv_t)) - logf((float)(int64_t)total * (1.f / kSampleOne));
      }
    }
  }
}

}  // namespace qd

using namespace qd;

extern "C" int qd_sample(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         const float* u, int64_t* tok, float* logprob, int pdl, cudaStream_t stream) {
  if (dtype != QD_BF16 && dtype != QD_FP16 && dtype != QD_FP32)
    return set_error(QD_ERR_UNSUPPORTED, "sample: element type %d", dtype);
  if (rows > 0 && (!logits || !u || !tok)) return set_error(QD_ERR_ARG, "sample: null logits, u or tok");
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || ld < vocab)
    return set_error(QD_ERR_ARG, "sample: %lld rows of %lld logits, stride %lld", (long long)rows, (long long)vocab,
                     (long long)ld);
  if (vocab > kSampleMaxVocab)
    return set_error(QD_ERR_UNSUPPORTED, "sample: vocabulary of %lld (at most %lld)", (long long)vocab,
                     (long long)kSampleMaxVocab);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == QD_FP32 ? 4 : 2))
    return set_error(QD_ERR_ARG, "sample: misaligned logits");
  if (rows == 0) return QD_OK;
  // The cluster: the fewest CTAs of which two fit an SM (so that one's loads and barriers hide behind the
  // other's arithmetic) and which fill the SMs, but at most one for 4096 logits. Measured on rows of 151,936 BF16
  // logits, with clusters of 4 / 8: 8 rows with top-p 29 / 22 us, 64 rows 50 / 65 us, 256 unfiltered 65 / 88 us.
  // However the choice ends, a warp has at most 512 vectors of 16 bytes, one per thread of its CTA, which the last
  // walk and the sums of halves rely on.
  constexpr int kFit = 110 * 1024, kFew = 8192, kMost = 16 * kSampleThreads;  // kMost: bytes of a warp's logits
  static_assert(kSampleMaxVocab / (kSampleMaxCluster * kSampleWarps) * 4 <= kMost, "the largest cluster");
  static_assert(kFew / kSampleWarps * 4 <= kMost, "few logits a CTA");
  static_assert((kFit - kSampleShared) / kSampleWarps + 8 * 4 <= kMost, "two CTAs an SM");
  const int size = dtype == QD_FP32 ? 4 : 2;
  int cluster = 1;
  while (cluster < kSampleMaxCluster && vocab >= (int64_t)kFew * cluster &&
         (rows * cluster < host_sm_count() || kSampleShared + vocab * size / cluster > kFit))
    cluster *= 2;
  SampleArgs a = {logits, ld, vocab, temperature, top_k, top_p, min_p, u, tok, logprob, 0, 0};
  const int parts = cluster * kSampleWarps;
  a.per_warp = (int)((vocab + parts - 1) / parts + 7) / 8 * 8;
  a.wide = aligned16(logits) && ld * size % 16 == 0;
  const int smem = kSampleShared + a.per_warp * kSampleWarps * size;
  const void* fn = dtype == QD_BF16   ? (const void*)sample_kernel<__nv_bfloat16>
                   : dtype == QD_FP16 ? (const void*)sample_kernel<__half>
                                      : (const void*)sample_kernel<float>;
  const int rc = set_max_dynamic_smem(fn, smem);
  if (rc != QD_OK) return rc;
  if (rows * cluster > INT32_MAX) return set_error(QD_ERR_UNSUPPORTED, "sample: %lld rows", (long long)rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  void* args[1] = {&a};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
  if (e != cudaSuccess) return set_error(QD_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return QD_OK;
}
