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
//   2  (top-k or top-p) a histogram of number and weight over up to 2048 equal steps of d down to the weights
//      that round to 0, summed over the cluster by shares of bins: the bin in which the prefix ends is exact
//   3  the tokens of that bin, a few hundred, are gathered into one CTA, which sorts them and finds the last
//      one kept; a bin of more than 512 (many ties, a high temperature) is cut again, by key, first
//   4  the kept weight of every warp, the warp in which u falls, and a walk through its tokens
// Without top-k and top-p only 1 and 4 are left, and the weights are computed once. What bounds it: the
// instructions per logit (exponential, conversion, 64-bit sums; shared-memory atomics in 2) for many rows,
// the cluster barriers for few.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qd_common.cuh"
#include "qd_host.h"

namespace qd {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = kSampleThreads;     // tokens that one CTA sorts, one a thread
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
// the step of d in which a d of -kSampleDeep to 0 lies (by an addition of 2^23 too: a conversion to int would
// take the exponentials' pipe)
__device__ __forceinline__ int depth_bin(float d, float per_d, int bins) {
  return min((int)(__float_as_uint(__fmaf_rd(-d, per_d, 8388608.0f)) - kHalfBits), bins - 1);
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

struct Pair64 {
  uint64_t a, b;
};
// Where a prefix ends: in one of the bins, `n` tokens, after `count` tokens of `weight` in the bins before it.
struct Bracket {
  uint64_t count, weight;
  int bin, n;
};
// The bin of which this thread has the cluster's sums (none: 0), and the sums before it.
struct BinSums {
  uint32_t n;
  uint64_t w, count, weight, total_count, total_weight;
};

struct SampleShared {
  uint64_t weight[kSampleBins];  // this CTA's histogram; then the lists of the bin that is cut
  uint32_t cnt[kSampleBins];
  Pair64 xch[2][kSampleMaxCluster];                             // a value of every CTA, two exchanges in turn
  uint64_t warp_a[kSampleWarps], warp_b[kSampleWarps];
  Bracket found;
  Pair64 cut;  // weight of the prefix, its last token
  int list_n[2];  // tokens of this CTA in that bin, for the cut by top-k and by top-p
  uint32_t key_min, key_max;
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
    sh.key_min = 0xffffffffu;
    sh.key_max = 0;
  }
  __syncthreads();
  int turn = 0;
  // (va, vb), known to warp 0, to every CTA of the cluster; all threads pass the barrier
  auto exchange = [&](uint64_t va, uint64_t vb) {
    if (tid < C) *cluster.map_shared_rank(&sh.xch[turn][rank], tid) = Pair64{va, vb};
    cluster.sync();
    const Pair64* r = sh.xch[turn];
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
    const Pair64* r = exchange(best, 0);
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

  if ((cut_k || cut_p) && !top_inf) {
    const int bins = min(kSampleBins, kSampleThreads * C), share = bins / C;  // a CTA's share: a bin a thread
    const float per_d = bins / kSampleDeep;
    // The tokens (number and weight) by bins: bin_of(logit, d), -1 for none, over the vectors that `in_part` is
    // true of. The weights' halves, with the bits above them, are added up apart: additions that return nothing,
    // and up to 4095 tokens of a bin leave 32 bits enough. Where a bin has more, 64-bit sums with a carry.
    auto histogram = [&](auto in_part, auto bin_of) {
      uint32_t* const words = reinterpret_cast<uint32_t*>(sh.weight);
      for (int i = tid; i < bins; i += kSampleThreads) {
        sh.cnt[i] = 0;
        sh.weight[i] = 0;
      }
      __syncthreads();
      each([&](const float* v, int) {
        if (!in_part(v)) return;
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float d = logit_depth(v[j], m, inv_t);
          const int bin = bin_of(v[j], d);
          if (bin >= 0) atomicAdd(&sh.cnt[bin], 1u);
          if (cut_p && bin >= 0) {  // (without top-p numbers are enough)
            uint32_t hi, lo;
            weight_halves(expf(d), hi, lo);
            atomicAdd(&words[2 * bin], lo);
            atomicAdd(&words[2 * bin + 1], hi);
          }
        }
      });
      __syncthreads();
      if (!cut_p) return;
      bool many = false;
      for (int i = tid; i < bins; i += kSampleThreads) {
        const uint32_t c = sh.cnt[i], off = c * kHalfBits;
        many |= c > 4095;
        sh.weight[i] = ((uint64_t)(words[2 * i + 1] - off) << 20) + (words[2 * i] - off);
      }
      if (!__syncthreads_or(many)) return;
      for (int i = tid; i < bins; i += kSampleThreads) sh.weight[i] = 0;
      __syncthreads();
      each([&](const float* v, int) {
        if (!in_part(v)) return;
#pragma unroll 1
        for (int j = 0; j < kVec; ++j) {
          const float d = logit_depth(v[j], m, inv_t);
          const int bin = bin_of(v[j], d);
          if (bin < 0) continue;
          const uint64_t w = depth_weight(d);
          const uint32_t old = atomicAdd(&words[2 * bin], (uint32_t)w);
          const uint32_t hi = (uint32_t)(w >> 32) + (old + (uint32_t)w < old ? 1u : 0u);
          if (hi) atomicAdd(&words[2 * bin + 1], hi);
        }
      });
    };
    // the cluster's histograms added up, each CTA a share of the bins, and the sums before this thread's
    auto sum_bins = [&]() {
      cluster.sync();
      BinSums s;
      uint64_t c = 0, w = 0;
      if (tid < share) {
        const int b = rank * share + tid;
#pragma unroll
        for (int q = 0; q < kSampleMaxCluster; ++q)
          if (q < C) c += *cluster.map_shared_rank(&sh.cnt[b], q);
        if (cut_p) {
#pragma unroll
          for (int q = 0; q < kSampleMaxCluster; ++q)
            if (q < C) w += *cluster.map_shared_rank(&sh.weight[b], q);
        }
      }
      s.n = (uint32_t)c;
      s.w = w;
      const uint64_t ci = warp_scan64(c, lane), wi = warp_scan64(w, lane);
      if (lane == 31) {
        sh.warp_a[warp] = ci;
        sh.warp_b[warp] = wi;
      }
      __syncthreads();
      s.count = ci - c;
      s.weight = wi - w;
      uint64_t ct = lane < kSampleWarps ? sh.warp_a[lane] : 0, wt = lane < kSampleWarps ? sh.warp_b[lane] : 0;
      s.count += warp_sum64(lane < warp ? ct : 0);
      s.weight += warp_sum64(lane < warp ? wt : 0);
      ct = warp_sum64(ct);
      wt = warp_sum64(wt);
      const Pair64* r = exchange(ct, wt);
      s.total_count = s.total_weight = 0;
      for (int q = 0; q < C; ++q) {
        if (q < rank) {
          s.count += r[q].a;
          s.weight += r[q].b;
        }
        s.total_count += r[q].a;
        s.total_weight += r[q].b;
      }
      return s;
    };
    // the bin in which the prefix of `want` tokens (of weight `want`) ends, given what lies above all bins
    auto find = [&](const BinSums& s, uint64_t want, bool by_weight, uint64_t count0, uint64_t weight0) {
      const uint64_t c = count0 + s.count, w = weight0 + s.weight;
      const uint64_t before = by_weight ? w : c, here = by_weight ? s.w : s.n;
      if (before < want && want <= before + here)
        for (int q = 0; q < C; ++q)
          *cluster.map_shared_rank(&sh.found, q) = Bracket{c, w, rank * share + tid, (int)s.n};
      cluster.sync();
      return sh.found;
    };
    // cuts the prefix within a step of d: thr, take; returns the prefix's weight
    auto cut = [&](const BinSums& s0, uint64_t want, bool by_weight) {
      Bracket br = find(s0, want, by_weight, 0, 0);
      const int step = br.bin;
      uint32_t k_lo = 0, k_hi = 0;  // by key, once the bracket is narrower than the step
      // logits of the step lie in between these, by more than the roundings of d (2^-20 of it and of l, m)
      // (a temperature that has no such bounds in fp32 gets none)
      const bool bounded = temp < 1e30f;
      const float slop = 1e-5f * (fabsf(m) + kSampleDeep * temp), width = kSampleDeep / bins;
      const float l_top = bounded ? m - step * width * temp + slop : INFINITY;
      const float l_low = bounded && step < bins - 1 ? m - (step + 1) * width * temp - slop : -INFINITY;
      auto may_be = [&](const float* v) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < kVec; ++j) any |= v[j] >= l_low && v[j] <= l_top;
        return any;
      };
      auto inside = [&](float l) {
        const float d = logit_depth(l, m, inv_t);
        const uint32_t key = logit_key(l);
        return l > -INFINITY && (k_hi ? key >= k_lo && key <= k_hi : d >= -kSampleDeep && depth_bin(d, per_d, bins) == step);
      };
      // a round leaves a 512th or less of the keys' range: 32 bits take four
      for (int round = 0; round < 4 && br.n > kSampleList; ++round) {
        if (!k_hi) {  // the keys in this step
          if (tid == 0) {
            sh.key_min = 0xffffffffu;
            sh.key_max = 0;
          }
          __syncthreads();
          uint32_t lo = 0xffffffffu, hi = 0;
          each([&](const float* v, int) {
            if (!may_be(v)) return;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              const bool in = inside(v[j]);
              lo = min(lo, in ? logit_key(v[j]) : 0xffffffffu);
              hi = max(hi, in ? logit_key(v[j]) : 0u);
            }
          });
          lo = __reduce_min_sync(0xffffffffu, lo);
          hi = __reduce_max_sync(0xffffffffu, hi);
          if (lane == 0) {
            atomicMin(&sh.key_min, lo);
            atomicMax(&sh.key_max, hi);
          }
          __syncthreads();
          const Pair64* r = exchange(sh.key_min, sh.key_max);
          k_lo = 0xffffffffu;
          for (int q = 0; q < C; ++q) {
            k_lo = min(k_lo, (uint32_t)r[q].a);
            k_hi = max(k_hi, (uint32_t)r[q].b);
          }
        }
        if (k_lo == k_hi) break;  // equal logits: arithmetic
        int shift = 0;
        while (((k_hi - k_lo) >> shift) >= (uint32_t)bins) ++shift;
        histogram(may_be, [&](float l, float) { return inside(l) ? (int)((k_hi - logit_key(l)) >> shift) : -1; });
        const BinSums s = sum_bins();
        br = find(s, want, by_weight, br.count, br.weight);
        k_hi -= (uint32_t)br.bin << shift;
        k_lo = max(k_lo, k_hi - ((1u << shift) - 1u));
      }
      uint64_t weight;
      if (br.n > kSampleList) {
        thr = key_logit(k_lo);
        const uint64_t w1 = depth_weight(logit_depth(thr, m, inv_t));
        take = by_weight ? (want - br.weight + w1 - 1) / w1 : want - br.count;
        weight = br.weight + take * w1;
      } else {
        uint64_t* const list = sh.weight;  // in place of the histogram, which all have read
        uint64_t* const sorted = list + kSampleList;
        uint64_t* const sums = sorted + kSampleList;
        int* const list_n = &sh.list_n[by_weight];
        // the bracket's tokens into this CTA's list, in any order; then every CTA takes all of them, one a thread
        each([&](const float* v, int i) {
          if (!may_be(v)) return;
          unsigned in = 0;
#pragma unroll
          for (int j = 0; j < kVec; ++j) in |= (unsigned)inside(v[j]) << j;
          if (in) {
            int to = atomicAdd(list_n, __popc(in));
#pragma unroll
            for (int j = 0; j < kVec; ++j)
              if (in >> j & 1u) list[to++] = ((uint64_t)logit_key(v[j]) << 32) | (uint32_t)~(i + j);
          }
        });
        cluster.sync();
        uint64_t me = 0;
        {
          const int share = lane < C ? *cluster.map_shared_rank(list_n, lane) : 0;
          int q = -1, at = 0;
          for (int c = 0, before = 0; c < C; ++c) {
            const int in_c = __shfl_sync(0xffffffffu, share, c);
            if (tid >= before && tid < before + in_c) {
              q = c;
              at = tid - before;
            }
            before += in_c;
          }
          if (q >= 0) me = *cluster.map_shared_rank(&list[at], q);
        }
        // sorted downwards within the warp; a token's place and the weight up to it are then sums over the warps
        // of what is above it in each, found by halving
#pragma unroll
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll
          for (int step = size / 2; step > 0; step /= 2) {
            const uint64_t o = __shfl_xor_sync(0xffffffffu, me, step);
            const bool keep_max = ((lane & step) == 0) == ((lane & size) == 0);
            me = (me > o) == keep_max ? me : o;
          }
        const uint64_t w = me ? depth_weight(logit_depth(key_logit((uint32_t)(me >> 32)), m, inv_t)) : 0;
        sorted[tid] = me;
        sums[tid] = warp_scan64(w, lane);
        __syncthreads();
        int place = 0;
        uint64_t upto = br.weight;
#pragma unroll 4
        for (int at = 0; at < br.n; at += 32) {
          int above = 0;  // of this warp's tokens, those not below this one
#pragma unroll
          for (int half = 16; half > 0; half /= 2) above += sorted[at + above + half - 1] >= me ? half : 0;
          above += sorted[at + above] >= me;
          place += above;
          upto += above ? sums[at + above - 1] : 0;
        }
        if (me && (by_weight ? upto - w < want && want <= upto : br.count + place == want)) sh.cut = Pair64{upto, me};
        __syncthreads();
        const uint64_t last = sh.cut.b;
        const int ties = __syncthreads_count(me >= last && (me >> 32) == (last >> 32));
        weight = sh.cut.a;
        thr = key_logit((uint32_t)(last >> 32));
        take = ties;
      }
      return weight;
    };

    // ---- 2, 3: the histogram over steps of d, and the cuts
    // (-inf and NaN are below every step)
    histogram([](const float*) { return true; },
              [&](float, float d) { return d >= -kSampleDeep ? depth_bin(d, per_d, bins) : -1; });
    const BinSums s = sum_bins();
    uint64_t weight = s.total_weight;
    // tokens too deep to be counted weigh nothing: a prefix that would reach them needs no cut
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
    if (!(most >= thr)) return;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      uint32_t h, l;
      weight_halves(expf(kept(v[j])), h, l);
      hi += h - kHalfBits;
      lo += l - kHalfBits;
      eq += v[j] == thr;
    }
  };
  {
    // halves of up to 2^20 a logit: 32 bits hold the sums of a lane's 512 vectors (2^18 logits over 128 or
    // more warps), and of the warp in 64
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
  const Pair64* r = exchange(sum_w, sum_eq);
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
    // its vectors, 32 to a warp (vecs <= 512), then the warp in whose vectors the sum passes, its lane, and that
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
  if (!logits || !u || !tok) return set_error(QD_ERR_ARG, "sample: null logits, u or tok");
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
  // other's arithmetic) and which fill the SMs, but at most one for 4096 logits. Measured on 64 / 256 rows of
  // 151,936 BF16 logits: see the kernel.
  const int size = dtype == QD_FP32 ? 4 : 2;
  int cluster = 1;
  while (cluster < kSampleMaxCluster && vocab >= (int64_t)8192 * cluster &&
         (rows * cluster < host_sm_count() || kSampleShared + vocab * size / cluster > 110 * 1024))
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
