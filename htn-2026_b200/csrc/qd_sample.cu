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
//   2  (top-k or top-p) a histogram of number and weight over 2048 equal steps of d down to the weights that
//      round to 0, summed over the cluster by shares of bins: the bin in which the prefix ends is exact
//   3  the tokens of that bin, a few hundred, are gathered into one CTA, which finds the last one kept; a
//      bin of more than that (many ties, a high temperature) is cut again, by key, first
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
constexpr int kSampleList = 512;                // tokens that one CTA resolves by comparing each with each
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
// d = (l - m) / temperature of the definition (NaN for a NaN logit: below every bound), and the weight in
// units of 2^-40
__device__ __forceinline__ float logit_depth(float l, float m, float inv_t) {
  return l == m ? 0.f : l == -INFINITY ? l : __fmul_rn(__fsub_rn(l, m), inv_t);
}
__device__ __forceinline__ uint64_t depth_weight(float d) { return __float2ull_rn(expf(d) * kSampleOne); }
__device__ __forceinline__ int depth_bin(float d) {
  return min((int)(-d * (kSampleBins / kSampleDeep)), kSampleBins - 1);
}

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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
// The cluster's bins of which this thread has the sums: up to 4, `count` and `weight` before the first.
struct BinSums {
  uint32_t n[4];
  uint64_t w[4], count, weight, total_count, total_weight;
};

struct SampleShared {
  uint32_t cnt[kSampleBins], lo[kSampleBins], hi[kSampleBins];  // this CTA's histogram
  uint64_t list[kSampleList], list_w[kSampleList];              // gathered tokens (key, ~index), their weights
  Pair64 xch[2][kSampleMaxCluster];                             // a value of every CTA, two exchanges in turn
  uint64_t warp_a[kSampleWarps], warp_b[kSampleWarps];
  Bracket found;
  Pair64 cut;  // weight of the prefix, (threshold key, ties taken)
  int list_n;
  uint32_t key_min, key_max;
};
constexpr int kSampleShared = (sizeof(SampleShared) + 15) / 16 * 16;

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
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
  uint64_t best = 0;  // (key, ~index): the lowest index among equals
  {
    constexpr int kAhead = 4;  // vectors in flight per lane
    float top = -INFINITY;
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
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (f[j] > top) {  // this lane's indices ascend, so the first of equals stays
            top = f[j];
            best = ((uint64_t)logit_key(f[j]) << 32) | (uint32_t)~(first + i * kVec + j);
          }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) sh.warp_a[warp] = best;
  if (tid == 0) {
    sh.list_n = 0;
    sh.key_min = 0xffffffffu;
    sh.key_max = 0;
  }
  __syncthreads();
  int turn = 0;
  // (va, vb) of thread 0 to every CTA of the cluster; all threads pass the barrier
  auto exchange = [&](uint64_t va, uint64_t vb) {
    if (tid == 0)
      for (int c = 0; c < C; ++c) *cluster.map_shared_rank(&sh.xch[turn][rank], c) = Pair64{va, vb};
    cluster.sync();
    const Pair64* r = sh.xch[turn];
    turn ^= 1;
    return r;
  };
  if (tid == 0)
    for (int w = 1; w < kSampleWarps; ++w) best = sh.warp_a[w] > best ? sh.warp_a[w] : best;
  {
    const Pair64* r = exchange(best, 0);
    best = 0;
    for (int c = 0; c < C; ++c) best = r[c].a > best ? r[c].a : best;
  }
  const float temp = a.temperature ? a.temperature[row] : 1.f;
  const float m = best ? key_logit((uint32_t)(best >> 32)) : -INFINITY;
  if (m == -INFINITY || !(temp >= 1e-5f)) {
    if (rank == 0 && tid == 0) {
      a.tok[row] = m == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
      if (a.logprob) a.logprob[row] = m == -INFINITY ? m : 0.f;
    }
    cluster.sync();  // no CTA may leave while another still writes to it
    return;
  }
  // +inf logits: the others weigh nothing at any temperature
  const float inv_t = m == INFINITY ? 1.f : __fdiv_rn(1.f, temp);

  // f(logit, index) over this warp's logits
  auto each = [&](auto f) {
#pragma unroll 1
    for (int i = lane; i < vecs; i += 32) {
      float v[kVec];
      Vec<T>::get(mine[i], v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f(v[j], first + i * kVec + j);
    }
  };


  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.f;
  const bool cut_k = k > 0 && k < n, cut_p = p < 1.f;
  float thr = -INFINITY;  // kept: logits above it ...
  uint64_t take = 0;      // ... and this many of those equal to it

  if (cut_k || cut_p) {
    const int bins = kSampleBins / C, per = (bins + kSampleThreads - 1) / kSampleThreads;  // per: 1 to 4
    auto clear = [&]() {
      for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.cnt[i] = sh.lo[i] = sh.hi[i] = 0;
      __syncthreads();
    };
    auto count_in = [&](int bin, float d) {
      atomicAdd(&sh.cnt[bin], 1u);
      if (!cut_p) return;  // numbers are enough
      const uint64_t w = depth_weight(d);
      const uint32_t w_lo = (uint32_t)w, old = atomicAdd(&sh.lo[bin], w_lo);
      const uint32_t w_hi = (uint32_t)(w >> 32) + (old + w_lo < old ? 1u : 0u);  // with the carry
      if (w_hi) atomicAdd(&sh.hi[bin], w_hi);
    };
    // the cluster's histograms added up, each CTA a share of the bins, and the sums before this thread's
    auto sum_bins = [&]() {
      cluster.sync();
      BinSums s;
      uint64_t c = 0, w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s.n[j] = 0;
        s.w[j] = 0;
        const int b = rank * bins + tid * per + j;
        if (j < per && tid * per + j < bins)
          for (int q = 0; q < C; ++q) {
            s.n[j] += *cluster.map_shared_rank(&sh.cnt[b], q);
            s.w[j] += *cluster.map_shared_rank(&sh.lo[b], q) + ((uint64_t)*cluster.map_shared_rank(&sh.hi[b], q) << 32);
          }
        c += s.n[j];
        w += s.w[j];
      }
      const uint64_t ci = warp_scan64(c, lane), wi = warp_scan64(w, lane);
      if (lane == 31) {
        sh.warp_a[warp] = ci;
        sh.warp_b[warp] = wi;
      }
      __syncthreads();
      s.count = ci - c;
      s.weight = wi - w;
      uint64_t ct = 0, wt = 0;
      for (int q = 0; q < kSampleWarps; ++q) {
        if (q < warp) {
          s.count += sh.warp_a[q];
          s.weight += sh.warp_b[q];
        }
        ct += sh.warp_a[q];
        wt += sh.warp_b[q];
      }
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
      uint64_t c = count0 + s.count, w = weight0 + s.weight;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t before = by_weight ? w : c, here = by_weight ? s.w[j] : s.n[j];
        if (before < want && want <= before + here)
          for (int q = 0; q < C; ++q)
            *cluster.map_shared_rank(&sh.found, q) = Bracket{c, w, rank * bins + tid * per + j, (int)s.n[j]};
        c += s.n[j];
        w += s.w[j];
      }
      cluster.sync();
      return sh.found;
    };
    // cuts the prefix within a step of d: thr, take; returns the prefix's weight
    auto cut = [&](const BinSums& s0, uint64_t want, bool by_weight) {
      Bracket br = find(s0, want, by_weight, 0, 0);
      const int step = br.bin;
      uint32_t k_lo = 0, k_hi = 0;  // by key, once the bracket is narrower than the step
      auto inside = [&](float l) {
        if (!(l > -INFINITY)) return false;
        if (k_hi) return logit_key(l) >= k_lo && logit_key(l) <= k_hi;
        const float d = logit_depth(l, m, inv_t);
        return d >= -kSampleDeep && depth_bin(d) == step;
      };
      while (br.n > kSampleList) {
        if (!k_hi) {  // the keys in this step
          if (tid == 0) {
            sh.key_min = 0xffffffffu;
            sh.key_max = 0;
          }
          __syncthreads();
          uint32_t lo = 0xffffffffu, hi = 0;
          each([&](float l, int) {
            if (inside(l)) {
              lo = min(lo, logit_key(l));
              hi = max(hi, logit_key(l));
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
        while (((k_hi - k_lo) >> shift) >= (uint32_t)kSampleBins) ++shift;
        clear();
        each([&](float l, int) {
          if (inside(l)) count_in((int)((k_hi - logit_key(l)) >> shift), logit_depth(l, m, inv_t));
        });
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
        // the bracket's tokens into the first CTA, where each is compared with each
        uint64_t* const list = cluster.map_shared_rank(sh.list, 0);
        int* const list_n = cluster.map_shared_rank(&sh.list_n, 0);
        each([&](float l, int i) {
          if (inside(l)) list[atomicAdd(list_n, 1)] = ((uint64_t)logit_key(l) << 32) | (uint32_t)~i;
        });
        cluster.sync();
        if (rank == 0) {
          const uint64_t me = tid < br.n ? sh.list[tid] : 0;
          const uint64_t w = tid < br.n ? depth_weight(logit_depth(key_logit((uint32_t)(me >> 32)), m, inv_t)) : 0;
          sh.list_w[tid] = w;
          __syncthreads();
          if (tid < br.n) {
            uint64_t c_up = br.count, w_up = br.weight;
            uint32_t ties = 0;
#pragma unroll 4
            for (int j = 0; j < br.n; ++j) {
              const uint64_t o = sh.list[j];
              if (o > me) {
                ++c_up;
                w_up += sh.list_w[j];
                ties += (o >> 32) == (me >> 32);
              }
            }
            if (by_weight ? w_up < want && want <= w_up + w : c_up + 1 == want)
              for (int q = 0; q < C; ++q)
                *cluster.map_shared_rank(&sh.cut, q) = Pair64{w_up + w, (me & 0xffffffff00000000ull) | (ties + 1)};
          }
          if (tid == 0) sh.list_n = 0;
        }
        cluster.sync();
        weight = sh.cut.a;
        thr = key_logit((uint32_t)(sh.cut.b >> 32));
        take = (uint32_t)sh.cut.b;
      }
      return weight;
    };

    // ---- 2, 3: the histogram over steps of d, and the cuts
    clear();
    each([&](float l, int) {
      if (l > -INFINITY) {
        const float d = logit_depth(l, m, inv_t);
        if (d >= -kSampleDeep) count_in(depth_bin(d), d);
      }
    });
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
  const float mp = a.min_p ? a.min_p[row] : 0.f;
  const float floor_d = mp > 0.f ? logf(fminf(mp, 1.f)) : -INFINITY;
  const bool tied = thr > -INFINITY && logit_depth(thr, m, inv_t) >= floor_d;
  const uint64_t w1 = tied ? depth_weight(logit_depth(thr, m, inv_t)) : 0;
  auto kept = [&](float l) {  // the weight of a logit above the threshold, 0 of others
    if (!(l > thr)) return (uint64_t)0;
    const float d = logit_depth(l, m, inv_t);
    return d >= floor_d ? depth_weight(d) : (uint64_t)0;
  };
  auto taken = [&](uint64_t before, uint64_t here) {  // the weight of `here` ties that come after `before` others
    return before >= take ? (uint64_t)0 : min(here, take - before) * w1;
  };
  {
    uint64_t w = 0;
    uint32_t eq = 0;
    each([&](float l, int) {
      w += kept(l);
      eq += tied && l == thr;
    });
    w = warp_sum64(w);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) {
      sh.warp_a[warp] = w;
      sh.warp_b[warp] = eq;
    }
  }
  __syncthreads();
  uint64_t sum_w = 0, sum_eq = 0;
  if (tid == 0)
    for (int q = 0; q < kSampleWarps; ++q) {
      sum_w += sh.warp_a[q];
      sum_eq += sh.warp_b[q];
    }
  const Pair64* r = exchange(sum_w, sum_eq);
  uint64_t total = 0, seen = 0, run = 0, seen0 = 0, here = 0;  // run, seen0: before this CTA; here: its weight
  for (int c = 0; c < C; ++c) {
    const uint64_t w = r[c].a + taken(seen, r[c].b);
    if (c == rank) {
      run = total;
      seen0 = seen;
      here = w;
    }
    total += w;
    seen += r[c].b;
  }
  const double at_d = floor((double)a.u[row] * (double)(int64_t)total);
  uint64_t at = at_d >= 1. ? (uint64_t)at_d : 0;  // NaN and negative numbers count as 0
  if (at >= total) at = total - 1;
  if (warp == 0 && run <= at && at < run + here) {
    // the warp's part in which the running sum passes `at`: lane q looks at part q
    uint64_t eq = lane < kSampleWarps ? sh.warp_b[lane] : 0, w = lane < kSampleWarps ? sh.warp_a[lane] : 0;
    uint64_t eq_before = seen0 + warp_scan64(eq, lane) - eq;
    w += taken(eq_before, eq);
    uint64_t incl = run + warp_scan64(w, lane);
    const int q = __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1;
    run = __shfl_sync(0xffffffffu, incl - w, q);
    seen = __shfl_sync(0xffffffffu, eq_before, q);
    const uint4* const from = part + q * vecs;
    const int base = (rank * kSampleWarps + q) * a.per_warp;
    for (int i0 = 0; i0 < vecs; i0 += 32) {
      float v[kVec];
      const int i = i0 + lane;
      uint64_t wl = 0, el = 0;
      if (i < vecs) {
        Vec<T>::get(from[i], v);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          wl += kept(v[j]);
          el += tied && v[j] == thr;
        }
      }
      const uint64_t e_before = seen + warp_scan64(el, lane) - el;
      const uint64_t wt = wl + taken(e_before, el), upto = run + warp_scan64(wt, lane);
      const unsigned past = __ballot_sync(0xffffffffu, upto > at);
      if (past) {
        if (lane == __ffs(past) - 1) {
          uint64_t sum = upto - wt, e = e_before;
          bool done = false;
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const bool tie = tied && v[j] == thr;
            sum += tie ? taken(e, 1) : kept(v[j]);
            e += tie;
            if (!done && sum > at) {
              done = true;
              a.tok[row] = base + i * kVec + j;
              if (a.logprob)
                a.logprob[row] = logit_depth(v[j], m, inv_t) - logf((float)(int64_t)total * (1.f / kSampleOne));
            }
          }
        }
        break;
      }
      run = __shfl_sync(0xffffffffu, upto, 31);
      seen = __shfl_sync(0xffffffffu, e_before + el, 31);
    }
  }
  cluster.sync();  // no CTA may leave while another still reads or writes its memory
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
  // The cluster: 4096 logits a CTA are enough to pay for its barriers (151,936 logits: 8 CTAs).
  int cluster = 1;
  while (cluster < kSampleMaxCluster && vocab >= (int64_t)8192 * cluster) cluster *= 2;
  SampleArgs a = {logits, ld, vocab, temperature, top_k, top_p, min_p, u, tok, logprob, 0, 0};
  const int size = dtype == QD_FP32 ? 4 : 2, parts = cluster * kSampleWarps;
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
