// A token per row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number.
//
// The weights are whole multiples of 2^-40 of the row's largest, so every sum is an exact 64-bit integer
// and the kept set and the token do not depend on how the additions are split. With the logits as
// order-preserving 32-bit keys the kept set is a prefix of the tokens ordered by (key descending, index):
// all keys above a threshold, and of the keys equal to it the first few by index. One CTA per row finds the
// threshold bit by bit (the largest key at which the keys from it up number top_k, or weigh top_p of the
// sum), then walks the kept weights in index order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qd_common.cuh"
#include "qd_host.h"

namespace qd {

constexpr int kSampleThreads = 1024;
constexpr float kSampleOne = 1099511627776.0f;  // 2^40
constexpr int64_t kSampleMaxVocab = 1 << 18;    // 2^18 weights of 2^40 stay below 2^63

struct SampleArgs {
  const void* logits;
  int64_t ld, vocab;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p, *u;
  int64_t* tok;
  float* logprob;
};

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_logit(const __half* p) { return __half2float(*p); }

// larger logit = larger key; -0 and +0 are the same key, NaN the key of -inf
__device__ __forceinline__ uint32_t logit_key(float l) {
  if (l != l) l = -INFINITY;
  const uint32_t u = __float_as_uint(l + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// d = (l - m) / temperature of the definition, and the weight in units of 2^-40
__device__ __forceinline__ float logit_depth(float l, float m, float inv_t) {
  return l == -INFINITY ? l : l == m ? 0.f : __fmul_rn(__fsub_rn(l, m), inv_t);
}
__device__ __forceinline__ uint64_t depth_weight(float d) { return __float2ull_rn(expf(d) * kSampleOne); }

// sums of (a, b) over the CTA, in every thread
struct Sum2 {
  uint64_t a, b;
};
__device__ __forceinline__ Sum2 block_sum2(uint64_t a, uint64_t b, uint64_t (*sh)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if (lane == 0) {
    sh[warp][0] = a;
    sh[warp][1] = b;
  }
  __syncthreads();
  a = sh[lane][0];
  b = sh[lane][1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return Sum2{a, b};
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ uint64_t sh[32][2];
  __shared__ uint64_t seg[kSampleThreads];
  __shared__ uint32_t ties[kSampleThreads];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, n = (int)a.vocab;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const float temp = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(temp >= 1e-5f);
  const float scale_t = greedy ? 1.f : __fdiv_rn(1.f, temp);
  // a thread's tokens are neighbours, so the threads' sums are in index order
  const int per = (n + kSampleThreads - 1) / kSampleThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);

  uint64_t best = 0;  // (key, ~index) of the largest logit, the lowest index among equals
  for (int i = i0; i < i1; ++i) {
    const uint64_t c = ((uint64_t)logit_key(load_logit(x + i)) << 32) | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if ((tid & 31) == 0) sh[tid >> 5][0] = best;
  __syncthreads();
  for (int w = 0; w < 32; ++w) best = sh[w][0] > best ? sh[w][0] : best;
  __syncthreads();
  const float m = key_logit((uint32_t)(best >> 32));
  const float inv_t = m == INFINITY ? 1.f : scale_t;  // +inf logits: the others weigh nothing at any temperature
  if (m == -INFINITY || greedy) {
    if (tid == 0) {
      a.tok[row] = m == -INFINITY ? -1 : (int64_t)(uint32_t)~(uint32_t)best;
      if (a.logprob) a.logprob[row] = m == -INFINITY ? m : 0.f;
    }
    return;
  }
  // (number, weight) of the tokens with key >= k
  auto from = [&](uint32_t k) {
    uint64_t c = 0, w = 0;
    for (int i = i0; i < i1; ++i) {
      const float l = load_logit(x + i);
      if (logit_key(l) >= k) {
        ++c;
        w += depth_weight(logit_depth(key_logit(logit_key(l)), m, inv_t));
      }
    }
    return block_sum2(c, w, sh);
  };
  // the kept prefix as a threshold key and how many of the keys equal to it belong
  uint32_t thr = 0;
  uint64_t take = ~0ull;  // of the ties
  // narrow (thr, take) to the fewest tokens whose number (by_weight: whose weight) reaches `want`
  auto cut = [&](uint64_t want, bool by_weight) {
    uint32_t k = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const Sum2 s = from(k | (1u << bit));
      if ((by_weight ? s.b : s.a) >= want) k |= 1u << bit;
    }
    // k: the largest key such that the tokens from k up reach `want`
    const Sum2 above = k == 0xffffffffu ? Sum2{0, 0} : from(k + 1);
    uint64_t need;
    if (by_weight) {
      const uint64_t w1 = depth_weight(logit_depth(key_logit(k), m, inv_t));
      need = w1 ? (want - above.b + w1 - 1) / w1 : ~0ull;
    } else {
      need = want - above.a;
    }
    if (k > thr || (k == thr && need < take)) {
      thr = k;
      take = need;
    }
  };
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < n) cut((uint64_t)k, false);
  auto kept_sum = [&]() {
    const Sum2 up = thr == 0xffffffffu ? Sum2{0, 0} : from(thr + 1), all = from(thr);
    const uint64_t eq = all.a - up.a, w1 = depth_weight(logit_depth(key_logit(thr), m, inv_t));
    return thr == 0 ? all.b : up.b + min(eq, take) * w1;
  };
  const float p = a.top_p ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    const double want = ceil((double)p * (double)(int64_t)kept_sum());
    cut(want >= 1. ? (uint64_t)want : 1u, true);
  }
  const float mp = a.min_p ? a.min_p[row] : 0.f;
  const float floor_d = mp > 0.f ? logf(fminf(mp, 1.f)) : -INFINITY;

  // each thread's kept weight, the ties counted apart (they all weigh the same)
  auto in_min = [&](float l) { return logit_depth(l, m, inv_t) >= floor_d; };
  uint64_t mine = 0;
  uint32_t eq = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t key = logit_key(load_logit(x + i));
    const float l = key_logit(key);
    if (l == -INFINITY || !in_min(l)) continue;
    if (key > thr) mine += depth_weight(logit_depth(l, m, inv_t));
    eq += key == thr;
  }
  seg[tid] = mine;
  ties[tid] = eq;
  __syncthreads();
  if (tid == 0) {
    const uint64_t w1 = depth_weight(logit_depth(key_logit(thr), m, inv_t));
    auto taken = [&](uint64_t before, uint64_t here) {  // ties taken out of `here` that come after `before`
      return before >= take ? (uint64_t)0 : min(here, take - before);
    };
    uint64_t total = 0, seen = 0;
    for (int s = 0; s < kSampleThreads; ++s) {
      total += seg[s] + (ties[s] ? taken(seen, ties[s]) * w1 : 0);
      seen += ties[s];
    }
    const double u = (double)a.u[row];
    const double at_d = floor(u * (double)(int64_t)total);
    uint64_t at = at_d >= 1. ? (uint64_t)at_d : 0;  // NaN and negative numbers count as 0
    if (at >= total) at = total - 1;
    uint64_t run = 0;
    seen = 0;
    int s = 0;
    for (;; ++s) {
      const uint64_t w = seg[s] + (ties[s] ? taken(seen, ties[s]) * w1 : 0);
      if (run + w > at) break;
      run += w;
      seen += ties[s];
    }
    int i = s * per;
    for (;; ++i) {
      const uint32_t key = logit_key(load_logit(x + i));
      const float l = key_logit(key);
      if (l == -INFINITY || !in_min(l) || key < thr) continue;
      if (key == thr && seen++ >= take) continue;
      run += depth_weight(logit_depth(l, m, inv_t));
      if (run > at) {
        a.tok[row] = i;
        if (a.logprob) a.logprob[row] = logit_depth(l, m, inv_t) - logf((float)(int64_t)total * (1.f / kSampleOne));
        break;
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
  SampleArgs a = {logits, ld, vocab, temperature, top_k, top_p, min_p, u, tok, logprob};
  const void* fn = dtype == QD_BF16   ? (const void*)sample_kernel<__nv_bfloat16>
                   : dtype == QD_FP16 ? (const void*)sample_kernel<__half>
                                      : (const void*)sample_kernel<float>;
  return launch_kernel(fn, dim3((unsigned)rows), dim3(kSampleThreads), 0, pdl, stream, &a);
}
