// What the paged-cache kernels share: the ragged batch's description, its lookups, and 16-bit element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qd_common.cuh"

namespace qd {

// Request i: token rows cu[i]..cu[i+1]-1, kv_len[i] cached positions (the new tokens' included), page table
// row i. Pools are [page][KV head][row of the page][dim].
struct PagedBatch {
  const int32_t *cu, *kv_len, *table;
  int64_t ld_table, tokens, n_pages, ps_page, ps_head;
  int batch, max_pages, page_size, page_shift, nq, nkv;
  int* err;
};

// Checks the arguments that the paged entry points share and fills in *b; a QD_* status.
int paged_batch_check(const char* what, int dtype, int64_t tokens, int nq, int nkv, int head_dim, const void* k_pages,
                      const void* v_pages, int64_t n_pages, int page_size, int64_t ps_page, int64_t ps_head,
                      const int32_t* cu, const int32_t* kv_len, int batch, const int32_t* table, int64_t ld_table,
                      int max_pages, int* err, PagedBatch* b);

// The same for pages of 8 bits: values of E4M3 and, per row, the exponent of the power of two that they are multiples of
// (+ 127) in pools [page][KV head][row of the page]; strides in bytes, the scales' ss_page and ss_head.
int paged_batch_check8(const char* what, int dtype, int64_t tokens, int nq, int nkv, int head_dim, const void* k_pages,
                       const void* v_pages, const void* k_scale, const void* v_scale, int64_t n_pages, int page_size,
                       int64_t ps_page, int64_t ps_head, int64_t ss_page, int64_t ss_head, const int32_t* cu,
                       const int32_t* kv_len, int batch, const int32_t* table, int64_t ld_table, int max_pages, int* err,
                       PagedBatch* b);
// The exponents that an 8-bit row can have: 2^-9 (the least code) and 448 times these are in FP16's range.
constexpr int kHeldLeastExp = -15, kHeldMostExp = 7;

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(bf_lo(u), bf_hi(u)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Elem<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// The batch's arrays may come from the kernel before: L2 loads, never moved above the wait for it.
__device__ __forceinline__ int ld_i32(const int32_t* p) { return __ldcg(p); }

__device__ __forceinline__ void flag_error(int* err, int code) {
  if (err) atomicOr(err, code);
}

// The request that token row t belongs to, or `batch` when t is past the last: the number of i < batch with
// cu[i + 1] <= t. A warp searches 32 ways at a time, so up to 32 requests take one round of loads and up
// to 1024 take two.
__device__ __forceinline__ int warp_find_request(const int32_t* cu, int batch, int t, int lane) {
  int lo = 0, n = batch;  // the answer is in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int i = lo + (lane + 1) * step;  // cu[i] <= t: at least i requests end at or before t
    const bool past = i <= lo + n && ld_i32(cu + i) <= t;
    const int k = __popc(__ballot_sync(0xffffffffu, past));
    const int end = lo + n;
    lo += k * step;
    n = min(step - 1, end - lo);
  }
  return lo;
}

}  // namespace qd
