// What the paged attention kernels share on the device: copies, exponentials, a row's end, tensor-memory helpers.
#pragma once

#include <cuda.h>

#include "qd_common.cuh"
#include "qd_umma.cuh"

namespace qd {

__device__ __forceinline__ void pg_tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "l"(policy)
      : "memory");
}
// announces bytes without arriving: the copies may start before the arrival
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
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
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};\n"
      "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

}  // namespace qd
