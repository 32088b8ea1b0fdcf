// q/k RMSNorm, rotary positions and the K/V append into cache pages, for a ragged batch of new tokens.
//
// Every element of the token's QKV row is read once and written once (to q_out or a page), so the kernel is
// bound by memory: 4 bytes per element, and for a few tokens by the latency of its dependent loads.
//
// A group of head_dim / 16 lanes holds one head: lane c the 16-byte chunks c of the first and of the second
// half of the rotated elements (the pair that one angle turns sits in one lane, so the rotation needs no
// exchange), and of the rest past 2 * rot_half two neighbouring chunks. The mean of squares is a butterfly
// over the group. A warp takes 4 heads (8 of head_dim 64) of one token, or twice as many, so the request
// lookup, the page and the cos / sin rows are the warp's.
//
// Into 8-bit pages the rotated K row and the V row go as E4M3 values and one power of two for the row: the least
// 2^e with |x| <= 448 * 2^e, from the exponent and the mantissa of the row's largest finite |x| (a butterfly over
// the head's lanes). A power of two because E4M3 has an exponent of its own: a scale between two powers would save
// less than a bit of its range and none of its precision, and with a power of two what is read back is exact in
// BF16 and in FP16 (e from -15 to 7 keeps the least and the largest code in FP16's range).
#include <cuda_fp8.h>

#include <cfloat>
#include <climits>

#include "qd_host.h"
#include "qd_paged_dev.cuh"

namespace qd {

struct AppendArgs {
  PagedBatch b;
  const char* qkv;
  const char *q_norm, *k_norm;
  const float *cos, *sin;
  char *q_out, *k_pages, *v_pages;
  int64_t ldqkv, ldq, ld_cs, n_pos;
  int rot_half;
  float eps;
  uint8_t *k_scale, *v_scale;  // 8-bit pages: the rows' exponents + 127, [page][KV head][row of the page]
  int64_t ss_page, ss_head;
};

// The exponent of a row whose largest finite |x| is `most`: the least e with most <= 448 * 2^e (448 = 1.75 * 2^8),
// within what FP16 can hold all codes of. A row of zeros has the least one.
__device__ __forceinline__ int row_exponent(float most) {
  const uint32_t u = __float_as_uint(most);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kHeldLeastExp), kHeldMostExp);
}
// Two values over the row's power of two as E4M3: beyond +-448 (where the exponent was cut) +-448.
__device__ __forceinline__ uint32_t held_pair(float a, float b, float inv) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}

constexpr int kAppendThreads = 128;
// CTAs an SM, which is 72 registers a thread: 16-bit pages need no more, and into 8-bit pages 14,771 tokens take 83 to 88
// us, where 96 registers without a spill take 102 (a warp waits for its loads most of the time). In twos the 8-bit
// instances spill: 96 bytes stored and 132 loaded in the code of a BF16 thread, 108 and 176 in FP16's
constexpr int kAppendResident = 7;

// kUnits: groups of heads of one token that a warp takes, all their loads in flight before the first is used.
// 14,771 prompt tokens of 48 heads of 128 take 69 to 73 us, 5.0 to 5.2 TB/s over the 364 MB that have to move (a copy
// reaches 6.5); 64 single tokens 3.0 us and one 2.2 us in a graph, of which the launch is most (a call takes the
// host 11.8). Into 8-bit pages the prompts take 83 to 88 us (3.8 to 4.0 TB/s over 334 MB): the rows' maxima and codes add
// a third to the instructions, and there are 28 warps an SM to wait for loads.
template <typename T, int D, int kUnits, bool kHeld>
__global__ void __launch_bounds__(kAppendThreads, kAppendResident) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int kLanes = D / 16, kHeads = 32 / kLanes;  // lanes per head, heads per unit
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, c = lane % kLanes;
  const int heads = a.b.nq + 2 * a.b.nkv, per = (heads + kHeads * kUnits - 1) / (kHeads * kUnits);
  const int64_t warp = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = warp / per;
  if (t >= a.b.tokens) return;
  const int h0 = (int)(warp - t * per) * kHeads * kUnits + lane / kLanes;
  // chunk offsets of this lane within a head
  const bool turned = c < a.rot_half / 8;
  const int e0 = turned ? 8 * c : 2 * a.rot_half + 16 * (c - a.rot_half / 8);
  const int e1 = turned ? a.rot_half + 8 * c : e0 + 8;
  const T* row = reinterpret_cast<const T*>(a.qkv) + t * a.ldqkv;
  uint4 u0[kUnits], u1[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {  // lanes past the last head follow it, and store nothing
    const T* x = row + (int64_t)min(h0 + k * kHeads, heads - 1) * D;
    u0[k] = __ldcs(reinterpret_cast<const uint4*>(x + e0));
    u1[k] = __ldcs(reinterpret_cast<const uint4*>(x + e1));
  }

  int i, pos;
  if (a.b.batch <= 32) {  // every request's end and length at once: one wait for memory in place of three
    const int end = lane < a.b.batch ? ld_i32(a.b.cu + lane + 1) : INT_MAX;
    const int kv = lane < a.b.batch ? ld_i32(a.b.kv_len + lane) : 0;
    i = __popc(__ballot_sync(0xffffffffu, end <= (int)t));
    if (i >= a.b.batch) return;  // a row that belongs to no request
    pos = __shfl_sync(0xffffffffu, kv - end, i) + (int)t;
  } else {
    i = warp_find_request(a.b.cu, a.b.batch, (int)t, lane);
    if (i >= a.b.batch) return;
    pos = ld_i32(a.b.kv_len + i) - ld_i32(a.b.cu + i + 1) + (int)t;
  }
  if (pos < 0 || pos >= a.n_pos) {
    if (lane == 0) flag_error(a.b.err, QD_DEVERR_POS);
    return;
  }
  int64_t page_at = -1, scale_at = 0;  // of this position's row of KV head 0
  if (h0 + (kUnits - 1) * kHeads >= a.b.nq) {
    const int entry = pos >> a.b.page_shift;
    const int page = entry < a.b.max_pages ? ld_i32(a.b.table + i * a.b.ld_table + entry) : -1;
    if (page >= 0 && page < a.b.n_pages) {
      page_at = page * a.b.ps_page + (int64_t)(pos & (a.b.page_size - 1)) * D;
      if constexpr (kHeld) scale_at = page * a.ss_page + (pos & (a.b.page_size - 1));
    } else if (c == 0) {
      flag_error(a.b.err, QD_DEVERR_PAGE);
    }
  }
  float cs[8], sn[8];
  if (turned) {
    const float4* cp = reinterpret_cast<const float4*>(a.cos + pos * a.ld_cs + 8 * c);
    const float4* sp = reinterpret_cast<const float4*>(a.sin + pos * a.ld_cs + 8 * c);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float4 x = cp[k], y = sp[k];
      cs[4 * k] = x.x, cs[4 * k + 1] = x.y, cs[4 * k + 2] = x.z, cs[4 * k + 3] = x.w;
      sn[4 * k] = y.x, sn[4 * k + 1] = y.y, sn[4 * k + 2] = y.z, sn[4 * k + 3] = y.w;
    }
  }
#pragma unroll
  for (int unit = 0; unit < kUnits; ++unit) {
    const int h = h0 + unit * kHeads;
    const bool is_v = h >= a.b.nq + a.b.nkv;
    const int kv_head = h - a.b.nq - (is_v ? a.b.nkv : 0);
    char* dst = nullptr;
    if (h < a.b.nq)
      dst = a.q_out + (t * a.ldq + (int64_t)h * D) * 2;
    else if (page_at >= 0)
      dst = (is_v ? a.v_pages : a.k_pages) + (page_at + kv_head * a.b.ps_head) * (kHeld ? 1 : 2);
    float x[16];
    auto unpack = [&]() {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = Elem<T>::unpack((&u0[unit].x)[k]), q = Elem<T>::unpack((&u1[unit].x)[k]);
        x[2 * k] = p.x;
        x[2 * k + 1] = p.y;
        x[8 + 2 * k] = q.x;
        x[8 + 2 * k + 1] = q.y;
      }
    };
    unpack();
    // (of 8-bit rows, whose instructions come on top of these, a warp's V heads alone need neither norm nor rotation)
    const bool plain = kHeld && h0 + unit * kHeads - lane / kLanes >= a.b.nq + a.b.nkv;
    if (a.q_norm && !plain) {  // every lane takes part in the sum; V heads do not use it
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) sq = fmaf(x[k], x[k], sq);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      const float rstd = rsqrtf(sq * (1.0f / D) + a.eps);
      const T* w = reinterpret_cast<const T*>(h < a.b.nq ? a.q_norm : a.k_norm);
      const uint4 w0 = *reinterpret_cast<const uint4*>(w + e0), w1 = *reinterpret_cast<const uint4*>(w + e1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = Elem<T>::unpack((&w0.x)[k]), q = Elem<T>::unpack((&w1.x)[k]);
        x[2 * k] *= rstd * p.x;
        x[2 * k + 1] *= rstd * p.y;
        x[8 + 2 * k] *= rstd * q.x;
        x[8 + 2 * k + 1] *= rstd * q.y;
      }
    }
    if (turned && !plain) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = x[k], q = x[8 + k];
        x[k] = p * cs[k] - q * sn[k];
        x[8 + k] = q * cs[k] + p * sn[k];
      }
    }
    if (kHeld && h0 + unit * kHeads - lane / kLanes + kHeads > a.b.nq) {  // (some head of the warp's is K or V)
      if (is_v && !plain) unpack();  // V goes in as it was
      auto largest = [&]() {  // of the row (NaN is passed over)
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) m = fmaxf(m, fabsf(x[k]));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
      };
      float most = largest();
      if (__any_sync(0xffffffffu, most > FLT_MAX)) {  // infinities are held as NaN, and are not what a row is measured by
        const float top = h < a.b.nq ? INFINITY : FLT_MAX;  // (queries are not held, and keep theirs)
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = fabsf(x[k]) <= top ? x[k] : __uint_as_float(0x7fffffffu);
        most = largest();
      }
      if (h >= heads || !dst) continue;
      if (h >= a.b.nq) {
        const int e = row_exponent(most);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = held_pair(x[4 * k], x[4 * k + 1], inv) | held_pair(x[4 * k + 2], x[4 * k + 3], inv) << 16;
        *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
        if (c == 0) (is_v ? a.v_scale : a.k_scale)[scale_at + kv_head * a.ss_head] = (uint8_t)(e + 127);
        continue;
      }
    }
    if (h >= heads || !dst) continue;
    uint4 o0 = u0[unit], o1 = u1[unit];  // V goes into the page as it is
    if (!is_v) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        (&o0.x)[k] = Elem<T>::pack(x[2 * k], x[2 * k + 1]);
        (&o1.x)[k] = Elem<T>::pack(x[8 + 2 * k], x[8 + 2 * k + 1]);
      }
    }
    *reinterpret_cast<uint4*>(dst + 2 * e0) = o0;
    *reinterpret_cast<uint4*>(dst + 2 * e1) = o1;
  }
}

template <typename T, int D>
static const void* append_kernel(bool two, bool held) {
  return held  ? (two ? (const void*)paged_append_kernel<T, D, 2, true> : (const void*)paged_append_kernel<T, D, 1, true>)
         : two ? (const void*)paged_append_kernel<T, D, 2, false>
               : (const void*)paged_append_kernel<T, D, 1, false>;
}

// Pages of `rows` elements of a head must not overlap: heads lie inside a page, or pages inside a head.
static bool pools_overlap(int64_t rows, int64_t ps_page, int64_t ps_head, int64_t n_pages, int nkv) {
  return ps_head < rows || ps_page < rows ||
         ((ps_page - rows) / ps_head < nkv - 1 && (ps_head - rows) / ps_page < n_pages - 1);
}

int paged_batch_check(const char* what, int dtype, int64_t tokens, int nq, int nkv, int head_dim, const void* k_pages,
                      const void* v_pages, int64_t n_pages, int page_size, int64_t ps_page, int64_t ps_head,
                      const int32_t* cu, const int32_t* kv_len, int batch, const int32_t* table, int64_t ld_table,
                      int max_pages, int* err, PagedBatch* b) {
  if (dtype != QD_BF16 && dtype != QD_FP16)
    return set_error(QD_ERR_UNSUPPORTED, "%s: element type %d (QD_BF16 or QD_FP16)", what, dtype);
  if (head_dim != 64 && head_dim != 128)
    return set_error(QD_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, head_dim);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return set_error(QD_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64 or 128)", what, page_size);
  if (nkv < 1 || nq < nkv || nq % nkv || nq / nkv > 128 || nq > 65536)
    return set_error(QD_ERR_ARG, "%s: %d query heads over %d KV heads", what, nq, nkv);
  const int some = tokens > 0;  // without tokens nothing is read: no requests, and null arrays, are allowed
  if (batch < some || max_pages < some || ld_table < max_pages || n_pages < 1 || n_pages > INT32_MAX || tokens < 0 ||
      tokens > INT32_MAX)
    return set_error(QD_ERR_ARG, "%s: batch %d, %d pages a row (stride %lld), %lld pages, %lld tokens", what, batch,
                     max_pages, (long long)ld_table, (long long)n_pages, (long long)tokens);
  if (!aligned16(k_pages) || !aligned16(v_pages) || (some && (!k_pages || !v_pages || !cu || !kv_len || !table)))
    return set_error(QD_ERR_ARG, "%s: null or misaligned pool, or null batch array", what);
  if (ps_head % 8 || ps_page % 8 || pools_overlap((int64_t)page_size * head_dim, ps_page, ps_head, n_pages, nkv))
    return set_error(QD_ERR_ARG, "%s: page stride %lld, head stride %lld", what, (long long)ps_page,
                     (long long)ps_head);
  *b = PagedBatch{cu, kv_len, table, ld_table, tokens, n_pages, ps_page, ps_head, batch, max_pages, page_size,
                  __builtin_ctz(page_size), nq, nkv, err};
  return QD_OK;
}

int paged_batch_check8(const char* what, int dtype, int64_t tokens, int nq, int nkv, int head_dim, const void* k_pages,
                       const void* v_pages, const void* k_scale, const void* v_scale, int64_t n_pages, int page_size,
                       int64_t ps_page, int64_t ps_head, int64_t ss_page, int64_t ss_head, const int32_t* cu,
                       const int32_t* kv_len, int batch, const int32_t* table, int64_t ld_table, int max_pages, int* err,
                       PagedBatch* b) {
  const int rc = paged_batch_check(what, dtype, tokens, nq, nkv, head_dim, k_pages, v_pages, n_pages, page_size, ps_page,
                                   ps_head, cu, kv_len, batch, table, ld_table, max_pages, err, b);
  if (rc != QD_OK) return rc;
  if (!aligned16(k_scale) || !aligned16(v_scale) || (tokens > 0 && (!k_scale || !v_scale)))
    return set_error(QD_ERR_ARG, "%s: null or misaligned scales", what);
  // whole 16-byte pieces: what a copy of a page takes
  if (ps_head % 16 || ps_page % 16 || ss_head % 16 || ss_page % 16 || pools_overlap(page_size, ss_page, ss_head, n_pages, nkv))
    return set_error(QD_ERR_ARG, "%s: page strides %lld, %lld, head strides %lld, %lld (values, scales)", what,
                     (long long)ps_page, (long long)ss_page, (long long)ps_head, (long long)ss_head);
  return QD_OK;
}

}  // namespace qd

using namespace qd;

// What both entry points check and launch: 16-bit pages without scales, 8-bit pages with.
static int launch_append(const char* what, const void* qkv, int64_t ldqkv, int dtype, int64_t tokens, int nq_heads,
                         int nkv_heads, int head_dim, const void* q_norm, const void* k_norm, float eps,
                         const float* cos, const float* sin, int64_t ld_cs, int64_t n_pos, int rot_half, void* q_out,
                         int64_t ldq, void* k_pages, void* v_pages, int pdl, cudaStream_t stream, bool held,
                         AppendArgs& a) {
  const int heads = nq_heads + 2 * nkv_heads;
  if ((tokens > 0 && (!qkv || !q_out)) || !aligned16(qkv) || !aligned16(q_out) || ldqkv % 8 || ldq % 8 ||
      ldqkv < (int64_t)heads * head_dim || ldq < (int64_t)nq_heads * head_dim)
    return set_error(QD_ERR_ARG, "%s: qkv / q_out null, misaligned or with a bad stride (%lld, %lld)", what,
                     (long long)ldqkv, (long long)ldq);
  if ((q_norm == nullptr) != (k_norm == nullptr) || !aligned16(q_norm) || !aligned16(k_norm))
    return set_error(QD_ERR_ARG, "%s: q_norm and k_norm go together, 16-byte aligned", what);
  if (!cos || !sin || !aligned16(cos) || !aligned16(sin) || rot_half < 8 || rot_half % 8 || 2 * rot_half > head_dim ||
      ld_cs < rot_half || ld_cs % 4 || n_pos < 1)
    return set_error(QD_ERR_ARG, "%s: tables of %lld positions, %d angles, stride %lld", what, (long long)n_pos,
                     rot_half, (long long)ld_cs);
  if (tokens == 0) return QD_OK;
  a.qkv = static_cast<const char*>(qkv);
  a.q_norm = static_cast<const char*>(q_norm);
  a.k_norm = static_cast<const char*>(k_norm);
  a.cos = cos;
  a.sin = sin;
  a.q_out = static_cast<char*>(q_out);
  a.k_pages = static_cast<char*>(k_pages);
  a.v_pages = static_cast<char*>(v_pages);
  a.ldqkv = ldqkv;
  a.ldq = ldq;
  a.ld_cs = ld_cs;
  a.n_pos = n_pos;
  a.rot_half = rot_half;
  a.eps = eps;
  // Two groups of heads a warp once there are warps enough to fill the SMs without: 64 tokens of 48 heads (768
  // groups of 4) take 3.0 us one by one and 3.3 in twos, 256 tokens 6.7 and 4.2, 14,771 tokens 85 and 71.
  const int group = 512 / head_dim;
  const bool two = tokens * ((heads + group - 1) / group) > 2048;
  const int per = (heads + group * (two ? 2 : 1) - 1) / (group * (two ? 2 : 1));
  const int64_t blocks = (tokens * per + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  if (blocks > INT32_MAX) return set_error(QD_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)tokens);
  const void* fn = dtype == QD_BF16
                       ? (head_dim == 128 ? append_kernel<__nv_bfloat16, 128>(two, held) : append_kernel<__nv_bfloat16, 64>(two, held))
                       : (head_dim == 128 ? append_kernel<__half, 128>(two, held) : append_kernel<__half, 64>(two, held));
  return launch_kernel(fn, dim3((unsigned)blocks), dim3(kAppendThreads), 0, pdl, stream, &a);
}

extern "C" int qd_paged_rope_append(const void* qkv, int64_t ldqkv, int dtype, int64_t tokens, int nq_heads,
                                    int nkv_heads, int head_dim, const void* q_norm, const void* k_norm, float eps,
                                    const float* cos, const float* sin, int64_t ld_cs, int64_t n_pos, int rot_half,
                                    const int32_t* cu_tokens, const int32_t* kv_len, int batch,
                                    const int32_t* page_table, int64_t ld_table, int max_pages, void* q_out,
                                    int64_t ldq, void* k_pages, void* v_pages, int64_t n_pages, int page_size,
                                    int64_t ps_page, int64_t ps_head, int* err, int pdl, cudaStream_t stream) {
  AppendArgs a = {};
  const int rc = paged_batch_check("paged append", dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages, v_pages,
                                   n_pages, page_size, ps_page, ps_head, cu_tokens, kv_len, batch, page_table,
                                   ld_table, max_pages, err, &a.b);
  if (rc != QD_OK) return rc;
  return launch_append("paged append", qkv, ldqkv, dtype, tokens, nq_heads, nkv_heads, head_dim, q_norm, k_norm, eps, cos,
                       sin, ld_cs, n_pos, rot_half, q_out, ldq, k_pages, v_pages, pdl, stream, false, a);
}

extern "C" int qd_paged_rope_append8(const void* qkv, int64_t ldqkv, int dtype, int64_t tokens, int nq_heads,
                                     int nkv_heads, int head_dim, const void* q_norm, const void* k_norm, float eps,
                                     const float* cos, const float* sin, int64_t ld_cs, int64_t n_pos, int rot_half,
                                     const int32_t* cu_tokens, const int32_t* kv_len, int batch,
                                     const int32_t* page_table, int64_t ld_table, int max_pages, void* q_out,
                                     int64_t ldq, void* k_pages, void* v_pages, void* k_scale, void* v_scale,
                                     int64_t n_pages, int page_size, int64_t ps_page, int64_t ps_head, int64_t ss_page,
                                     int64_t ss_head, int* err, int pdl, cudaStream_t stream) {
  AppendArgs a = {};
  const int rc = paged_batch_check8("paged append (8 bits)", dtype, tokens, nq_heads, nkv_heads, head_dim, k_pages,
                                    v_pages, k_scale, v_scale, n_pages, page_size, ps_page, ps_head, ss_page, ss_head,
                                    cu_tokens, kv_len, batch, page_table, ld_table, max_pages, err, &a.b);
  if (rc != QD_OK) return rc;
  a.k_scale = static_cast<uint8_t*>(k_scale);
  a.v_scale = static_cast<uint8_t*>(v_scale);
  a.ss_page = ss_page;
  a.ss_head = ss_head;
  return launch_append("paged append (8 bits)", qkv, ldqkv, dtype, tokens, nq_heads, nkv_heads, head_dim, q_norm, k_norm, eps, cos,
                       sin, ld_cs, n_pos, rot_half, q_out, ldq, k_pages, v_pages, pdl, stream, true, a);
}
