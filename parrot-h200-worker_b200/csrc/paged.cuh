// Device helpers of the paged key/value cache (paged.cu, paged_attn.cu).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace parrot {

// A row's scale is 2^e, kept as the byte e + 127.  An e4m3 number keeps its
// four significant bits at any power of two, so a finer scale would buy
// nothing, and number * 2^e is an exact bf16 value: reading the cache back
// adds no rounding.  The exponents are clamped where that stays a normal bf16
// (the smallest number is 2^-9, the largest 448 = 1.75 * 2^8).
constexpr int kScaleBias = 127;
constexpr int kScaleMinExp = -110, kScaleMaxExp = 119;

// The least e with amax <= 448 * 2^e, clamped.  amax finite or infinite, >= 0.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  // amax = (1 + f) 2^x: 1 + f <= 1.75 needs e = x - 8, else x - 7
  // (subnormal amax: x = -127 and below, under the clamp either way)
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleMinExp), kScaleMaxExp);
}

__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four e4m3 numbers (one register) times 2^e as two packed bf16 pairs, exact.
// The bits s eeee mmm moved to the top of a bf16 stand for the same number
// times 2^-120 (exponent biases 7 and 127; both formats' subnormals follow),
// so a product with 2^120 and one with 2^e, both exact, restore it.  NaN is
// the pattern s 1111 111: it would come out as 480 and is put back by hand.
__device__ __forceinline__ uint32_t mul_bf16x2_exact(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t scale_pair(int byte) {  // 2^(byte - 127) twice, as bf16
  const uint32_t one = (uint32_t)byte << 7;
  return one | (one << 16);
}
// Without the scale, and with NaN as 480: for numbers known not to be NaN.
__device__ __forceinline__ uint2 e4m3x4_finite(uint32_t w) {
  constexpr uint32_t k2p120 = ((120u + 127u) << 7) * 0x10001u;
  // bytes (0, 1) and (2, 3) into the upper bytes of the halves of a register
  const uint32_t lo = __byte_perm(w, 0, 0x1404), hi = __byte_perm(w, 0, 0x3424);
  uint2 r;
  r.x = mul_bf16x2_exact((lo & 0x80008000u) | ((lo >> 4) & 0x07f007f0u), k2p120);
  r.y = mul_bf16x2_exact((hi & 0x80008000u) | ((hi >> 4) & 0x07f007f0u), k2p120);
  return r;
}
// A byte of w that is NaN (0x7f or 0xff) sets its top bit here, and no other does.
__device__ __forceinline__ uint32_t e4m3_nan_bits(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint2 e4m3_put_nan(uint2 r, uint32_t nan) {
  if (nan & 0x00000080u) r.x |= 0x00007fffu;
  if (nan & 0x00008000u) r.x |= 0x7fff0000u;
  if (nan & 0x00800000u) r.y |= 0x00007fffu;
  if (nan & 0x80000000u) r.y |= 0x7fff0000u;
  return r;
}
// Sixteen numbers as bf16 (two vectors).
__device__ __forceinline__ void e4m3x16_numbers(const uint4& v, uint4 (&out)[2]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint2 r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = e4m3x4_finite(w[i]);
  if (e4m3_nan_bits(v.x) | e4m3_nan_bits(v.y) | e4m3_nan_bits(v.z) | e4m3_nan_bits(v.w)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = e4m3_put_nan(r[i], e4m3_nan_bits(w[i]));
  }
  out[0] = make_uint4(r[0].x, r[0].y, r[1].x, r[1].y);
  out[1] = make_uint4(r[2].x, r[2].y, r[3].x, r[3].y);
}
__device__ __forceinline__ uint2 e4m3x4_to_bf16(uint32_t w, uint32_t scale2) {
  uint2 r = e4m3x4_finite(w);
  if (const uint32_t nan = e4m3_nan_bits(w)) r = e4m3_put_nan(r, nan);
  r.x = mul_bf16x2_exact(r.x, scale2);
  r.y = mul_bf16x2_exact(r.y, scale2);
  return r;
}

// Tokens [lo, hi) of sequence b in the ragged batch, clamped so that a broken
// query_start can only lose rows, never reach past the batch.
__device__ __forceinline__ int2 batch_rows(const PagedBatch& s, int b) {
  const int lo = min(max(s.query_start[b], 0), s.tokens);
  const int hi = min(max(s.query_start[b + 1], lo), s.tokens);
  return make_int2(lo, hi);
}

// Sequence of batch row i: the last b with query_start[b] <= i (empty
// sequences before it are stepped over), or -1 behind the last sequence.
__device__ __forceinline__ int sequence_of(const PagedBatch& s, int i) {
  int lo = 0, hi = s.batch;  // query_start[lo] <= i < query_start[hi] is sought
  if (i < s.query_start[0] || i >= s.query_start[hi]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.query_start[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A context length as given, at most what the table can hold.
__device__ __forceinline__ int clamp_context(const PagedBatch& s, const PagedKV& kv, int n,
                                             int* status) {
  const long long most = (long long)s.table_width << kv.page_shift;
  if (n > most) {
    report_status(status, kStatusBadIndex, 51, n);
    return (int)most;
  }
  return max(n, 0);
}
__device__ __forceinline__ int context_of(const PagedBatch& s, const PagedKV& kv, int b,
                                          int* status) {
  return clamp_context(s, kv, s.context_len[b], status);
}

// Page of position p of sequence b; -1 (reported) if the table names none.
__device__ __forceinline__ int page_of(const PagedBatch& s, const PagedKV& kv, int b, int p,
                                       int* status) {
  const int page = s.page_table[(long long)b * s.table_width + (p >> kv.page_shift)];
  if ((unsigned)page >= (unsigned)kv.pages) {
    report_status(status, kStatusBadIndex, 52, page);
    return -1;
  }
  return page;
}

// Row index of (page, head, position) in a pool.
__device__ __forceinline__ long long pool_row(const PagedKV& kv, int page, int head, int p) {
  return (((long long)page * kv.kv_heads + head) << kv.page_shift) + (p & kv.page_mask);
}

}  // namespace parrot
