// The paged key/value cache: appending a step's rows (rotary embedding and
// 8-bit numbers included) and reading sequences back as a dense cache.
//
// Both kernels move rows of D numbers, 16-byte vectors of bf16 per thread, and
// are bound by memory or, at decode sizes, by the launch.  Measured: the new rows
// of eight sequences (8 + 2 + 2 heads of 96) appended in 2.5 us; 8-bit contexts of
// 17,994 tokens (2 heads of 96) read back in 7.1 us, 4.5 TB/s, a latent cache of 42,034
// tokens of 128 in 5.2 us, 5.3 TB/s (one vector a thread at a time: 11.7 and 8.7).
#include "paged.cuh"

namespace parrot {

namespace {

constexpr int kAppendThreads = 256;

// Lanes that share a row: the power of two >= D / 8, so a row's largest
// magnitude is a shuffle reduction (D = 96 leaves 4 of 16 lanes idle).
__host__ __device__ constexpr int row_lanes(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : 16; }

}  // namespace

// One row group = (token, head), heads in the projection's order: q, k, v.
//   q, k: (e, o) -> (e cos - o sin, e sin + o cos) at the token's position, in
//   fp32 from fp32 tables, rounded once (to bf16, or to e4m3 for a cached k);
//   the products and the sum are separate roundings (no contraction), so the
//   value does not depend on how the compiler fuses them.
// e4m3: amax over the row's finite and infinite numbers by shuffles, then one
// exact scaling and one rounding to nearest even; infinities saturate, NaN
// stays NaN.
template <int D, bool E4M3>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(PagedAppendArgs a) {
  constexpr int L = row_lanes(D);
  griddep_wait();
  griddep_launch();
  const long long t = (long long)blockIdx.x * kAppendThreads + threadIdx.x;
  const int heads = a.q_heads + a.kv.kv_heads * (a.kv.value != nullptr ? 2 : 1);
  const long long row = t / L;
  const int c = (int)(t % L);  // this thread's 8 columns
  const int token = (int)(row / heads), h = (int)(row - (long long)token * heads);
  bool live = token < a.batch.tokens;
  int b = -1, pos = 0;
  if (live) b = sequence_of(a.batch, token);
  if (b >= 0) {
    const int2 r = batch_rows(a.batch, b);
    pos = a.batch.context_len[b] - (r.y - token);
  }
  live = b >= 0 && c < D / 8;
  const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv.kv_heads;
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  if (live && (pos < 0 || (a.cos_t != nullptr && pos >= a.rope_positions))) {
    report_status(a.status, kStatusBadIndex, 50, pos);
    live = false;
  }
  if (live) {
    const uint4 v = *(reinterpret_cast<const uint4*>(a.qkv + (long long)token * a.qkv_row +
                                                         (long long)h * D + c * 8));
    bf16x8_to_float(v, f);
    if (a.cos_t != nullptr && (is_q || is_k)) {
      const float4 co = *(reinterpret_cast<const float4*>(a.cos_t + (long long)pos * (D / 2)) + c);
      const float4 si = *(reinterpret_cast<const float4*>(a.sin_t + (long long)pos * (D / 2)) + c);
      const float cs[4] = {co.x, co.y, co.z, co.w}, sn[4] = {si.x, si.y, si.z, si.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = f[2 * i], o = f[2 * i + 1];
        f[2 * i] = __fsub_rn(__fmul_rn(e, cs[i]), __fmul_rn(o, sn[i]));
        f[2 * i + 1] = __fadd_rn(__fmul_rn(e, sn[i]), __fmul_rn(o, cs[i]));
      }
    }
  }
  if (is_q) {
    if (live)
      reinterpret_cast<uint4*>(a.q_out + ((long long)token * a.q_heads + h) * D)[c] =
          float_to_bf16x8(f);
    if (!E4M3) return;
  }
  const int kvh = is_k ? h - a.q_heads : h - a.q_heads - a.kv.kv_heads;
  long long at = 0;
  if (live && !is_q) {
    int page = -1;
    if (pos < ((long long)a.batch.table_width << a.kv.page_shift))
      page = page_of(a.batch, a.kv, b, pos, a.status);
    else
      report_status(a.status, kStatusBadIndex, 51, pos);
    live = page >= 0;
    at = live ? pool_row(a.kv, page, kvh, pos) : 0;
  }
  if constexpr (!E4M3) {
    if (live)
      reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(is_k ? a.kv.key : a.kv.value) +
                               at * D)[c] = float_to_bf16x8(f);
  } else {
    // every lane of the warp takes part in the shuffles
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));  // fmaxf passes over NaN
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (is_q || !live) return;
    const int e = scale_exponent(amax);
    const float inv = pow2(-e);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
          make_float2(f[4 * i] * inv, f[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
          make_float2(f[4 * i + 2] * inv, f[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
      w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_k ? a.kv.key : a.kv.value) + at * D)[c] =
        make_uint2(w[0], w[1]);
    if (c == 0) (is_k ? a.kv.key_scale : a.kv.value_scale)[at] = (uint8_t)(e + kScaleBias);
  }
}

// Sequence b's rows as dense [B, KVH, max_len, D] bf16; zeros past its
// context.  A CTA writes 64 or 128 rows; a thread asks for all of its vectors
// (16 bytes of bf16, 8 of e4m3) before it stores the first.
constexpr int kGatherThreads = 256;
__host__ __device__ constexpr int gather_rows(int d) { return d <= 64 ? 128 : 64; }

template <int D, bool E4M3>
__global__ void __launch_bounds__(kGatherThreads) paged_gather_kernel(PagedGatherArgs a) {
  constexpr int NV = D / 8;  // vectors of a row
  constexpr int U = gather_rows(D) * NV / kGatherThreads;
  static_assert(U * kGatherThreads == gather_rows(D) * NV, "whole vectors per thread");
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.z, h = blockIdx.y % a.kv.kv_heads;
  const bool is_k = blockIdx.y < (unsigned)a.kv.kv_heads;
  const int n = min(context_of(a.batch, a.kv, b, a.status), a.max_len);
  const void* pool = is_k ? a.kv.key : a.kv.value;
  const uint8_t* scale = is_k ? a.kv.key_scale : a.kv.value_scale;
  const long long p0 = (long long)blockIdx.x * gather_rows(D);
  uint4* out = reinterpret_cast<uint4*>(is_k ? a.key_out : a.value_out) +
               (((long long)b * a.kv.kv_heads + h) * a.max_len + p0) * NV;
  const int left = (int)min((long long)gather_rows(D), a.max_len - p0);
  long long row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int p = (threadIdx.x + u * kGatherThreads) / NV;
    row[u] = -1;
    if (p0 + p < n) {
      const int page = page_of(a.batch, a.kv, b, (int)p0 + p, a.status);
      if (page >= 0) row[u] = pool_row(a.kv, page, h, (int)p0 + p);
    }
  }
  uint4 v[U];
  uint32_t s2[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (threadIdx.x + u * kGatherThreads) % NV;
    v[u] = make_uint4(0u, 0u, 0u, 0u);
    s2[u] = 0u;
    if (row[u] < 0) continue;
    if constexpr (E4M3) {
      const uint2 w = reinterpret_cast<const uint2*>(pool)[row[u] * NV + c];
      v[u].x = w.x, v[u].y = w.y;
      s2[u] = scale[row[u]];
    } else {
      v[u] = reinterpret_cast<const uint4*>(pool)[row[u] * NV + c];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = threadIdx.x + u * kGatherThreads;
    if (E4M3 && row[u] >= 0) {
      const uint32_t pair = scale_pair(s2[u]);
      const uint2 lo = e4m3x4_to_bf16(v[u].x, pair), hi = e4m3x4_to_bf16(v[u].y, pair);
      v[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    if (i / NV < left) out[i] = v[u];
  }
}

template <int D>
static int launch_append_d(const PagedAppendArgs& a, cudaStream_t stream) {
  const long long heads = a.q_heads + a.kv.kv_heads * (a.kv.value != nullptr ? 2 : 1);
  const long long threads = (long long)a.batch.tokens * heads * row_lanes(D);
  const long long blocks = (threads + kAppendThreads - 1) / kAppendThreads;
  if (blocks > 0x7fffffffll) return -1;
  auto k = a.kv.key_scale != nullptr ? paged_append_kernel<D, true> : paged_append_kernel<D, false>;
  return launch_pdl(k, dim3((unsigned)blocks), dim3(kAppendThreads), 0, stream, a) == cudaSuccess
             ? 0
             : -2;
}

int launch_paged_append(const PagedAppendArgs& a, cudaStream_t stream) {
  switch (a.kv.head_dim) {
    case 32: return launch_append_d<32>(a, stream);
    case 64: return launch_append_d<64>(a, stream);
    case 96: return launch_append_d<96>(a, stream);
    case 128: return launch_append_d<128>(a, stream);
  }
  return -1;
}

template <int D>
static int launch_gather_d(const PagedGatherArgs& a, cudaStream_t stream) {
  const dim3 grid((unsigned)(((long long)a.max_len + gather_rows(D) - 1) / gather_rows(D)),
                  (unsigned)(a.kv.kv_heads * (a.kv.value != nullptr ? 2 : 1)),
                  (unsigned)a.batch.batch);
  auto k = a.kv.key_scale != nullptr ? paged_gather_kernel<D, true> : paged_gather_kernel<D, false>;
  return launch_pdl(k, grid, dim3(kGatherThreads), 0, stream, a) == cudaSuccess ? 0 : -2;
}

int launch_paged_gather(const PagedGatherArgs& a, cudaStream_t stream) {
  switch (a.kv.head_dim) {
    case 32: return launch_gather_d<32>(a, stream);
    case 64: return launch_gather_d<64>(a, stream);
    case 96: return launch_gather_d<96>(a, stream);
    case 128: return launch_gather_d<128>(a, stream);
  }
  return -1;
}

}  // namespace parrot
