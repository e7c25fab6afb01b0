// Attention of a ragged batch of queries over the paged cache.
//
//   out[i, h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_ih . k_j - m_i)
// over the keys j that token i (at position p of its sequence) sees:
//   j <= p, and without a window or p - j < window or j < sinks.
// A token that sees no key gets zeros.
#include "paged.cuh"

namespace parrot {

namespace {
constexpr int kAttnThreads = 128;
}

// One CTA per (token, query head); a thread scores one key per step, then the
// CTA adds the step's weighted values, a column per thread.
template <int D, bool E4M3>
__global__ void __launch_bounds__(kAttnThreads) paged_attn_kernel(PagedAttnArgs a) {
  __shared__ float q_s[D], p_s[kAttnThreads], red_s[kAttnThreads / 32];
  __shared__ long long row_s[kAttnThreads];
  griddep_wait();
  griddep_launch();
  const int token = blockIdx.x, h = blockIdx.y, kvh = h / (a.heads / a.kv.kv_heads);
  const int b = sequence_of(a.batch, token);
  if (b < 0) return;
  const int2 rows = batch_rows(a.batch, b);
  const int n = context_of(a.batch, a.kv, b, a.status);
  const int pos = n - (rows.y - token);
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int sinks = min(a.sinks, lo);  // keys [0, sinks) and [lo, pos]
  const int seen = pos < 0 ? 0 : sinks + pos - lo + 1;
  const int x = threadIdx.x;
  if (x < D) q_s[x] = __bfloat162float(a.q[(long long)token * a.q_row + h * D + x]);
  auto load8 = [&](const void* pool, const uint8_t* scale, long long r, int c, float* f) {
    uint4 v;
    if constexpr (E4M3) {
      const uint2 w = reinterpret_cast<const uint2*>(pool)[r * (D / 8) + c];
      const uint32_t s2 = scale_pair(scale[r]);
      const uint2 l = e4m3x4_to_bf16(w.x, s2), u = e4m3x4_to_bf16(w.y, s2);
      v = make_uint4(l.x, l.y, u.x, u.y);
    } else {
      v = reinterpret_cast<const uint4*>(pool)[r * (D / 8) + c];
    }
    bf16x8_to_float(v, f);
  };
  const bool sep = a.kv.value != nullptr;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int k0 = 0; k0 < seen; k0 += kAttnThreads) {
    __syncthreads();
    const int i = k0 + x;
    float s = -INFINITY;
    if (i < seen) {
      const int j = i < sinks ? i : lo + i - sinks;
      const int page = page_of(a.batch, a.kv, b, j, a.status);
      const long long r = page < 0 ? -1 : pool_row(a.kv, page, kvh, j);
      row_s[x] = r;
      float dot = 0.f;
      if (r >= 0)
        for (int c = 0; c < D / 8; ++c) {
          float f[8];
          load8(a.kv.key, a.kv.key_scale, r, c, f);
          for (int e = 0; e < 8; ++e) dot = fmaf(q_s[c * 8 + e], f[e], dot);
        }
      s = dot * a.scale;
    }
    float mx = warp_max(s);
    if ((x & 31) == 0) red_s[x >> 5] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red_s[0], red_s[1]), fmaxf(red_s[2], red_s[3]));
    const float mn = fmaxf(m, mx);
    const float corr = __expf(m - mn);
    const float p = i < seen ? __expf(s - mn) : 0.f;
    p_s[x] = p;
    const float ps = warp_sum(p);
    __syncthreads();
    if ((x & 31) == 0) red_s[x >> 5] = ps;
    __syncthreads();
    l = l * corr + red_s[0] + red_s[1] + red_s[2] + red_s[3];
    m = mn;
    acc *= corr;
    if (x < D) {
      const int here = min(kAttnThreads, seen - k0);
      for (int j = 0; j < here; ++j) {
        const long long r = row_s[j];
        if (r < 0) continue;
        float f[8];
        load8(sep ? a.kv.value : a.kv.key, sep ? a.kv.value_scale : a.kv.key_scale, r, x >> 3, f);
        acc = fmaf(p_s[j], f[x & 7], acc);
      }
    }
  }
  if (x < D)
    a.out[((long long)token * a.heads + h) * D + x] = __float2bfloat16_rn(seen > 0 ? acc / l : 0.f);
}

template <int D>
static int launch_attn_d(const PagedAttnArgs& a, cudaStream_t stream) {
  auto k = a.kv.key_scale != nullptr ? paged_attn_kernel<D, true> : paged_attn_kernel<D, false>;
  return launch_pdl(k, dim3(a.batch.tokens, a.heads), dim3(kAttnThreads), 0, stream, a) ==
                 cudaSuccess
             ? 0
             : -2;
}

int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t stream) {
  switch (a.kv.head_dim) {
    case 32: return launch_attn_d<32>(a, stream);
    case 64: return launch_attn_d<64>(a, stream);
    case 96: return launch_attn_d<96>(a, stream);
    case 128: return launch_attn_d<128>(a, stream);
  }
  return -1;
}

}  // namespace parrot
