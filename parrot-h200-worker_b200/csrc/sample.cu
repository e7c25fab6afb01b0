// Drawing the next token from given random numbers.
//
// For a row of logits l, temperature T, and w_i = exp((l_i - max l) / T):
//   1. the k tokens of largest w (the lower index first among equals);
//   2. of those, in that order, each whose predecessors' mass is below
//      top_p times the mass of them all;
//   3. of those, each with w_i >= min_p (the largest w is 1);
// the first token always stays.  The token drawn is the first, by index, whose
// cumulative mass over the kept set exceeds uniform times the set's mass.
//
// A draw near a border between two tokens must not depend on rounding or on
// the order of a sum, so masses are 64-bit fixed point: w in double, rounded
// once to multiples of 2^-44.  Integer sums are exact in any order, 2^19
// tokens fit 63 bits, and the 2^-45 error of a term is far below a double's
// error over a sum of that length.
#include "common.cuh"
#include "kernels.h"

namespace parrot {

namespace {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kMassBits = 44;

typedef unsigned long long u64;

// Order-preserving keys: a larger logit has a larger key; NaN and -inf, which
// are never drawn, have key 0.
__device__ __forceinline__ uint32_t key_of(__nv_bfloat16 x) {
  const uint32_t b = __bfloat16_as_ushort(x);
  if ((b & 0x7fffu) > 0x7f80u || b == 0xff80u) return 0u;
  return b & 0x8000u ? 0xffffu & ~b : (b == 0 ? 0x8000u : b | 0x8000u);
}
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u || b == 0xff800000u) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key, __nv_bfloat16) {
  const uint32_t b = key & 0x8000u ? key & 0x7fffu : 0xffffu & ~key;
  return __uint_as_float(b << 16);
}
__device__ __forceinline__ float value_of(uint32_t key, float) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// -0 and +0 are equal logits: one key for both (the negative's complement
// would be the next key below).
__device__ __forceinline__ __nv_bfloat16 plus_zero(__nv_bfloat16 x) {
  return __bfloat16_as_ushort(x) == 0x8000u ? __ushort_as_bfloat16(0) : x;
}
__device__ __forceinline__ float plus_zero(float x) { return x == 0.f ? 0.f : x; }

struct Scratch {
  u64 sum[kSampleWarps];
  u64 out;
};

__device__ __forceinline__ u64 block_sum(u64 v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = s.sum[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, Scratch& s) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, (uint32_t)s.sum[threadIdx.x & 31]);
}

// Sum over the threads before this one.
__device__ __forceinline__ u64 block_before(u64 v, Scratch& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += t;
  }
  __syncthreads();
  if (lane == 31) s.sum[warp] = in;
  __syncthreads();
  u64 w = s.sum[lane], all = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, all, o);
    if (lane >= o) all += t;
  }
  return __shfl_sync(0xffffffffu, all - w, warp) + in - v;
}

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  __shared__ Scratch s;
  __shared__ int pick_s;
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.x, V = a.vocab, x = threadIdx.x;
  const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.row_stride;
  const float temp = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  const float u = a.uniform[row];
  int k = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  // thread x holds tokens [x * per, (x + 1) * per): prefix sums by thread are
  // prefix sums by index
  const int per = (V + kSampleThreads - 1) / kSampleThreads;
  const int i0 = min(V, x * per), i1 = min(V, i0 + per);
  auto key = [&](int i) { return key_of(plus_zero(logits[i])); };

  uint32_t top = 0;
  for (int i = i0; i < i1; ++i) top = max(top, key(i));
  top = block_max(top, s);
  if (x == 0) pick_s = V;
  __syncthreads();
  auto finish = [&](int token, float logp) {
    a.ids[row] = token;
    if (a.logprobs != nullptr) a.logprobs[row] = logp;
  };
  if (top == 0) {  // every logit is -inf or NaN
    if (x == 0) finish(-1, -INFINITY);
    return;
  }
  // the lowest index among the largest logits
  for (int i = i0; i < i1; ++i)
    if (key(i) == top) {
      atomicMin(&pick_s, i);
      break;
    }
  __syncthreads();
  const int best = pick_s;
  if (!(temp > 0.f)) {  // 0 (or NaN): the largest
    if (x == 0) finish(best, 0.f);
    return;
  }
  const double top_v = value_of(top, T()), inv_t = 1.0 / (double)temp;
  auto weight = [&](uint32_t ky) {
    return ky == 0 ? 0.0 : ky == top ? 1.0 : exp(((double)value_of(ky, T()) - top_v) * inv_t);
  };
  auto mass = [&](uint32_t ky) { return (u64)__double2ll_rn(weight(ky) * (double)(1ull << kMassBits)); };

  // The kept set is {key > cut} plus the first `ties` tokens with key == cut.
  uint32_t cut = 1;
  u64 ties = (u64)V;
  // 1. top-k: the largest cut with at least k tokens at or above it
  if (k > 0 && k < V) {
    uint32_t lo = 0, hi = top;  // count(>= lo) >= k (key 0 counts everything)
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      u64 n = 0;
      for (int i = i0; i < i1; ++i) n += key(i) >= mid;
      if (block_sum(n, s) >= (u64)k) lo = mid;
      else hi = mid - 1;
    }
    if (lo > 0) {
      u64 above = 0;
      for (int i = i0; i < i1; ++i) above += key(i) > lo;
      cut = lo;
      ties = (u64)k - block_sum(above, s);
    }
  }
  // mass above a cut and count at it
  auto above_of = [&](uint32_t c) {
    u64 m = 0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t ky = key(i);
      if (ky > c) m += mass(ky);
    }
    return block_sum(m, s);
  };
  auto count_at = [&](uint32_t c) {
    u64 n = 0;
    for (int i = i0; i < i1; ++i) n += key(i) == c;
    return block_sum(n, s);
  };
  ties = min(ties, count_at(cut));
  u64 total = above_of(cut) + ties * mass(cut);
  // 2. top-p: the smallest cut whose predecessors' mass is below the share
  if (!(top_p >= 1.f)) {
    const double share = (double)top_p * (double)total;
    uint32_t lo = cut, hi = top;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((double)above_of(mid) < share) hi = mid;
      else lo = mid + 1;
    }
    const u64 f = above_of(lo), w = mass(lo);
    const u64 here = lo == cut ? ties : count_at(lo);
    // of the tokens at lo, those whose predecessors' mass f + j w is below it
    u64 a0 = 0, a1 = here;
    while (a0 < a1) {
      const u64 mid = a0 + (a1 - a0) / 2;
      if ((double)(f + mid * w) < share) a0 = mid + 1;
      else a1 = mid;
    }
    ties = max(a0, (u64)1);
    cut = lo;
  }
  // 3. min-p
  if (min_p > 0.f) {
    uint32_t lo = cut, hi = top;
    if (!((double)min_p <= 1.0)) {
      lo = top;
      if (cut < top) ties = 1;
      else ties = min(ties, (u64)1);
    } else {
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (weight(mid) >= (double)min_p) hi = mid;
        else lo = mid + 1;
      }
      if (lo > cut) ties = (u64)V;
    }
    cut = lo;
  }
  // the kept tokens of this thread, in index order
  u64 at_cut = 0;
  for (int i = i0; i < i1; ++i) at_cut += key(i) == cut;
  const u64 ties_before = block_before(at_cut, s);
  const u64 w_cut = mass(cut);
  u64 mine = 0, seen = ties_before;
  for (int i = i0; i < i1; ++i) {
    const uint32_t ky = key(i);
    if (ky > cut) mine += mass(ky);
    else if (ky == cut && seen++ < ties) mine += w_cut;
  }
  const u64 before = block_before(mine, s);
  total = block_sum(mine, s);
  const double want = (double)u * (double)total;
  u64 target = want > 0.0 ? (u64)want : 0;
  if (target >= total) target = total - 1;  // uniform must be below 1
  if (mine > 0 && before <= target && target < before + mine) {
    u64 run = before;
    seen = ties_before;
    for (int i = i0; i < i1; ++i) {
      const uint32_t ky = key(i);
      u64 w = 0;
      if (ky > cut) w = mass(ky);
      else if (ky == cut && seen++ < ties) w = w_cut;
      run += w;
      if (run > target) {
        finish(i, (float)log((double)w / (double)total));
        break;
      }
    }
  }
}

int launch_sample(const SampleArgs& a, cudaStream_t stream) {
  auto k = a.logits_f32 ? sample_kernel<float> : sample_kernel<__nv_bfloat16>;
  return launch_pdl(k, dim3(a.rows), dim3(kSampleThreads), 0, stream, a) == cudaSuccess ? 0 : -2;
}

}  // namespace parrot
