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
// A draw near a border between two tokens must not depend on the order of a
// sum, so masses are 64-bit fixed point: w in double, rounded once to multiples of
// 2^-44.  Integer sums are exact in any order, and the masses of 2^19 tokens (2^63
// at most) fit.  A mass is off by at most 2^-45 of the largest, so a border by at
// most vocab * 2^-45: 2^-30 for 32,768 tokens and 2^-26 for 2^19, below the 2^-24
// of an fp32 uniform.  Over a long flat tail these errors have one sign: a token of
// w <= 2^-45 has no mass at all and is never drawn.
//
// A cluster of CTAs shares a row (one CTA where the rows fill the GPU).  The
// logits become order-preserving integer keys in shared memory, read from HBM
// once.  A filter cuts that order at one place: a histogram of the keys over
// 512 equal steps of max l - l (counts for top-k, exact masses for
// top-p), summed from the top, names the step that the cut falls into; the few
// keys of that step are collected in the first CTA, where one warp bisects them
// for the key and how many of its equals stay.  The draw needs each warp's
// kept mass, then one warp walks its part of the row.  CTAs exchange sums and
// histograms over distributed shared memory.  Bound by the latency of the steps (a
// cluster meets four to ten times) and by the instructions of the exponentials in
// double (two per logit under top-p).  Measured at 32,768 logits: one row with
// top-p 20.6 us, 64 rows of mixed settings 35 us (17 without filters), 256 rows 80.
#include <algorithm>

#include "kernels.h"
#include "tc.cuh"

namespace parrot {

namespace {

constexpr int kSampleThreads = 512;
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

constexpr int kSampleMaxRanks = 8;
constexpr int kBins = 512;       // equal steps below the largest logit, one a thread
constexpr int kList = 2048;      // keys of one step collected
constexpr int kSteps = 128;      // table of 2^(j / 128)
constexpr int kSampleFixed = 2 * kBins * 4 + kList * 12 + kSteps * 8;
constexpr int kSampleStaged = 190464;  // most bytes of keys in shared memory
static_assert(kBins == kSampleThreads, "a thread sums one step over the cluster");

struct Scratch {
  u64 sum[kSampleWarps], eq[kSampleWarps];  // of this CTA's warps
  u64 xch[2][2][kSampleMaxRanks];           // one pair from each CTA, two exchanges deep
  u64 above;
  u64 ties;
  uint32_t cut;
  int bin, listed, pick;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t atom_cluster_inc(uint32_t addr) {
  uint32_t old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;"
               : "=r"(old)
               : "r"(addr)
               : "memory");
  return old;
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_upto(u64 v, int lane) {  // inclusive prefix sum
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

__device__ __forceinline__ u64 block_sum(u64 v, Scratch& s) {
  v = warp_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum_u64((threadIdx.x & 31) < kSampleWarps ? s.sum[threadIdx.x & 31] : 0);
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, Scratch& s) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.sum[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < kSampleWarps ? (uint32_t)s.sum[threadIdx.x & 31] : 0u);
}

// Sum over the threads before this one.
__device__ __forceinline__ u64 block_before(u64 v, Scratch& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 in = warp_upto(v, lane);
  __syncthreads();
  if (lane == 31) s.sum[warp] = in;
  __syncthreads();
  const u64 w = lane < kSampleWarps ? s.sum[lane] : 0;
  return __shfl_sync(0xffffffffu, warp_upto(w, lane) - w, warp) + in - v;
}

// Every CTA of the cluster gives a pair (the same in all its threads); after
// it, s.xch[turn] holds all of them, and what the CTAs wrote before it is
// visible to each other.  Two exchanges may be under way: the pairs alternate.
struct Exchange {
  int ranks, rank, turn;
  __device__ __forceinline__ void operator()(u64 v0, u64 v1, Scratch& s) {
    turn ^= 1;
    if (ranks == 1) {
      if (threadIdx.x == 0) {
        s.xch[turn][0][0] = v0;
        s.xch[turn][1][0] = v1;
      }
      __syncthreads();
      return;
    }
    if (threadIdx.x < ranks) {
      st_cluster_u64(tc::mapa_shared(&s.xch[turn][0][rank], threadIdx.x), v0);
      st_cluster_u64(tc::mapa_shared(&s.xch[turn][1][rank], threadIdx.x), v1);
    }
    __syncwarp();
    tc::cluster_sync();
  }
  __device__ __forceinline__ u64 sum(int which, const Scratch& s) const {
    u64 t = 0;
    for (int r = 0; r < ranks; ++r) t += s.xch[turn][which][r];
    return t;
  }
};

template <typename T>
struct KeyType;
template <>
struct KeyType<__nv_bfloat16> {
  typedef uint16_t type;
};
template <>
struct KeyType<float> {
  typedef uint32_t type;
};

}  // namespace

template <typename T, int PER_SM>
__global__ void __launch_bounds__(kSampleThreads, PER_SM) sample_kernel(SampleArgs a) {
  typedef typename KeyType<T>::type Key;
  constexpr int N = 16 / sizeof(T);  // logits, or keys, of a 16-byte vector
  __shared__ Scratch s;
  extern __shared__ __align__(16) unsigned char sample_smem[];
  uint32_t* hist_lo = reinterpret_cast<uint32_t*>(sample_smem);
  uint32_t* hist_hi = hist_lo + kBins;
  u64* list_mass = reinterpret_cast<u64*>(hist_hi + kBins);
  uint32_t* list_key = reinterpret_cast<uint32_t*>(list_mass + kList);
  double* pow_s = reinterpret_cast<double*>(list_key + kList);
  uint4* keys = reinterpret_cast<uint4*>(sample_smem + kSampleFixed);
  const int x = threadIdx.x, warp = x >> 5, lane = x & 31;
  if (x < kSteps) pow_s[x] = exp2((double)x / kSteps);
  griddep_wait();
  griddep_launch();
  Exchange exchange{a.cluster, (int)(blockIdx.x % a.cluster), 0};
  // arrive now, wait before the first access: every CTA of the cluster has started
  if (exchange.ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int ranks = exchange.ranks, rank = exchange.rank;
  const int row = blockIdx.x / ranks, V = a.vocab;
  const T* logits = static_cast<const T*>(a.logits) + (long long)row * a.row_stride;
  const float temp = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  const float u = a.uniform[row];
  const int k = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  const bool aligned = (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  // CTA r holds the vectors [r of_cta, (r + 1) of_cta) of the row, its warps
  // equal runs of them in order, the lanes of a warp side by side
  const int vecs = (V + N - 1) / N;
  const int of_cta = (vecs + ranks - 1) / ranks;
  const bool staged = of_cta * 16 <= kSampleStaged;
  const int cta0 = min(vecs, rank * of_cta), cta1 = min(vecs, cta0 + of_cta);
  const int per = (of_cta + kSampleWarps - 1) / kSampleWarps;
  const int v0 = min(cta1, cta0 + warp * per), v1 = min(cta1, v0 + per);

  // the keys of vector v, key 0 behind the row's end
  auto fetch = [&](int v, uint32_t (&ky)[N]) {
    if (aligned && v * N + N <= V) {
      const uint4 w = reinterpret_cast<const uint4*>(logits)[v];
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int i = 0; i < N; ++i) ky[i] = key_of(plus_zero(e[i]));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) ky[i] = v * N + i < V ? key_of(plus_zero(logits[v * N + i])) : 0u;
    }
  };
  auto load = [&](int v, uint32_t (&ky)[N]) {
    if (staged) {
      const uint4 w = keys[v - cta0];
      const Key* e = reinterpret_cast<const Key*>(&w);
#pragma unroll
      for (int i = 0; i < N; ++i) ky[i] = e[i];
    } else {
      fetch(v, ky);
    }
  };

  uint32_t top = 0, low = 0xffffffffu;  // the largest key, and the least but 0
  auto take = [&](int v, const uint32_t (&ky)[N]) {
    if (staged) {
      uint4 w;
      Key* e = reinterpret_cast<Key*>(&w);
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = (Key)ky[i];
      keys[v - cta0] = w;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      top = max(top, ky[i]);
      low = min(low, ky[i] - 1);  // key 0 wraps round
    }
  };
  int v = v0 + lane;
  if (aligned) {  // four vectors on their way at once
    for (; v + 96 < v1 && (v + 97) * N <= V; v += 128) {
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const uint4*>(logits)[v + 32 * j];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T* e = reinterpret_cast<const T*>(&w[j]);
        uint32_t ky[N];
#pragma unroll
        for (int i = 0; i < N; ++i) ky[i] = key_of(plus_zero(e[i]));
        take(v + 32 * j, ky);
      }
    }
  }
  for (; v < v1; v += 32) {
    uint32_t ky[N];
    fetch(v, ky);
    take(v, ky);
  }
  if (x == 0) s.pick = V;
  top = block_max(top, s);
  low = block_max(~low, s);
  if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  exchange(top, low, s);
  top = low = 0;
  for (int r = 0; r < ranks; ++r) {
    top = max(top, (uint32_t)s.xch[exchange.turn][0][r]);
    low = max(low, (uint32_t)s.xch[exchange.turn][1][r]);
  }
  low = ~low + 1;
  auto finish = [&](int token, float logp) {
    a.ids[row] = token;
    if (a.logprobs != nullptr) a.logprobs[row] = logp;
  };
  if (top == 0) {  // every logit is -inf or NaN
    if (x == 0 && rank == 0) finish(-1, -INFINITY);
    return;
  }
  if (!(temp > 0.f)) {  // 0 (or NaN): the lowest index among the largest logits
    for (int v = v0 + lane; v < v1; v += 32) {
      uint32_t ky[N];
      load(v, ky);
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (ky[i] == top) atomicMin(&s.pick, v * N + i);
    }
    __syncthreads();
    exchange(s.pick, 0, s);
    if (x == 0 && rank == 0) {
      int best = V;
      for (int r = 0; r < ranks; ++r) best = min(best, (int)s.xch[exchange.turn][0][r]);
      finish(best, 0.f);
    }
    return;
  }
  const float top_v = value_of(top, T());
  // mass(key) = 2^44 2^(y / 128), y = 128 log2(e) (l - max l) / T, in double:
  // y = n + r with n whole and |r| <= 1/2, 2^(n / 128) from the table and an
  // exponent, 2^(r / 128) = sum (r ln2 / 128)^k / k! to k = 4 (the rest is below
  // 2^-49), rounded once to a whole number.  Whole parts are read off the low
  // bits of a sum with 1.5 2^52, and the logit is widened by its bits: the
  // conversion instructions run at a quarter of the products' rate.
  const double rate = 128.0 * 1.4426950408889634 / (double)temp;
  const double top_y = (double)top_v * rate;
  // No branches, so that a thread's keys are worked on side by side.
  auto mass = [&](uint32_t ky) -> u64 {
    const uint32_t b = __float_as_uint(value_of(ky, T()));
    const bool tiny = (b & 0x7f800000u) == 0;  // below 2^-126: as zero
    const uint32_t hi = (b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + (896u << 20));
    const double v = __hiloint2double(tiny ? 0u : hi, tiny ? 0u : b << 29);
    const double y = fma(v, rate, -top_y);
    const bool some = y >= -7680.0;  // else below 2^-60, or an infinite logit above all others
    constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
    const double n = y + kWhole;
    const int whole = __double2loint(n);
    const double r = y - (n - kWhole);
    constexpr double c1 = 0.0054152123481245727;  // ln2 / 128, and its powers over k!
    constexpr double c2 = c1 * c1 / 2, c3 = c1 * c2 / 3, c4 = c1 * c3 / 4;
    const double p = fma(fma(fma(fma(c4, r, c3), r, c2), r, c1), r, 1.0) * pow_s[whole & (kSteps - 1)];
    // times 2^(44 + whole / 128), then rounded by the sum with 2^52
    const double w = __hiloint2double(__double2hiint(p) + ((kMassBits + (whole >> 7)) << 20), __double2loint(p));
    const u64 m = (u64)__double_as_longlong(w + 4503599627370496.0) & ((1ull << 52) - 1);
    return ky == top ? 1ull << kMassBits : some && ky != 0 ? m : 0;
  };
  // equal steps over the row's range, at least 8 an octave of probability (64
  // octaves down no mass is left); not increasing in the key
  const float step = fminf(fmaxf((kBins / 64) * 1.44269504f / temp,
                                 (float)(kBins - 1) / (top_v - value_of(low, T()))), 1e30f);
  auto bin_of = [&](uint32_t ky) {
    const float d = (top_v - value_of(ky, T())) * step;
    return ky == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;
  };
  // f(key) for every key of this thread
  auto each = [&](auto f) {
    for (int v = v0 + lane; v < v1; v += 32) {
      uint32_t ky[N];
      load(v, ky);
#pragma unroll
      for (int i = 0; i < N; ++i) f(ky[i]);
    }
  };
  // f(keys of 32 lanes) for each element whose test holds in some lane: after a
  // filter few do, and the rest need no exponentials
  auto each_where = [&](auto test, auto f) {
    for (int v = v0 + lane; v - lane < v1; v += 32) {
      uint32_t ky[N];
#pragma unroll
      for (int i = 0; i < N; ++i) ky[i] = 0;
      if (v < v1) load(v, ky);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (__any_sync(0xffffffffu, test(ky[i]))) f(ky[i]);
    }
  };
  auto clear_hist = [&]() {
    __syncthreads();
    for (int i = x; i < 2 * kBins; i += kSampleThreads) hist_lo[i] = 0;
    if (x == 0) {
      s.listed = 0;
      s.bin = kBins - 1;
    }
    __syncthreads();
  };
  // this thread's step of the cluster's histogram
  auto merged = [&](bool wide) {
    u64 c = 0;
    for (int r = 0; r < ranks; ++r) {
      c += ld_cluster_u32(tc::mapa_shared(hist_lo + x, r));
      if (wide) c += (u64)ld_cluster_u32(tc::mapa_shared(hist_hi + x, r)) << 32;
    }
    return c;
  };
  // s.bin: the first bin whose inclusive sum from bin 0 satisfies `reaches`;
  // s.above: the sum before it.  c: the content of bin x.
  auto find_bin = [&](u64 c, auto reaches) {
    const u64 at = block_before(c, s);
    if (!reaches(at) && reaches(at + c)) {
      s.bin = x;
      s.above = at;
    }
    __syncthreads();
  };
  // The keys of a step: bin_of does not increase with the key, so they are a
  // range, found by 32 lanes trying 32 keys at a time.
  auto last_key = [&](int bin) {  // the largest key with bin_of(key) >= bin, at least `low`
    uint32_t lo = low, hi = top;
    while (lo < hi) {
      const uint32_t part = (hi - lo) / 32 + 1;
      const uint32_t ky = lo + part * (lane + 1);
      const unsigned in = __ballot_sync(0xffffffffu, ky <= hi && ky > lo && bin_of(ky) >= bin);
      const uint32_t n = __popc(in);  // a run of the first lanes
      hi = min(hi, lo + part * (n + 1) - 1);
      lo = lo + part * n;
    }
    return lo;
  };
  // the cluster's keys of s.bin above `floor_key` to the first CTA's list
  auto make_list = [&](uint32_t floor_key, bool with_mass) {
    const int bin = s.bin;
    uint32_t from = bin + 1 < kBins ? last_key(bin + 1) : low - 1;
    if (bin + 1 < kBins && from == low && bin_of(low) <= bin) from = low - 1;
    from = max(from, floor_key);
    const uint32_t upto = last_key(bin);
    const uint32_t count = tc::mapa_shared(&s.listed, 0);
    const uint32_t key_at = tc::mapa_shared(list_key, 0), mass_at = tc::mapa_shared(list_mass, 0);
    each([&](uint32_t ky) {
      if (ky > from && ky <= upto) {
        const uint32_t at = atom_cluster_inc(count);
        if (at < kList) {
          st_cluster_u32(key_at + at * 4, ky);
          if (with_mass) st_cluster_u64(mass_at + at * 8, mass(ky));
        }
      }
    });
  };
  // The first CTA's first warp gives everyone its cut.
  auto publish = [&](uint32_t cut, u64 ties) {
    if (lane < ranks) {
      st_cluster_u32(tc::mapa_shared(&s.cut, lane), cut);
      st_cluster_u64(tc::mapa_shared(&s.ties, lane), ties);
    }
  };

  // The kept set is {key > cut} plus the first `ties` tokens with key == cut.
  uint32_t cut = 1;
  u64 ties = (u64)V;
  // 1. top-k
  if (k > 0 && k < V) {
    clear_hist();
    each([&](uint32_t ky) {
      if (ky != 0) atomicAdd(&hist_lo[bin_of(ky)], 1u);
    });
    exchange(0, 0, s);
    const u64 c = merged(false);
    if (block_sum(c, s) > (u64)k) {
      find_bin(c, [&](u64 n) { return n >= (u64)k; });
      const u64 want = (u64)k - s.above;  // tokens of s.bin, at least one
      const int bin = s.bin;
      make_list(0, false);
      exchange(0, 0, s);
      const uint32_t listed = ld_cluster_u32(tc::mapa_shared(&s.listed, 0));
      if (listed <= kList) {
        if (rank == 0 && warp == 0) {
          auto count = [&](uint32_t from) {  // listed keys at or above `from`
            uint32_t c = 0;
            for (uint32_t i = lane; i < listed; i += 32) c += list_key[i] >= from;
            return __reduce_add_sync(0xffffffffu, c);
          };
          uint32_t least = 0xffffffffu, most = 0;
          for (uint32_t i = lane; i < listed; i += 32) {
            least = min(least, list_key[i]);
            most = max(most, list_key[i]);
          }
          // the largest key with `want` keys at or above it
          uint32_t lo = __reduce_min_sync(0xffffffffu, least), hi = __reduce_max_sync(0xffffffffu, most);
          while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            if (count(mid) >= want) lo = mid;
            else hi = mid - 1;
          }
          publish(lo, want - (lo == 0xffffffffu ? 0 : count(lo + 1)));
        }
        exchange(0, 0, s);
        cut = s.cut;
        ties = s.ties;
      } else {
        // many near-equal logits: the same bisection over the whole row
        auto count = [&](uint32_t from) {
          u64 c = 0;
          each([&](uint32_t ky) { c += ky >= from && ky != 0 && bin_of(ky) == bin; });
          exchange(block_sum(c, s), 0, s);
          return exchange.sum(0, s);
        };
        uint32_t lo = 1, hi = top;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          if (count(mid) >= want) lo = mid;
          else hi = mid - 1;
        }
        cut = lo;
        ties = want - (lo == 0xffffffffu ? 0 : count(lo + 1));
      }
    }
  }
  // 2. top-p: the smallest key whose predecessors' mass is below the share
  if (!(top_p >= 1.f)) {
    if (k > 0 && k < V) exchange(0, 0, s);  // the histograms and the list have been read
    clear_hist();
    u64 at_cut = 0;
    auto add = [&](uint32_t ky, u64 w) {
      const uint32_t lo = (uint32_t)w;
      const int bin = bin_of(ky);
      const uint32_t old = atomicAdd(&hist_lo[bin], lo);
      const uint32_t up = (uint32_t)(w >> 32) + (old + lo < lo ? 1u : 0u);
      if (up) atomicAdd(&hist_hi[bin], up);
    };
    if (cut > 1) {
      each_where([&](uint32_t ky) { return ky >= cut; }, [&](uint32_t ky) {
        const u64 w = mass(ky);
        if (ky > cut) add(ky, w);
        at_cut += ky == cut;
      });
    } else {
      for (int v = v0 + lane; v < v1; v += 32) {
        uint32_t ky[N];
        u64 w[N];
        load(v, ky);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = mass(ky[i]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (ky[i] > cut && w[i] != 0) add(ky[i], w[i]);
          at_cut += ky[i] == cut;
        }
      }
    }
    exchange(block_sum(at_cut, s), 0, s);
    at_cut = min(exchange.sum(0, s), ties);
    const u64 w_cut = at_cut > 0 ? mass(cut) : 0;
    u64 c = merged(true);
    if (at_cut > 0 && x == bin_of(cut)) c += at_cut * w_cut;
    const double share = (double)top_p * (double)block_sum(c, s);
    if (!(share > 0.0)) {
      cut = top;
      ties = 1;
    } else {
      find_bin(c, [&](u64 m) { return !((double)m < share); });
      const u64 above = s.above;
      const int bin = s.bin;
      const uint32_t floor_key = cut;
      make_list(floor_key, true);
      exchange(0, 0, s);
      const uint32_t listed = ld_cluster_u32(tc::mapa_shared(&s.listed, 0));
      // of `here` tokens of mass w, those whose predecessors' mass f + j w is
      // below the share
      auto stay = [&](u64 f, u64 w, u64 here) {
        u64 a0 = 0, a1 = here;
        while (a0 < a1) {
          const u64 mid = a0 + (a1 - a0) / 2;
          if ((double)(f + mid * w) < share) a0 = mid + 1;
          else a1 = mid;
        }
        return max(a0, (u64)1);
      };
      if (listed <= kList) {
        if (rank == 0 && warp == 0) {
          auto above_of = [&](uint32_t cc) {  // mass of the keys above cc, cc in the bin or below
            u64 m = 0;
            for (uint32_t i = lane; i < listed; i += 32)
              if (list_key[i] > cc) m += list_mass[i];
            return above + warp_sum_u64(m);
          };
          uint32_t least = 0xffffffffu, most = floor_key;
          for (uint32_t i = lane; i < listed; i += 32) {
            least = min(least, list_key[i]);
            most = max(most, list_key[i]);
          }
          least = __reduce_min_sync(0xffffffffu, least);
          most = __reduce_max_sync(0xffffffffu, most);
          uint32_t lo = floor_key, hi = floor_key;  // if all listed keys stay, the cut is the old one
          if (listed > 0 && !((double)above_of(least - 1) < share)) {
            lo = least;
            hi = most;
          }
          while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if ((double)above_of(mid) < share) hi = mid;
            else lo = mid + 1;
          }
          uint32_t here = 0;
          for (uint32_t i = lane; i < listed; i += 32) here += list_key[i] == lo;
          here = __reduce_add_sync(0xffffffffu, here);
          publish(lo, stay(above_of(lo), mass(lo), lo > floor_key ? (u64)here : at_cut));
        }
        exchange(0, 0, s);
        cut = s.cut;
        ties = s.ties;
      } else {
        auto above_of = [&](uint32_t cc) {
          u64 m = 0;
          each([&](uint32_t ky) {
            if (ky > cc && ky > floor_key && bin_of(ky) == bin) m += mass(ky);
          });
          exchange(block_sum(m, s), 0, s);
          return above + exchange.sum(0, s);
        };
        uint32_t lo = floor_key, hi = top;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo) / 2;
          if ((double)above_of(mid) < share) hi = mid;
          else lo = mid + 1;
        }
        const u64 f = above_of(lo);
        u64 here = 0;
        each([&](uint32_t ky) { here += ky == lo; });
        exchange(block_sum(here, s), 0, s);
        cut = lo;
        ties = stay(f, mass(lo), lo > floor_key ? exchange.sum(0, s) : at_cut);
      }
    }
  }
  // 3. min-p is a test of each mass; above 1 it leaves the first token alone
  if (min_p > 1.f) {
    ties = cut == top ? min(ties, (u64)1) : 1;
    cut = top;
  }
  const u64 least = min_p > 0.f && min_p <= 1.f
                        ? (u64)__double2ll_rn((double)min_p * (double)(1ull << kMassBits))
                        : 0;
  auto kept = [&](uint32_t ky) {  // mass of a token above the cut
    const u64 w = mass(ky);
    return w >= least ? w : 0;
  };
  const u64 w_cut = kept(cut);

  // each warp's kept mass: of the tokens at the cut, the first `ties` by index
  u64 mine = 0, eq = 0;
  if (cut > 1) {
    each_where([&](uint32_t ky) { return ky >= cut; }, [&](uint32_t ky) {
      const u64 w = kept(ky);
      mine += ky > cut ? w : 0;
      eq += ky == cut;
    });
  } else {
    each([&](uint32_t ky) {
      const u64 w = kept(ky);
      mine += ky > cut ? w : 0;
      eq += ky == cut;
    });
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mine += __shfl_xor_sync(0xffffffffu, mine, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  __syncthreads();
  if (lane == 0) {
    s.sum[warp] = mine;
    s.eq[warp] = eq;
  }
  __syncthreads();
  const u64 eq_w = lane < kSampleWarps ? s.eq[lane] : 0;
  const u64 above_w = lane < kSampleWarps ? s.sum[lane] : 0;
  exchange(warp_sum_u64(above_w), warp_sum_u64(eq_w), s);
  u64 total = 0, base = 0, eq_base = 0, eq_all = 0;
  for (int r = 0; r < ranks; ++r) {
    const u64 e = s.xch[exchange.turn][1][r];
    const u64 m = s.xch[exchange.turn][0][r] + min(ties > eq_all ? ties - eq_all : 0, e) * w_cut;
    if (r < rank) {
      base += m;
      eq_base += e;
    }
    total += m;
    eq_all += e;
  }
  const double want = (double)u * (double)total;
  u64 target = want > 0.0 ? (u64)want : 0;
  if (target >= total) target = total - 1;  // uniform belongs below 1
  const u64 eq_before_w = eq_base + warp_upto(eq_w, lane) - eq_w;
  const u64 sum_w = above_w + min(eq_before_w < ties ? ties - eq_before_w : 0, eq_w) * w_cut;
  const u64 upto_w = base + warp_upto(sum_w, lane);
  const unsigned past = __ballot_sync(0xffffffffu, lane < kSampleWarps && upto_w > target);
  if (target < base || warp != __ffs(past) - 1) return;
  // the drawn token is in this warp's part; its logarithm by (l - max l) / T, which
  // needs no second logarithm
  const double log_total = log((double)total * (1.0 / (double)(1ull << kMassBits)));
  auto log_mass = [&](uint32_t ky) {
    return ky == top ? 0.0 : ((double)value_of(ky, T()) - (double)top_v) / (double)temp;
  };
  u64 run = __shfl_sync(0xffffffffu, upto_w - sum_w, warp);
  u64 eq_run = __shfl_sync(0xffffffffu, eq_before_w, warp);
  for (int vb = v0; vb < v1; vb += 32) {
    const int v = vb + lane;
    uint32_t ky[N];
#pragma unroll
    for (int i = 0; i < N; ++i) ky[i] = 0;
    if (v < v1) load(v, ky);
    u64 n_eq = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n_eq += ky[i] == cut;
    const u64 eq_upto = warp_upto(n_eq, lane);
    u64 at = eq_run + eq_upto - n_eq;  // equals before this vector
    u64 w[N], sum = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u64 m = kept(ky[i]);
      w[i] = ky[i] > cut ? m : ky[i] == cut && at < ties ? w_cut : 0;
      at += ky[i] == cut;
      sum += w[i];
    }
    const u64 upto = warp_upto(sum, lane);
    u64 r = run + upto - sum;
    if (r <= target && target < run + upto) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (r <= target && target < r + w[i])
          finish(v * N + i, (float)(log_mass(ky[i]) - log_total));
        r += w[i];
      }
    }
    run += __shfl_sync(0xffffffffu, upto, 31);
    eq_run += __shfl_sync(0xffffffffu, eq_upto, 31);
    if (run > target) break;
  }
}

// CTAs per row: as many as leave each thread a vector while all rows' CTAs
// are resident at once, `per_sm` on an SM.
static int sample_ranks(int rows, int vecs, int sms, int per_sm) {
  int ranks = 1;
  while (ranks < kSampleMaxRanks && vecs >= 2 * ranks * kSampleThreads &&
         2LL * ranks * rows <= (long long)per_sm * sms)
    ranks *= 2;
  return ranks;
}

// One CTA an SM has 110 registers a thread, two have 64: with few rows the
// latency of each step counts (32 rows of 32,768: 28.8 us with one, 30.5 with
// two), with rows for a quarter of the SMs the second CTA's warps cover it (64
// rows: 37.7 and 35.0 us; 256: 91.6 and 80.3).  Rows of less than two vectors
// a thread gain nothing (64 of 4096: 19.9 and 20.6).
static bool sample_two_per_sm(int rows, int vecs, int sms) {
  return 4LL * rows > sms && vecs >= 2 * kSampleThreads;
}

template <typename T, int PER_SM>
static int launch_sample_t(SampleArgs a, int vecs, int sms, cudaStream_t stream) {
  a.cluster = sample_ranks(a.rows, vecs, sms, PER_SM);
  if ((long long)a.rows * a.cluster > 0x7fffffffll) return -2;
  const int bytes = (vecs + a.cluster - 1) / a.cluster * 16;
  const int smem = kSampleFixed + (bytes <= kSampleStaged ? bytes : 0);
  static std::atomic<unsigned long long> done{0};
  if (!once_per_device(done, [&] { return allow_shared(sample_kernel<T, PER_SM>, kSampleFixed + kSampleStaged); }))
    return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * a.cluster));
  cfg.blockDim = dim3(kSampleThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)a.cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, PER_SM>, a) == cudaSuccess ? 0 : -2;
}

template <typename T>
static int launch_sample_of(const SampleArgs& a, int sms, cudaStream_t stream) {
  const int n = 16 / (int)sizeof(T);
  const int vecs = (a.vocab + n - 1) / n;
  return sample_two_per_sm(a.rows, vecs, sms) ? launch_sample_t<T, 2>(a, vecs, sms, stream)
                                              : launch_sample_t<T, 1>(a, vecs, sms, stream);
}

int launch_sample(const SampleArgs& a, int sms, cudaStream_t stream) {
  return a.logits_f32 ? launch_sample_of<float>(a, sms, stream)
                      : launch_sample_of<__nv_bfloat16>(a, sms, stream);
}

}  // namespace parrot
