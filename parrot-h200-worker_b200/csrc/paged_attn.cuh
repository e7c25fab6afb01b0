// Device helpers shared by the two kernels of attention over the paged cache.
#pragma once

#include <atomic>

#include <algorithm>
#include <numeric>
#include <type_traits>

#include "paged.cuh"
#include "tc.cuh"

namespace parrot {

// How many clusters of `ranks` CTAs of a kernel the current device holds at once,
// asked once for each device and size: clusters of CTAs that fill an SM do not
// fill the GPU's partitions evenly (8 CTAs: fewer than a GPU's SMs / 8), and one
// cluster too many doubles a launch's time.
struct ClusterCapacity {
  std::atomic<int> plus_one[16][17];
};
template <typename K>
inline int cluster_capacity(ClusterCapacity& cache, K kernel, int threads, int smem, int ranks) {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 16 && (n = cache.plus_one[dev][ranks].load(std::memory_order_relaxed)) > 0) return n - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)ranks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (dev < 16) cache.plus_one[dev][ranks].store(n + 1, std::memory_order_relaxed);
  return n;
}

// No more tiles of `rows_per` rows than this: a sequence's rows are a multiple of
// d = gcd(group, rows_per), so its last tile wants rows_per - d at most.
inline long long most_tiles(const PagedAttnArgs& a, int rows_per) {
  const long long n = a.batch.tokens, group = a.heads / a.kv.kv_heads;
  const long long seqs = std::min<long long>(a.batch.batch, n), d = std::gcd(group, (long long)rows_per);
  return (n * group + seqs * (rows_per - d)) / rows_per;
}
// No more keys in sight of a tile of `rows` rows than this.
inline long long most_keys(const PagedAttnArgs& a, int rows, int step) {
  const long long keys = (long long)a.batch.table_width << a.kv.page_shift;
  const long long tokens = rows / (a.heads / a.kv.kv_heads) + 1;
  return a.window > 0 ? std::min(keys, (long long)a.window + a.sinks + tokens + 2 * step) : keys;
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four numbers of the output, from element `at` on.
template <bool F32>
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, long long at, float4 v) {
  if constexpr (F32)
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint2(tc::pack_bf16x2(v.x, v.y), tc::pack_bf16x2(v.z, v.w));
}

// 1 / sum of the weights of a row at position `pos`.  A row before the first
// position sees no key: zeros.  One that sees keys of weight 0 alone (scores of
// -infinity) has 0 / 0: NaN.
__device__ __forceinline__ float row_inverse(float sum, int pos) {
  return sum != 0.f ? 1.f / sum : pos < 0 ? 0.f : __uint_as_float(0x7fffffffu);
}

// A pair as two pairs of bf16, high parts and what they leave, together 2^-16 of
// each number or better.
struct Bf16Pairs {
  uint32_t hi, lo;
};
// Of probabilities: both parts rounded to nearest.
__device__ __forceinline__ Bf16Pairs split_weights(float x, float y) {
  Bf16Pairs p;
  p.hi = tc::pack_bf16x2(x, y);
  const float2 h = bf16x2_to_float2(p.hi);
  p.lo = tc::pack_bf16x2(x - h.x, y - h.y);
  return p;
}
// Of queries: the high part cut off, so that the low part has its sign, and a low
// part that would be zero 2^-24 of the high one.  An infinite key then gives both
// products the same infinity, as it would give the number itself; zero stays zero.
__device__ __forceinline__ float query_high(float x) {
  const uint32_t b = __float_as_uint(x);
  return x != x ? x : __uint_as_float(b & 0xffff0000u);
}
__device__ __forceinline__ float query_low(float x, float high) {
  const float rest = x - high;
  return rest != 0.f && fabsf(high) < INFINITY ? rest : high * 5.9604644775390625e-08f;
}
__device__ __forceinline__ Bf16Pairs split_queries(float x, float y) {
  const float hx = query_high(x), hy = query_high(y);
  Bf16Pairs p;
  p.hi = tc::pack_bf16x2(hx, hy);
  p.lo = tc::pack_bf16x2(query_low(x, hx), query_low(y, hy));
  return p;
}

// A tile: `rows_per` consecutive (token, head) rows of one sequence.
struct Tile {
  int b;           // sequence, -1: no such tile
  int first;       // batch row of the sequence's first token
  int n;           // its tokens in the batch
  int row0;        // first (token, head) row of the tile
  int ctx;         // its context length, as given
};

// Rows of a tile as tokens and heads of the group: one division a tile, and for
// a row a product with the reciprocal, exact for so small numbers.
struct RowMap {
  int group, token0, rest;
  float inverse;
  __device__ __forceinline__ RowMap(int row0, int g) : group(g) {
    token0 = row0 / g;
    rest = row0 - token0 * g;
    inverse = 1.f / (float)g;
  }
  // (token of the sequence's rows, head of the group) of row r of the tile, r < 4096
  __device__ __forceinline__ int2 operator()(int r) const {
    const int x = rest + r, q = (int)(((float)x + 0.5f) * inverse);
    return make_int2(token0 + q, x - q * group);
  }
};

// The tile with this number, sequences in order, ceil(n_b * group / rows_per)
// tiles each (tokens * heads fits 31 bits).  A whole warp calls; 32 sequences a step, their lengths loaded
// side by side.
__device__ __forceinline__ Tile find_tile(const PagedBatch& s, int group, int rows_per, int tile) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < s.batch; b0 += 32) {
    const int b = b0 + lane;
    int2 r = make_int2(0, 0);
    if (b < s.batch) r = batch_rows(s, b);
    const int n = r.y - r.x, len = b < s.batch ? s.context_len[b] : 0;
    const int mine = (int)(((unsigned)(n * group) + rows_per - 1) / rows_per);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + upto > tile);
    if (hit) {
      const int l = __ffs(hit) - 1;
      Tile t;
      t.b = b0 + l;
      t.first = __shfl_sync(0xffffffffu, r.x, l);
      t.n = __shfl_sync(0xffffffffu, n, l);
      t.ctx = __shfl_sync(0xffffffffu, len, l);
      t.row0 = (tile - base - __shfl_sync(0xffffffffu, upto - mine, l)) * rows_per;
      return t;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Tile{-1, 0, 0, 0, 0};
}

// As find_tile with the sequences' tiles taken from their ends in turn: all
// last tiles first, which see the most keys, then those before them, so that
// what is left to the end of the launch is short.  Up to 32 sequences (above,
// no tile is a large part of the work, and the order is find_tile's reversed).
__device__ __forceinline__ Tile find_tile_from_ends(const PagedBatch& s, int group, int rows_per,
                                                    int index, int most) {
  if (s.batch > 32) return find_tile(s, group, rows_per, most - 1 - index);
  const int lane = threadIdx.x & 31;
  int2 r = make_int2(0, 0);
  int len = 0;
  if (lane < s.batch) {
    r = batch_rows(s, lane);
    len = s.context_len[lane];
  }
  const int n = r.y - r.x;
  const int tiles = (int)(((unsigned)(n * group) + rows_per - 1) / rows_per);
  if (index >= (int)__reduce_add_sync(0xffffffffu, (unsigned)tiles)) return Tile{-1, 0, 0, 0, 0};
  // the round: the last one before which at most `index` tiles were taken
  int lo = 0, hi = (int)__reduce_max_sync(0xffffffffu, (unsigned)tiles);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((int)__reduce_add_sync(0xffffffffu, (unsigned)min(tiles, mid)) <= index) lo = mid;
    else hi = mid;
  }
  const int left = index - (int)__reduce_add_sync(0xffffffffu, (unsigned)min(tiles, lo));
  const unsigned open = __ballot_sync(0xffffffffu, tiles > lo);
  const unsigned before = open & ((1u << lane) - 1u);
  const unsigned hit = __ballot_sync(0xffffffffu, (open >> lane & 1) && __popc(before) == left);
  const int l = __ffs(hit) - 1;
  Tile t;
  t.b = l;
  t.first = __shfl_sync(0xffffffffu, r.x, l);
  t.n = __shfl_sync(0xffffffffu, n, l);
  t.ctx = __shfl_sync(0xffffffffu, len, l);
  t.row0 = (__shfl_sync(0xffffffffu, tiles, l) - 1 - lo) * rows_per;
  return t;
}

// This CTA's place in its cluster, the cluster's in the grid, and their number:
// what divisions of blockIdx.x would give.
struct ClusterPlace {
  int rank, index, count;
};
__device__ __forceinline__ ClusterPlace cluster_place() {
  ClusterPlace c;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(c.rank));
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(c.index));
  asm("mov.u32 %0, %%nclusterid.x;" : "=r"(c.count));
  return c;
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t mapa_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

}  // namespace parrot
