// Attention of many queries per sequence over the paged cache: the tensor-core
// kernel behind launch_paged_attention (paged_attn.cu states the formula and
// takes the batches of few queries).
//
// A CTA takes 384 (token, head) rows of one sequence and key head in three groups
// of 128 (head width 128: 256 rows in two), and streams the keys they see in
// tiles of 64 (128):
//   S_g = Q_g K^T (tcgen05, both operands in shared memory, S in TMEM),
//   one thread per row: running maximum, p = 2^(s - m), P in bf16 back into
//   TMEM over S, O_g += P_g V (tcgen05, P from TMEM, V from shared memory).
// A group's threads wait for its two products, about a third of its time; the
// other groups' exponentials (16 a clock and SM) and products fill it.  TMEM
// holds three groups of S and O up to width 96.  A row's maximum m is only moved
// when it grows by more than 2^8 (p then stays below 2^8, and O and the sum are
// fp32), so O is rarely rescaled.  The sum is of the unrounded p.
// Measured (8 heads on 2, width 96, a window of 2048): four prompts of 4096 in 116
// us, 660 TFLOP/s of what the mask leaves, the exponential unit busy for half of
// the time and the tensor cores for 36%; what is left is the wait of a group for
// its products and the start and end of a tile.  Slower on the same prompts: two
// groups with tiles of 128 keys (135 us); with P in shared memory (its reads and
// Q's fill shared memory's bandwidth: 151 us); with 96 keys, P apart from S and the
// next scores computed early (152 us); with steps of 64 keys over two S blocks a
// group (146 us); with two threads a row (145 us); with the maximum taken a tile
// late (126 us).
//
// Warps: the groups' rows first, then three (eight for e4m3) that bring K and V,
// then the one that issues the matrix instructions.  A bf16 cache comes by TMA, a
// page's rows of 32 columns at a time into a 64-byte-swizzled tile (three boxes for
// a 96-wide head).  An e4m3 cache is read, widened and stored to the same tiles by
// the eight: four for K and four for V, each half's loads a unit ahead of its
// widening (a prompt of 4096: 69 us, 57 in bf16; seven warps for both sides in
// turn: 104 us with the lists read where they are used, 91 with them ahead).
//
// Tiles at an edge of what the rows see (the diagonal, the window's start, the
// sinks) pass through two of the three first: in a product 0 * NaN would carry a
// number from a masked place to every row, so rows of V that nobody sees become
// zeros, and numbers that are not finite are taken out and noted by sign; a row
// that does see one gets that infinity, or NaN, in that column.  Of a latent they
// are taken out of the key as well, and a row that sees it puts its score right.
//
// With few tiles a cluster of CTAs shares one, each taking a run of its key
// tiles, and merges the results over distributed shared memory.
//
// F32 (a bf16 latent): fp32 queries and results.  Queries and probabilities are two
// bf16 numbers each, a high part and what it leaves (2^-16 or better): a product of Q
// K^T is two, of the two parts of Q in shared memory, and P's low parts take the half
// of S that its high ones leave free in TMEM.  Twice the products, and two stages of
// keys instead of four at width 128: 8 pieces of 256 at 4096 74.6 us (bf16 queries
// 45.5), a prompt of 4096 122 (71).
#include "paged_attn.cuh"

namespace parrot {

namespace {

using namespace tc;

constexpr int kGroup = 128;             // rows of a group
constexpr int kMaxGroups = 3;
constexpr int kMaxRanks = 8;
constexpr float kGrowth = 8.f;          // log2 of the growth of a maximum let through

// Groups of rows, and keys of a tile.
__host__ __device__ constexpr int tile_groups(int d) { return d == 128 ? 2 : 3; }
__host__ __device__ constexpr int tile_keys(int d) { return d == 128 ? 128 : 64; }
// Rows of a TMA box: as many as a page and a tile both hold whole.
__host__ __device__ constexpr int paged_box_rows(int d, int page) {
  return page < tile_keys(d) ? page : tile_keys(d);
}

template <int D, bool E4M3, bool SEP, bool F32 = false>
struct PrefillShape {
  static_assert(!F32 || (!E4M3 && !SEP), "fp32 queries: a bf16 latent");
  static constexpr int kGroups = tile_groups(D), kKeys = tile_keys(D);
  static constexpr int kRows = kGroup * kGroups, kRowWarps = 4 * kGroups;
  static constexpr int kLoadWarps = E4M3 ? 8 : 3;  // widening takes more
  // whole warpgroups: an e4m3 kernel's matrix warp has three idle beside it
  static constexpr int kMmaWarp = kRowWarps + kLoadWarps;
  static constexpr int kThreads = 32 * (kMmaWarp + (E4M3 ? 4 : 1));
  // Registers of a thread of the rows', of the loading warps and of the matrix
  // warp's group (bf16: the loading warps are in it; 0: no split).  setmaxnreg
  // draws on what the launch gave the CTA, the same for each of the SM's four
  // schedulers, and a warpgroup has a warp on each: their sum stays within it.
  // (Width 128, e4m3, 8 pieces of 256 at 4096: 62.9 us with 144 and 72, 63.7 with 152
  // and 64, 79 with 136 and 80.)
  static constexpr int kRowRegs = E4M3 ? (kGroups == 2 ? 144 : 104) : kGroups == 2 ? 208 : 0;
  static constexpr int kLoadRegs = E4M3 ? (kGroups == 2 ? 72 : 64) : 88;
  static constexpr int kMmaRegs = E4M3 ? (kGroups == 2 ? 48 : 40) : 88;
  static_assert(kThreads % 128 == 0, "whole warpgroups");
  static constexpr int kLaunchRegs = 65536 / kThreads / 8 * 8;
  static constexpr int kSplitRegs =
      kRowRegs == 0 ? 0 : kRowRegs * kRowWarps + (E4M3 ? kLoadRegs * kLoadWarps : 0) + kMmaRegs * 4;
  static_assert(kSplitRegs <= kLaunchRegs * (kThreads / 32), "register split");
  // TMEM columns: S (and P over it) of group g at g * kKeys, O behind
  static constexpr uint32_t kTmemO = kGroups * kKeys;
  static_assert(kGroups * (kKeys + D) <= 512, "S and O of all groups");
  static constexpr int kSlabs = D / 32;              // 64-byte columns of a tile
  static constexpr int kTile = kKeys * D * 2;
  static constexpr int kSlab = kKeys * 64;
  static constexpr int kStages = D == 128 ? (SEP || F32 ? 2 : 4) : SEP || F32 ? 4 : 6;
  static constexpr int kSides = SEP ? 2 : 1;
  static constexpr int kQGroup = kGroup * D * 2, kQSlab = kGroup * 64;
  static constexpr int kQHigh = kGroups * kQGroup;   // F32: the low parts lie behind
  static constexpr int kQ = kQHigh * (F32 ? 2 : 1);
  static constexpr int kRing = kStages * kTile;
  // noted columns of each row of a V tile: those that are +inf or NaN, those that are
  // -inf or NaN (e4m3 has only NaN)
  static constexpr int kMarks = E4M3 ? 1 : 2;
  static constexpr int kBad = kStages * kKeys * 16 * kMarks;
  static constexpr int kPart = kRows * D * 4;        // a CTA's result, over Q and the rings
  static constexpr int kBytes0 = kQ + kSides * kRing + kBad + 1024;
  static_assert(kPart <= kQ + kSides * kRing, "the result fits the tiles");
  // one CTA per SM: each takes all of the TMEM
  static constexpr int kBytes = kBytes0 < 118784 ? 118784 : kBytes0;
};

template <int D, bool E4M3>
struct PrefillState {
  static constexpr int kRows = kGroup * tile_groups(D);
  uint64_t k_full[6], k_empty[6], v_full[6], v_empty[6], raw[6];
  uint64_t s_full[kMaxGroups], p_ready[kMaxGroups], o_done[kMaxGroups], drain;
  uint32_t tmem;
  int abort;
  int bad[6];
  uint64_t* armed[2][6];       // the barrier of each stage's last copy, and its phase
  uint32_t armed_parity[2][6];
  // e4m3, of three units of each half of the loading warps
  int row[2][3][E4M3 ? 128 : 1];    // pool row of each key, -1: zeros
  int scale[2][3][E4M3 ? 128 : 1];  // its scale byte
  uint4 poison[E4M3 ? 1 : 2][kRows];  // columns of each row, as they are noted
  float m[kRows], l[kRows];    // merge
};

// Shared-memory descriptors as two words: tiles with a 64-byte swizzle, 512 B
// between 8-row groups; `lead` bytes between slabs (columns contiguous: V).
// The low word moves with the address, the high word is a constant.
__device__ __forceinline__ uint32_t sw64_lo(uint32_t addr, uint32_t lead) {
  return (addr >> 4 & 0x3FFFu) | (lead >> 4) << 16;
}
constexpr uint32_t kSw64Hi = 32u          // stride byte offset 512
                             | 1u << 14   // descriptor version (sm_100)
                             | 4u << 29;  // 64-byte swizzle

// The matrix instructions, by one thread of a warp that stays together: the
// operands are then uniform values, and the issue is not held up by moving
// them between register files (measured: 1150 clocks for ten instructions
// issued from a divergent thread, beside the exponentials of the other warps).
// D (+)= A B, both from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kSw64Hi), "r"(leader));
}
// D (+)= A B with A (bf16 pairs, one row a lane) in TMEM
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kSw64Hi), "r"(leader));
}
__device__ __forceinline__ void commit_to(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// The bounded wait of these warps: the thread sleeps in the barrier for up to
// 0.1 ms at a time instead of polling, so that waiting warps leave the issue
// slots to the exponentials (polling cost the other warps of a scheduler half
// their speed).
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity,
                                            volatile int* abort_flag, int* status, int site) {
  const uint32_t at = smem_u32(bar);
  uint64_t t0 = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      report_status(status, kStatusWaitTimeout, site, (int)blockIdx.x);
      return false;
    }
  }
}
// a barrier of the first `threads` threads that name it, and the or of a flag
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool named_or(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// byte offset of 16-byte vector c of row r in a 64-byte-swizzled tile of R rows
template <int R>
__device__ __forceinline__ uint32_t sw64_at(int r, int c) {
  return (uint32_t)((c >> 2) * (R * 64) + r * 64 + (((c & 3) ^ ((r >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t low_bits(int n) {  // the n lowest bits, n clamped to 0 .. 32
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}

// bits of the four bf16 pairs of a vector that are not finite, one a number
__device__ __forceinline__ uint32_t not_finite8(const uint4& v) {
  uint32_t bits = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bits |= (w[i] & 0x7f80u) == 0x7f80u ? 1u << (2 * i) : 0u;
    bits |= (w[i] & 0x7f800000u) == 0x7f800000u ? 2u << (2 * i) : 0u;
  }
  return bits;
}
// of those: the ones that are +inf or NaN, and the ones that are -inf or NaN
__device__ __forceinline__ uint2 marks8(const uint4& v, uint32_t bits) {
  uint2 marks = make_uint2(0, 0);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = w[i >> 1] >> (16 * (i & 1));
    const bool nan = (h & 0x7fu) != 0, minus = (h & 0x8000u) != 0;
    if (nan || !minus) marks.x |= bits & 1u << i;
    if (nan || minus) marks.y |= bits & 1u << i;
  }
  return marks;
}
__device__ __forceinline__ void or_into(uint4& a, const uint4& b) {
  a.x |= b.x;
  a.y |= b.y;
  a.z |= b.z;
  a.w |= b.w;
}
__device__ __forceinline__ uint32_t keep_mask(uint32_t bits, int i) {  // of pair i
  return (bits >> (2 * i) & 1 ? 0u : 0xffffu) | (bits >> (2 * i) & 2 ? 0u : 0xffff0000u);
}

// A tile's results of up to K CTAs joined: U of the tile's 16-byte vectors at a
// time, all of their remote loads on their way together.
template <int D, bool F32, int K, int U, typename St>
__device__ __forceinline__ void merge_rows(const PagedAttnArgs& a, St& st, const float* part,
                                           const Tile& tile, const RowMap& map, int pos0, int rows,
                                           int kvh, int rank, int ranks, uint32_t live, int threads) {
  const int total = rows * (D / 4), stride = ranks * threads;
  for (int v0 = rank * threads + threadIdx.x; v0 < total; v0 += U * stride) {
    float mk[U][K], lk[U][K];
    float4 x[U][K];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = min(v0 + u * stride, total - 1), r = v / (D / 4), c = v - r * (D / 4);
      const uint32_t at = smem_u32(part + r * D + ((c ^ (r & 7)) << 2));
      const uint32_t m_at = smem_u32(&st.m[r]), l_at = smem_u32(&st.l[r]);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        mk[u][k] = -INFINITY;
        lk[u][k] = 0.f;
        x[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live >> k & 1) {
          mk[u][k] = ld_cluster_f1(mapa_addr(m_at, k));
          lk[u][k] = ld_cluster_f1(mapa_addr(l_at, k));
          x[u][k] = ld_cluster_f4(mapa_addr(at, k));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * stride, r = v / (D / 4), c = v - r * (D / 4);
      if (v >= total) break;
      float mx = mk[u][0], sum = 0.f;
#pragma unroll
      for (int k = 1; k < K; ++k) mx = fmaxf(mx, mk[u][k]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float f = mk[u][k] == -INFINITY ? 0.f : exp2_fast(mk[u][k] - mx);
        sum = fmaf(f, lk[u][k], sum);
        o.x = fmaf(f, x[u][k].x, o.x);
        o.y = fmaf(f, x[u][k].y, o.y);
        o.z = fmaf(f, x[u][k].z, o.z);
        o.w = fmaf(f, x[u][k].w, o.w);
      }
      const int2 th = map(r);
      const float inv = row_inverse(sum, pos0 + th.x);
      const long long at = ((long long)(tile.first + th.x) * a.heads + kvh * map.group + th.y) * D + c * 4;
      store_out<F32>(a, at, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
  }
}

// The end of the rows' warps: with several CTAs to a tile, each merges its share
// of the tile's vectors.  (Working each row's weights out first and keeping eight
// vectors on their way whatever the cluster: 3 us slower with eight CTAs.)
template <int D, bool F32, typename St>
__device__ __forceinline__ void finish_rows(const PagedAttnArgs& a, St& st,
                                            unsigned char* smem, const Tile& tile,
                                            const RowMap& map, int pos0, int rows, int kvh, int rank, int ranks,
                                            int all, int threads) {
  tc_fence_before();
  __syncthreads();
  if (ranks == 1) return;
  uint32_t live = 0;  // the CTAs that had key tiles (the others stored nothing)
  for (int k = 0, left = 0; k < ranks; ++k) {
    left += all;
    if (left >= ranks) {
      live |= 1u << k;
      left -= ranks;
    }
  }
  cluster_sync();
  const float* part = reinterpret_cast<const float*>(smem);
  if (ranks == 2)
    merge_rows<D, F32, 2, 4>(a, st, part, tile, map, pos0, rows, kvh, rank, ranks, live, threads);
  else if (ranks <= 4)
    merge_rows<D, F32, 4, 2>(a, st, part, tile, map, pos0, rows, kvh, rank, ranks, live, threads);
  else
    merge_rows<D, F32, kMaxRanks, 1>(a, st, part, tile, map, pos0, rows, kvh, rank, ranks, live, threads);
  cluster_sync();  // nobody leaves while its result may be read
}

}  // namespace

template <int D, bool E4M3, bool SEP, bool F32>
__global__ void __launch_bounds__(PrefillShape<D, E4M3, SEP, F32>::kThreads, 1)
    paged_prefill_kernel(const PagedAttnArgs a, const __grid_constant__ CUtensorMap k_map,
                         const __grid_constant__ CUtensorMap v_map) {
  using S = PrefillShape<D, E4M3, SEP, F32>;
  constexpr int NS = S::kStages, T = S::kKeys, NG = S::kGroups, R = S::kRows;
  extern __shared__ unsigned char pf_raw[];
  __shared__ PrefillState<D, E4M3> st;
  // tiles start on 1024 bytes, the swizzle's period and more
  unsigned char* smem = pf_raw + (1024 - (smem_u32(pf_raw) & 1023)) % 1024;
  const uint32_t q_u = smem_u32(smem), k_u = q_u + S::kQ, v_u = SEP ? k_u + S::kRing : k_u;
  uint4* bad_cols = reinterpret_cast<uint4*>(smem + S::kQ + S::kSides * S::kRing);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ClusterPlace place = cluster_place();
  const int ranks = a.cluster, rank = place.rank;
  const int group = a.heads / a.kv.kv_heads, index = place.index / a.kv.kv_heads;
  const int kvh = place.index - index * a.kv.kv_heads;
  volatile int* abort_flag = &st.abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&st.k_full[s], E4M3 ? S::kLoadWarps / 2 : 1);
      mbar_init(&st.k_empty[s], 1);
      mbar_init(&st.v_full[s], E4M3 ? S::kLoadWarps / 2 : 1);
      mbar_init(&st.v_empty[s], 1);
      mbar_init(&st.raw[s], 1);
      st.bad[s] = 0;
      st.armed[0][s] = st.armed[1][s] = nullptr;
    }
    for (int h = 0; h < NG; ++h) {
      mbar_init(&st.s_full[h], 1);
      mbar_init(&st.p_ready[h], 4);
      mbar_init(&st.o_done[h], 1);
    }
    mbar_init(&st.drain, 1);
    st.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  __syncthreads();
  griddep_wait();
  const Tile tile = find_tile_from_ends(a.batch, group, R, index, place.count / a.kv.kv_heads);
  if (tile.b < 0) return;  // the whole cluster, before any wait
  const int rows = min(R, tile.n * group - tile.row0);
  const int ctx = clamp_context(a.batch, a.kv, tile.ctx, a.status);
  const int groups = (rows + kGroup - 1) / kGroup;
  const int pos0 = ctx - tile.n;
  const RowMap map(tile.row0, group);
  const int pmin = pos0 + map.token0, pmax = pos0 + map(rows - 1).x;
  // key tiles: the sinks' that lie before the window's first, then the window's
  const int lo = a.window > 0 ? max(0, pmin - a.window + 1) : 0;
  const int t_lo = lo / T;
  const int sink_tiles = min((min(a.sinks, lo) + T - 1) / T, t_lo);
  const int all = pmax < 0 ? 0 : sink_tiles + pmax / T - t_lo + 1;
  // all < 2^26: a position is below 2^31
  const int i0 = (int)((unsigned)(all * rank) / (unsigned)ranks);
  const int i1 = (int)((unsigned)(all * (rank + 1)) / (unsigned)ranks);
  const int n = i1 - i0;  // of this CTA
  const bool loads = warp >= S::kRowWarps && warp != S::kMmaWarp;  // these need neither Q nor TMEM
  if (warp == S::kMmaWarp) tmem_alloc(&st.tmem, 512);
  if (warp < S::kRowWarps) {  // the warp's 32 queries, swizzled; rows that do not exist are zeros
    const int r = warp * 32 + lane;
    const int2 th = map(r);
    const long long q_at = (long long)(tile.first + th.x) * a.q_row + (long long)(kvh * group + th.y) * D;
    const void* mine = static_cast<const char*>(a.q) + q_at * (F32 ? 4 : 2);
    const unsigned long long at = r < rows ? reinterpret_cast<unsigned long long>(mine) : 0ull;
    constexpr int VR = D / 8;
    if constexpr (!F32) {
      uint4 v[VR];
#pragma unroll
      for (int x = 0; x < VR; ++x) {  // side by side: 32 vectors of the warp's rows a step
        const int i = 32 * x + lane;
        const uint4* src = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, at, i / VR));
        v[x] = src != nullptr ? src[i % VR] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int x = 0; x < VR; ++x) {
        const int i = 32 * x + lane;
        *reinterpret_cast<uint4*>(smem + (warp >> 2) * S::kQGroup +
                                  sw64_at<kGroup>((warp & 3) * 32 + i / VR, i % VR)) = v[x];
      }
    } else {
#pragma unroll 4
      for (int x = 0; x < VR; ++x) {
        const int i = 32 * x + lane;
        const float4* src = reinterpret_cast<const float4*>(__shfl_sync(0xffffffffu, at, i / VR));
        float4 f[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        if (src != nullptr) {
          f[0] = src[2 * (i % VR)];
          f[1] = src[2 * (i % VR) + 1];
        }
        const Bf16Pairs p0 = split_queries(f[0].x, f[0].y), p1 = split_queries(f[0].z, f[0].w);
        const Bf16Pairs p2 = split_queries(f[1].x, f[1].y), p3 = split_queries(f[1].z, f[1].w);
        unsigned char* dst = smem + (warp >> 2) * S::kQGroup + sw64_at<kGroup>((warp & 3) * 32 + i / VR, i % VR);
        *reinterpret_cast<uint4*>(dst) = make_uint4(p0.hi, p1.hi, p2.hi, p3.hi);
        *reinterpret_cast<uint4*>(dst + S::kQHigh) = make_uint4(p0.lo, p1.lo, p2.lo, p3.lo);
      }
    }
    fence_async_shared();
  }
  if (!loads) {
    tc_fence_before();
    named_sync(2, 32 * (S::kRowWarps + 1));
    tc_fence_after();
  }
  const uint32_t tmem = st.tmem;
  // not before: a kernel launched early may want TMEM, and holds it until this
  // one has finished
  if (!loads) griddep_launch();

  auto base_of = [&](int i) {
    i += i0;
    return (i < sink_tiles ? i : i - sink_tiles + t_lo) * T;
  };
  auto some_row_sees = [&](int j) {
    return j <= pmax && (a.window == 0 || j > pmin - a.window || j < a.sinks);
  };
  auto is_edge = [&](int base) {  // not every row sees every key of the tile
    return base + T - 1 > pmin ||
           (a.window > 0 && base <= pmax - a.window && base + T > a.sinks);
  };

  if (warp < S::kRowWarps) {
    // ---------------- rows ----------------
    if constexpr (S::kRowRegs > 0)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kRowRegs));
    const int g = warp >> 2, quarter = warp & 3, r = warp * 32 + lane;
    const int pos = pos0 + map(min(r, rows - 1)).x;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lane_addr + g * T, o_at = lane_addr + S::kTmemO + g * D;
    const float scale2 = a.scale * kLog2e;
    const float growth = kGrowth / scale2;
    float m = -INFINITY, l = 0.f;
    bool poison = false;  // st.poison[r]: the columns that are NaN
    const bool busy = g < groups && n > 0;
    bool ok = true;
    for (int i = 0; busy && i < n; ++i) {
      if (!(ok = wait_asleep(&st.s_full[g], i & 1, abort_flag, a.status, 60))) break;
      tc_fence_after();
      constexpr int NC = T / 32;
      uint32_t s[NC][32];
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_ld32_async(s_at + 32 * c, s[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c) tmem_wait_ld(s[c]);
      const int base = base_of(i);
      const bool edge = is_edge(base);
      if (edge) {
        // bit k of a word: the row sees key 32 c + k of the tile
        const int hi = pos - base;  // keys up to hi, and from low or before sk
        const int low = a.window > 0 ? hi - a.window + 1 : 0, sk = a.sinks - base;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint32_t seen = low_bits(hi + 1 - 32 * c) & (~low_bits(low - 32 * c) | low_bits(sk - 32 * c));
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c][k] = seen >> k & 1 ? s[c][k] : 0xff800000u;
        }
        if constexpr (!SEP && !E4M3) {
          // A latent's numbers that are not finite were taken out of the key too: what
          // they would have added to its score, an infinity by the query's sign or NaN.
          const int stage = i % NS;
          if (!(ok = wait_asleep(&st.k_full[stage], (i / NS) & 1, abort_flag, a.status, 61))) break;
          if (*reinterpret_cast<volatile int*>(&st.bad[stage])) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              uint32_t up = 0, down = 0;  // a bit per key
#pragma unroll 1
              for (int k = 0; k < 32; ++k) {
                const int key = base + 32 * c + k;
                if (!(key <= pos && (a.window == 0 || pos - key < a.window || key < a.sinks))) continue;
                const uint32_t* marks = reinterpret_cast<const uint32_t*>(bad_cols + (stage * T + 32 * c + k) * 2);
#pragma unroll 1
                for (int col = 0; col < D; ++col) {
                  const bool plus = marks[col >> 5] >> (col & 31) & 1, minus = marks[4 + (col >> 5)] >> (col & 31) & 1;
                  if (!plus && !minus) continue;
                  const uint32_t q = *reinterpret_cast<const unsigned short*>(
                      smem + g * S::kQGroup + sw64_at<kGroup>(r & (kGroup - 1), col >> 3) + (col & 7) * 2);
                  const bool nan = (plus && minus) || (q & 0x7fffu) == 0 || (q & 0x7fffu) > 0x7f80u;
                  const bool turned = (q & 0x8000u) != 0;
                  if (nan || plus != turned) up |= 1u << k;
                  if (nan || plus == turned) down |= 1u << k;
                }
              }
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                if (up >> k & 1) s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) + INFINITY);
                if (down >> k & 1) s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) - INFINITY);
              }
            }
          }
        }
      }
      float mx[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        mx[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
        for (int k = 2; k < 32; k += 2)
          mx[c] = fmaxf(mx[c], fmaxf(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1])));
      }
      float top = mx[0];
#pragma unroll
      for (int c = 1; c < NC; ++c) top = fmaxf(top, mx[c]);
      const bool move = top > m + growth || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, move)) {
        const float corr = move ? exp2_fast((m - top) * scale2) : 1.f;
        if (move) m = top;
        l *= corr;
        if (i > 0) {  // the previous product is complete: S was issued after it
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(o_at + 16 * c, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
            tmem_st16(o_at + 16 * c, o);
          }
        }
      }
      const float off = m == -INFINITY ? 0.f : -m * scale2;
      const float2 scale_2 = make_float2(scale2, scale2), off_2 = make_float2(off, off);
      float2 sum[4] = {make_float2(l, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t p[16];
        [[maybe_unused]] uint32_t pl[F32 ? 16 : 1];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float2 x = make_float2(__uint_as_float(s[c][2 * k]), __uint_as_float(s[c][2 * k + 1]));
          x = __ffma2_rn(x, scale_2, off_2);
          x.x = exp2_fast(x.x);
          x.y = exp2_fast(x.y);
          sum[k & 3] = __fadd2_rn(sum[k & 3], x);
          if constexpr (F32) {
            const Bf16Pairs w = split_weights(x.x, x.y);
            p[k] = w.hi;
            pl[k] = w.lo;
          } else {
            p[k] = pack_bf16x2(x.x, x.y);
          }
        }
        tmem_st16(s_at + 16 * c, p);
        if constexpr (F32) tmem_st16(s_at + T / 2 + 16 * c, pl);
      }
      sum[0] = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
      l = sum[0].x + sum[0].y;
      tmem_wait_st();
      if (edge) {
        // was a value taken out of the tile that this row sees?
        const int stage = i % NS;
        uint64_t* full = SEP ? &st.v_full[stage] : &st.k_full[stage];
        if (!(ok = wait_asleep(full, (i / NS) & 1, abort_flag, a.status, 61))) break;
        if (*reinterpret_cast<volatile int*>(&st.bad[stage])) {
          uint4 cols[S::kMarks];
#pragma unroll
          for (int w = 0; w < S::kMarks; ++w) cols[w] = poison ? st.poison[w][r] : make_uint4(0, 0, 0, 0);
          for (int k = 0; k < T; ++k) {
            const int key = base + k;
            if (key <= pos && (a.window == 0 || pos - key < a.window || key < a.sinks)) {
#pragma unroll
              for (int w = 0; w < S::kMarks; ++w) {
                or_into(cols[w], bad_cols[(stage * T + k) * S::kMarks + w]);
                // a latent's infinity has the weight 0 (score -inf) or NaN (score +inf)
                if (!SEP && !E4M3) or_into(cols[w], bad_cols[(stage * T + k) * S::kMarks + 1 - w]);
              }
            }
          }
#pragma unroll
          for (int w = 0; w < S::kMarks; ++w) st.poison[w][r] = cols[w];
          poison = true;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st.p_ready[g]);
    }
    // ---------------- result ----------------
    // a CTA's result for the cluster, or in fp32, lies over all groups' tiles
    for (int h = 0; h < groups && n > 0; ++h)
      if (h == g || ranks > 1 || F32) ok = wait_asleep(&st.o_done[h], 0, abort_flag, a.status, 62) && ok;
    tc_fence_after();
    // a wait that ran out: NaN, here or through the cluster's sum, not what is there by then
    if (!ok) l = __uint_as_float(0x7fffffffu);
    const float inv = row_inverse(l, pos);
    float* part = reinterpret_cast<float*>(smem);
    unsigned char* own = smem + g * S::kQGroup;  // the warp's rows, bf16, where Q was
    // loops, not straight lines: this runs once, and fetching its instructions
    // is much of what it costs
#pragma unroll 1
    for (int c = 0; c < S::kSlabs; ++c) {
      uint32_t o[32];
      if (busy) {
        tmem_ld32(o_at + 32 * c, o);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0;
      }
      if (poison) {
        const uint32_t plus = reinterpret_cast<const uint32_t*>(&st.poison[0][r])[c];
        const uint32_t minus = reinterpret_cast<const uint32_t*>(&st.poison[S::kMarks - 1][r])[c];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          if (plus >> k & 1) o[k] = __float_as_uint(__uint_as_float(o[k]) + INFINITY);
          if (minus >> k & 1) o[k] = __float_as_uint(__uint_as_float(o[k]) - INFINITY);
        }
      }
      if (ranks == 1 && !F32) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          uint4 w;
          w.x = pack_bf16x2(__uint_as_float(o[8 * v]) * inv, __uint_as_float(o[8 * v + 1]) * inv);
          w.y = pack_bf16x2(__uint_as_float(o[8 * v + 2]) * inv, __uint_as_float(o[8 * v + 3]) * inv);
          w.z = pack_bf16x2(__uint_as_float(o[8 * v + 4]) * inv, __uint_as_float(o[8 * v + 5]) * inv);
          w.w = pack_bf16x2(__uint_as_float(o[8 * v + 6]) * inv, __uint_as_float(o[8 * v + 7]) * inv);
          *reinterpret_cast<uint4*>(own + sw64_at<kGroup>(r & (kGroup - 1), c * 4 + v)) = w;
        }
      } else if (n > 0 || ranks == 1) {
        if (F32 && ranks == 1) {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inv);
        }
        // rows of D floats, 16-byte vectors exchanged by the row's low bits so
        // that the lanes' stores fall in different banks
#pragma unroll
        for (int v = 0; v < 8; ++v)
          *reinterpret_cast<uint4*>(part + r * D + (((c * 8 + v) ^ (r & 7)) << 2)) =
              make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
    }
    if (ranks == 1) {
      const int2 th = map(min(r, rows - 1));
      const long long out_at = ((long long)(tile.first + th.x) * a.heads + kvh * group + th.y) * D;
      void* out = static_cast<char*>(a.out) + out_at * (F32 ? 4 : 2);
      const unsigned long long at = r < rows ? reinterpret_cast<unsigned long long>(out) : 0ull;
      constexpr int VR = F32 ? D / 4 : D / 8;  // 16-byte vectors of a row
      // (in fp32 over the tiles: with a wait that ran out, copies may still land there)
      const uint32_t lost = F32 ? __ballot_sync(0xffffffffu, !ok) : 0u;
      __syncwarp();
#pragma unroll 4
      for (int x = 0; x < VR; ++x) {
        const int i = 32 * x + lane, ri = i / VR, c = i % VR;
        uint4* dst = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, at, ri));
        const void* src = F32 ? static_cast<const void*>(part + (warp * 32 + ri) * D + ((c ^ (ri & 7)) << 2))
                              : static_cast<const void*>(own + sw64_at<kGroup>(quarter * 32 + ri, c));
        uint4 w = *static_cast<const uint4*>(src);
        if (lost >> ri & 1) w = make_uint4(0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu);
        if (dst != nullptr) dst[c] = w;
      }
    }
    st.m[r] = m * scale2;
    st.l[r] = l;
    finish_rows<D, F32>(a, st, smem, tile, map, pos0, rows, kvh, rank, ranks, all, 32 * S::kRowWarps);
    return;
  }
  if constexpr (S::kRowRegs > 0) {
    if (E4M3 && warp < S::kMmaWarp)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kLoadRegs));
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kMmaRegs));
  }
  if (warp < S::kMmaWarp) {
    // ---------------- keys and values ----------------
    const int lt = threadIdx.x - 32 * S::kRowWarps;
    uint32_t raw_phase = 0;            // a bit per stage
    if constexpr (!E4M3) {
      if (warp == S::kRowWarps) {
        bool ok = true;
        const int box = paged_box_rows(D, 1 << a.kv.page_shift);
        const int pieces = T / box;
        const int beyond = a.kv.pages * a.kv.kv_heads << a.kv.page_shift;  // past the pool: zeros
        for (int i = 0; ok && i < n; ++i) {
          const int s = i % NS;
          const int base = base_of(i);
          const bool edge = is_edge(base);
          // lane p holds the pool row of piece p
          int at = beyond;
          if (lane < pieces) {
            const int j0 = base + lane * box;
            // a piece that some row sees part of (its sinks, or a key up to pmax
            // behind the window's start)
            if (j0 <= pmax && (j0 < a.sinks || a.window == 0 || j0 + box - 1 > pmin - a.window)) {
              // a page partly in sight: its first position that is
              const int page = page_of(a.batch, a.kv, tile.b, j0, a.status);
              if (page >= 0) at = (int)pool_row(a.kv, page, kvh, j0);
            }
          }
          for (int side = 0; side < S::kSides; ++side) {
            uint64_t* empty = side ? &st.v_empty[s] : &st.k_empty[s];
            if (i >= NS && !wait_asleep(empty, (i / NS - 1) & 1, abort_flag, a.status, 63)) {
              ok = false;
              break;
            }
            uint64_t* full = side ? &st.v_full[s] : &st.k_full[s];
            // the side that holds the values passes the check at an edge
            if (edge && side == S::kSides - 1) full = &st.raw[s];
            if (lane == 0) mbar_arrive_expect_tx(full, S::kTile);
            __syncwarp();
            unsigned char* dst = smem + S::kQ + side * S::kRing + s * S::kTile;
            for (int b0 = 0; b0 < pieces * S::kSlabs; b0 += 32) {
              const int b = b0 + lane, piece = b / S::kSlabs, slab = b - piece * S::kSlabs;
              const int y = __shfl_sync(0xffffffffu, at, piece & 31);
              if (b < pieces * S::kSlabs)
                tma_load_2d(dst + slab * S::kSlab + piece * box * 64, side ? &v_map : &k_map,
                            slab * 32, y, full);
            }
            // what is to be waited for should the CTA give up
            if (full == &st.raw[s]) raw_phase ^= 1u << s;
            if (lane == 0) {
              st.armed[side][s] = full;
              st.armed_parity[side][s] =
                  full == &st.raw[s] ? (raw_phase >> s & 1) ^ 1 : (uint32_t)(i / NS) & 1;
            }
            __syncwarp();
          }
        }
        // if a wait ran out somewhere: copies on their way land before the CTA goes on
        if (lane == 0 && *abort_flag) {
          for (int side = 0; side < S::kSides; ++side)
            for (int s = 0; s < NS; ++s)
              if (st.armed[side][s] != nullptr) mbar_drain(st.armed[side][s], st.armed_parity[side][s]);
        }
        __syncwarp();
      } else {
        // the other two warps: the edge tiles' values
        const int ct = lt - 32;
        for (int i = 0; i < n; ++i) {
          const int base = base_of(i);
          if (!is_edge(base)) continue;
          const int s = i % NS;
          const bool mine = wait_asleep(&st.raw[s], raw_phase >> s & 1, abort_flag, a.status, 64);
          if (named_or(1, 64, !mine)) break;  // both warps stop together
          raw_phase ^= 1u << s;
          unsigned char* tile_p = smem + S::kQ + (S::kSides - 1) * S::kRing + s * S::kTile;
          bool any = false;
          for (int k = ct; k < T; k += 64) {
            const bool seen = some_row_sees(base + k);
            uint32_t plus[4] = {0, 0, 0, 0}, minus[4] = {0, 0, 0, 0};
            bool row_bad = false;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
              uint4* p = reinterpret_cast<uint4*>(tile_p + sw64_at<T>(k, c));
              if (!seen) {
                *p = make_uint4(0, 0, 0, 0);
                continue;
              }
              uint4 v = *p;
              const uint32_t bits = not_finite8(v);
              if (bits) {
                const uint2 marks = marks8(v, bits);
                plus[c >> 2] |= marks.x << (8 * (c & 3));
                minus[c >> 2] |= marks.y << (8 * (c & 3));
                row_bad = true;
                v.x &= keep_mask(bits, 0);
                v.y &= keep_mask(bits, 1);
                v.z &= keep_mask(bits, 2);
                v.w &= keep_mask(bits, 3);
                *p = v;
              }
            }
            bad_cols[(s * T + k) * 2] = make_uint4(plus[0], plus[1], plus[2], plus[3]);
            bad_cols[(s * T + k) * 2 + 1] = make_uint4(minus[0], minus[1], minus[2], minus[3]);
            any |= row_bad;
          }
          fence_async_shared();
          any = named_or(1, 64, any);
          if (ct == 0) {
            st.bad[s] = any;
            mbar_arrive(SEP ? &st.v_full[s] : &st.k_full[s]);
          }
        }
      }
    } else {
      // A unit is one side of a tile (of a latent, a tile); the even units are the
      // first four warps', the odd ones the others'.  A unit's raw vectors are
      // loaded while the one before is widened, and the list of its rows takes
      // three steps (page, row and scale, list), one a unit, so that no load is
      // waited for where it is issued.
      constexpr int LT = 16 * S::kLoadWarps;            // threads of a half
      constexpr int VR = D / 16;                        // 16-byte vectors of a raw row
      constexpr int kPer = T * VR / LT;                 // of a thread
      static_assert(T <= LT && kPer * LT == T * VR, "whole vectors, one row or none per thread");
      const int half = lt / LT, ht = lt - half * LT;
      // unit x of this half
      auto tile_of = [&](int x) { return SEP ? x : 2 * x + half; };
      const int units = SEP ? n : (n - half + 1) / 2;
      const bool values = SEP && half == 1;
      const uint4* pool = reinterpret_cast<const uint4*>(values ? a.kv.value : a.kv.key);
      const uint8_t* pool_scale = values ? a.kv.value_scale : a.kv.key_scale;
      uint64_t* full_bars = values ? st.v_full : st.k_full;
      uint64_t* empty_bars = values ? st.v_empty : st.k_empty;
      uint4 raw[kPer];
      int page = -1, at = -1, scale = 0;  // of this thread's key: units x + 3, x + 2
      auto page_step = [&](int x) {
        const int j = base_of(tile_of(x)) + ht;
        page = x < units && ht < T && some_row_sees(j)
                   ? a.batch.page_table[(long long)tile.b * a.batch.table_width + (j >> a.kv.page_shift)]
                   : -1;
      };
      auto row_step = [&](int x) {
        const int j = base_of(tile_of(x)) + ht;
        at = -1;
        scale = 0;
        if (x < units && ht < T && some_row_sees(j)) {
          if ((unsigned)page < (unsigned)a.kv.pages) {
            at = (int)pool_row(a.kv, page, kvh, j);
            scale = pool_scale[at];
          } else {
            report_status(a.status, kStatusBadIndex, 52, page);
          }
        }
      };
      auto list_step = [&](int x) {
        if (ht < T) {
          st.row[half][x % 3][ht] = at;
          st.scale[half][x % 3][ht] = scale;
        }
      };
      auto fetch = [&](int x) {
        if (x >= units) return;
        const int* list = st.row[half][x % 3];
#pragma unroll
        for (int v = 0; v < kPer; ++v) {
          const int i = ht + LT * v, k = i / VR;
          const int r = list[k];
          raw[v] = r >= 0 ? pool[(long long)r * VR + (i - k * VR)] : make_uint4(0, 0, 0, 0);
        }
      };
      page_step(0);
      row_step(0);
      page_step(1);
      list_step(0);
      row_step(1);
      page_step(2);
      list_step(1);
      named_sync(3 + half, LT);
      fetch(0);
      row_step(2);
      page_step(3);
      for (int x = 0; x < units; ++x) {
        const int i = tile_of(x), s = i % NS;
        const bool check = (!SEP || values) && is_edge(base_of(i));
        const bool mine = i < NS || wait_asleep(&empty_bars[s], (i / NS - 1) & 1, abort_flag, a.status, 63);
        if (check && mine) {  // nobody reads what this stage noted before
          if (ht < T) bad_cols[s * T + ht] = make_uint4(0, 0, 0, 0);
          if (ht == 0) st.bad[s] = 0;
        }
        // all stop together; the lists and notes above are complete
        if (named_or(3 + half, LT, !mine)) break;
        unsigned char* dst = smem + S::kQ + (values ? S::kRing : 0) + s * S::kTile;
        const int* list = st.scale[half][x % 3];
#pragma unroll
        for (int v = 0; v < kPer; ++v) {
          const int e = ht + LT * v, k = e / VR, c = e - k * VR;
          const uint32_t s2 = scale_pair(list[k]);
          uint4 o[2];
          e4m3x16_numbers(raw[v], o);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            o[h].x = mul_bf16x2_exact(o[h].x, s2);
            o[h].y = mul_bf16x2_exact(o[h].y, s2);
            o[h].z = mul_bf16x2_exact(o[h].z, s2);
            o[h].w = mul_bf16x2_exact(o[h].w, s2);
            if (check) {
              const uint32_t bits = not_finite8(o[h]);
              if (bits) {
                const int c8 = 2 * c + h;
                uint32_t* cols = reinterpret_cast<uint32_t*>(bad_cols + s * T + k);
                if (SEP) {
                  atomicOr(cols + (c8 >> 2), bits << (8 * (c8 & 3)));
                } else {  // a latent's key is its value: with a NaN in it the score is NaN
                  for (int q = 0; q < 4; ++q) atomicOr(cols + q, 0xffffffffu);
                }
                *reinterpret_cast<volatile int*>(&st.bad[s]) = 1;
                o[h].x &= keep_mask(bits, 0);
                o[h].y &= keep_mask(bits, 1);
                o[h].z &= keep_mask(bits, 2);
                o[h].w &= keep_mask(bits, 3);
              }
            }
            *reinterpret_cast<uint4*>(dst + sw64_at<T>(k, 2 * c + h)) = o[h];
          }
        }
        fetch(x + 1);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full_bars[s]);
        list_step(x + 2);
        row_step(x + 3);
        page_step(x + 4);
      }
    }
  } else if (warp == S::kMmaWarp) {
    // ---------------- matrix instructions ----------------
    if (n > 0) {
      const uint32_t leader = elect_one();
      const uint32_t id_s = make_idesc(kGroup, T);
      const uint32_t id_o = make_idesc(kGroup, D) | (1u << 16);  // V: columns contiguous
      bool ok = true;
      auto scores = [&](int h, int s) {
        const uint32_t qd = sw64_lo(q_u + h * S::kQGroup, 16), kd = sw64_lo(k_u + s * S::kTile, 16);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(tmem + h * T, qd + ((uint32_t)((k >> 1) * S::kQSlab + (k & 1) * 32) >> 4),
                 kd + ((uint32_t)((k >> 1) * S::kSlab + (k & 1) * 32) >> 4), id_s, k != 0, leader);
        if constexpr (F32) {
          const uint32_t ql = qd + (S::kQHigh >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tmem + h * T, ql + ((uint32_t)((k >> 1) * S::kQSlab + (k & 1) * 32) >> 4),
                   kd + ((uint32_t)((k >> 1) * S::kSlab + (k & 1) * 32) >> 4), id_s, 1u, leader);
        }
      };
      auto values = [&](int h, int s, uint32_t accumulate) {
        const uint32_t vd = sw64_lo(v_u + s * S::kTile, S::kSlab);
#pragma unroll
        for (int k = 0; k < T / 16; ++k)
          mma_ts(tmem + S::kTmemO + h * D, tmem + h * T + k * 8, vd + (uint32_t)(k * 1024 >> 4), id_o,
                 k == 0 ? accumulate : 1u, leader);
        if constexpr (F32) {
#pragma unroll
          for (int k = 0; k < T / 16; ++k)
            mma_ts(tmem + S::kTmemO + h * D, tmem + h * T + T / 2 + k * 8, vd + (uint32_t)(k * 1024 >> 4), id_o, 1u,
                   leader);
        }
      };
      if ((ok = wait_asleep(&st.k_full[0], 0, abort_flag, a.status, 66))) {
        tc_fence_after();
        for (int h = 0; h < groups; ++h) {
          scores(h, 0);
          commit_to(&st.s_full[h], leader);
        }
        if (SEP) commit_to(&st.k_empty[0], leader);
      }
      // Copies are waited for ahead of the rows: what this warp does between a
      // group's P and its next scores is time that group waits.
      for (int i = 0; ok && i < n; ++i) {
        const int s = i % NS, s1 = (i + 1) % NS;
        const bool more = i + 1 < n;
        if (SEP && !(ok = wait_asleep(&st.v_full[s], (i / NS) & 1, abort_flag, a.status, 67))) break;
        if (more && !(ok = wait_asleep(&st.k_full[s1], ((i + 1) / NS) & 1, abort_flag, a.status, 66))) break;
        for (int h = 0; h < groups; ++h) {
          if (!(ok = wait_asleep(&st.p_ready[h], i & 1, abort_flag, a.status, 68))) break;
          tc_fence_after();
          values(h, s, i > 0);
          if (more) {
            scores(h, s1);
            commit_to(&st.s_full[h], leader);
          } else {
            commit_to(&st.o_done[h], leader);
          }
        }
        if (!ok) break;
        commit_to(SEP ? &st.v_empty[s] : &st.k_empty[s], leader);
        if (SEP && more) commit_to(&st.k_empty[s1], leader);
      }
      // all matrix instructions have finished before TMEM is freed
      commit_to(&st.drain, leader);
      mbar_drain(&st.drain, 0);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // freed before the cluster waits: a CTA that waits for TMEM on this SM may
  // be the one that a peer of this cluster waits behind
  if (warp == S::kMmaWarp) tmem_dealloc(tmem, 512);
  if (ranks > 1) {
    cluster_sync();
    cluster_sync();
  }
}

namespace {

template <int D, bool E4M3, bool SEP, bool F32 = false>
int launch_prefill(PagedAttnArgs a, const CUtensorMap& k_map, const CUtensorMap& v_map, int sms,
                   cudaStream_t stream) {
  using S = PrefillShape<D, E4M3, SEP, F32>;
  auto k = paged_prefill_kernel<D, E4M3, SEP, F32>;
  const long long tiles = most_tiles(a, S::kRows);
  static std::atomic<unsigned long long> done{0};
  if (!once_per_device(done, [&] {
        // what the compiler gave the launch covers the split, or its waits would not end
        cudaFuncAttributes got;
        return cudaFuncGetAttributes(&got, k) == cudaSuccess &&
               got.numRegs / 8 * 8 * (S::kThreads / 32) >= S::kSplitRegs && allow_shared(k, S::kBytes);
      }))
    return -2;
  // CTAs per tile, while all are resident at once: the time of a tile's longest run
  // of key tiles, and for a cluster three key tiles and a bit for each CTA.
  // Measured, one piece alone, with 1, 2, 4 and 8 CTAs: 64 tokens at 4096 (width 96)
  // 43, 28, 19 and 16 us; 512 at 512 18, 17, 15 and 16; 256 at 256 11.5, 15, 13 and
  // 14; a latent (width 128) 64 at 4096 69, 44, 28 and 21, 512 at 512 17, 20, 18 and,
  // with more clusters than are resident, 34.
  const long long key_tiles = (most_keys(a, S::kRows, S::kKeys) + S::kKeys - 1) / S::kKeys;
  const long long clusters = tiles * a.kv.kv_heads;
  static ClusterCapacity capacity;
  int ranks = 1;
  long long best = 10 * key_tiles;
  for (int r = 2; r <= kMaxRanks && clusters * r <= sms; ++r) {
    const long long cost = 10 * ((key_tiles + r - 1) / r) + 30 + r;
    if (cost < best && clusters <= cluster_capacity(capacity, k, S::kThreads, S::kBytes, r)) {
      ranks = r;
      best = cost;
    }
  }
  a.cluster = ranks;
  if (tiles * ranks * a.kv.kv_heads > 0x7fffffffll) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * ranks * a.kv.kv_heads));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)ranks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k, a, k_map, v_map) == cudaSuccess ? 0 : -2;
}

template <int D>
int launch_prefill_d(const PagedAttnArgs& a, const CUtensorMap& k, const CUtensorMap& v, int sms,
                     cudaStream_t stream) {
  const bool sep = a.kv.value != nullptr;
  if (a.f32) return launch_prefill<D, false, false, true>(a, k, v, sms, stream);
  if (a.kv.key_scale != nullptr)
    return sep ? launch_prefill<D, true, true>(a, k, v, sms, stream)
               : launch_prefill<D, true, false>(a, k, v, sms, stream);
  return sep ? launch_prefill<D, false, true>(a, k, v, sms, stream)
             : launch_prefill<D, false, false>(a, k, v, sms, stream);
}

}  // namespace

int paged_prefill_box_rows(int head_dim, int page_size) { return paged_box_rows(head_dim, page_size); }

int launch_paged_prefill(const PagedAttnArgs& a, const CUtensorMap& k_map,
                         const CUtensorMap& v_map, int sms, cudaStream_t stream) {
  switch (a.kv.head_dim) {
    case 32: return launch_prefill_d<32>(a, k_map, v_map, sms, stream);
    case 64: return launch_prefill_d<64>(a, k_map, v_map, sms, stream);
    case 96: return launch_prefill_d<96>(a, k_map, v_map, sms, stream);
    case 128: return launch_prefill_d<128>(a, k_map, v_map, sms, stream);
  }
  return -1;
}

}  // namespace parrot
