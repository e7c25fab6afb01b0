// Attention of a ragged batch of queries over the paged cache.
//
//   out[i, h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_ih . k_j - m_i)
// over the keys j that token i (at position p of its sequence) sees:
//   j <= p, and without a window or p - j < window or j < sinks.
// A token that sees no key gets zeros.
//
// The query heads of one key head and a run of tokens share their keys: a
// tile is 16 consecutive (token, head) rows of one sequence, token major, so
// each key is read once for all of them.
#include "paged_attn.cuh"

namespace parrot {

namespace {

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the same with f16 operands
__device__ __forceinline__ void mma_16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two e4m3 numbers as a pair of f16, exact (NaN stays NaN)
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)w));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// *p, or zeros.  Volatile, as the products are: the load stays where it is written,
// ahead of a chunk's softmax (moved behind it by the compiler: 64 sequences 26.4 us
// and not 23.9).
__device__ __forceinline__ uint2 load_or_zero(const uint2* p, bool live) {
  uint2 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
      "@p ld.global.v2.u32 {%0, %1}, [%2];\n\t}"
      : "=&r"(v.x), "=&r"(v.y)
      : "l"(p), "r"((int)live));
  return v;
}

__device__ __forceinline__ bool finite_bf16(uint32_t h) { return (h & 0x7f80u) != 0x7f80u; }

// ---------------------------------------------------------------------------
// Few rows per sequence (decode): bound by reading the keys.
//
// A tile's visible keys are cut into 32-key chunks.  The chunks are dealt to
// the warps of a cluster of CTAs; each warp keeps its own ring of chunks in
// flight (16-byte asynchronous copies, no barrier between warps), multiplies
// with m16n8k16 matrix instructions (the 16 rows of the tile; at 8 rows or fewer
// half of the product is idle, which reading the keys hides) and carries its
// own running maximum, sum and fp32 weighted values.  The warps' results are
// merged in shared memory, the CTAs' over distributed shared memory, in a
// fixed order: no workspace, no second launch, no atomics.
//
// An e4m3 cache halves the bytes, and widening them becomes what counts.  Keys
// and values go from memory straight to the products' registers as f16, one
// conversion instruction for two numbers: a thread's 8 bytes of a key are its
// share of two products when the query's columns are permuted alike, and its 4
// bytes of four keys' values, transposed by byte permutations, its share of
// four column tiles when the output's columns are.  The query goes to f16 with a
// power of two per row that puts its largest magnitude at 2^8 (what f16 loses is
// below 2^-32 of that); the keys' scales multiply the scores.  The values'
// scales multiply the probabilities, w = p 2^e, and these go to f16 relative to
// a power of two W per row, at 2^14 W^-1: 11 bits down to 2^-28 W, nothing lost
// above 2^-39 W.  W is a power of two above the largest w so far, each w taken at
// the present maximum, and at most 2^7 times that: it falls when the maximum has
// moved and what it stood for no longer counts (a W that only grew made keys of
// small scales vanish behind those of large ones that softmax had since put out of
// account).
//
// Measured (8 heads on 2, width 96, a window of 2048, contexts of 4096): one
// sequence 7.5 us, most of it the launch, the lists and the merge; 64 sequences
// 25.7 us (3.9 TB/s) in bf16 and 24.0 (2.1 TB/s) in 8 bits, 256 of 2048 87 us
// (4.6 TB/s) and 77.  In 8 bits what bounds it is the chain of a chunk's
// instructions in each of the few warps that fit (246 registers, two CTAs an SM;
// the schedulers issue in a fifth of the cycles); three CTAs of 168 registers are
// slower, 34 us at 64 sequences, and so was the way over a widened tile in shared
// memory (37 us).
// ---------------------------------------------------------------------------
constexpr int kDecKeys = 32;
constexpr int kDecRows = 16;

// Warps of a CTA: four, two CTAs an SM; for few tiles as many as one CTA's
// registers and shared memory hold.
template <int D, bool E4M3, bool SEP, bool WIDE>
struct DecodeShape {
  static constexpr int kWarps = !WIDE ? 4 : D == 128 && SEP && !E4M3 ? 6 : 8;
  static constexpr int kStages = 2;
  // bf16 rows are padded by 16 bytes: an odd number of 16-byte units, so the
  // eight rows of a matrix load fall in different banks
  static constexpr int kRow = 2 * D + 16;
  static constexpr int kTile = kDecKeys * kRow;
  static constexpr int kSide = kTile;
  static constexpr int kStage = kSide * (SEP ? 2 : 1);
  static constexpr int kPoison = kDecRows * 16;  // e4m3: columns of each row that are NaN
  static constexpr int kWarp = E4M3 ? kDecRows * D * 4 + 2 * kDecRows * 4 + kPoison : kStage * kStages;
  static constexpr int kPart = kDecRows * D * 4 + 2 * kDecRows * 4;  // a CTA's result
  static constexpr int kBytes = kWarp * kWarps + kPart;
  static_assert(kWarp >= kPart, "a warp's ring holds its result");
};

// F32 (a bf16 latent): fp32 queries and results.  Queries and probabilities go to
// the products as two bf16 numbers each, a high part and what it leaves, 2^-16 or
// better: as good as fp32 beside the latents' own bf16, and what the single-token
// kernel of the dense latent cache keeps.  Measured (8 heads, width 128, contexts of
// 4096): one sequence 12.2 us, 64 sequences 25.2 (bf16 queries 10.2 and 22.1).
template <int D, bool E4M3, bool SEP, bool WIDE, bool F32>
__global__ void __launch_bounds__(32 * DecodeShape<D, E4M3, SEP, WIDE>::kWarps, WIDE ? 1 : 2)
    paged_decode_kernel(PagedAttnArgs a) {
  using S = DecodeShape<D, E4M3, SEP, WIDE>;
  constexpr int W = S::kWarps;
  constexpr int KS = D / 16;  // k steps of q . k
  constexpr int NT = D / 8;   // column tiles of the output
  extern __shared__ __align__(128) unsigned char dec_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const ClusterPlace place = cluster_place();
  const int ranks = a.cluster, rank = place.rank;
  const int kvh = blockIdx.y, group = a.heads / a.kv.kv_heads;
  griddep_wait();
  griddep_launch();
  const Tile tile = find_tile(a.batch, group, kDecRows, place.index);
  if (tile.b < 0) return;  // the whole cluster
  const int n = clamp_context(a.batch, a.kv, tile.ctx, a.status);
  const int rows = min(kDecRows, tile.n * group - tile.row0);
  const int pos0 = n - tile.n;  // position of the sequence's first batch row
  const RowMap map(tile.row0, group);
  const int pmin = pos0 + map.token0, pmax = pos0 + map(rows - 1).x;

  // the two (token, head) rows of this thread in the product's layout
  int pos[2];
  uint32_t qf[KS][4];
  [[maybe_unused]] uint32_t ql[F32 ? KS : 1][4];  // the low parts
  float row_scale[2];
  typedef typename std::conditional<F32, float, __nv_bfloat16>::type Q;
  const Q* qrow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int2 th = map(min(g + 8 * i, rows - 1));
    pos[i] = pos0 + th.x;
    qrow[i] = static_cast<const Q*>(a.q) + (long long)(tile.first + th.x) * a.q_row +
              (long long)(kvh * group + th.y) * D;
    row_scale[i] = a.scale * kLog2e;
  }
  if constexpr (F32) {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = *reinterpret_cast<const float2*>(qrow[j & 1] + k * 16 + 2 * t + 8 * (j >> 1));
        const Bf16Pairs p = split_queries(f.x, f.y);
        qf[k][j] = p.hi;
        ql[k][j] = p.lo;
      }
  } else if constexpr (!E4M3) {
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        qf[k][j] = *reinterpret_cast<const uint32_t*>(qrow[j & 1] + k * 16 + 2 * t + 8 * (j >> 1));
  } else {
    // columns 32 b + 8 t .. + 7 are this thread's of products 2 b and 2 b + 1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float amax = 0.f;
      float f[KS / 2][8];
#pragma unroll
      for (int b = 0; b < KS / 2; ++b) {
        bf16x8_to_float(*reinterpret_cast<const uint4*>(qrow[i] + 32 * b + 8 * t), f[b]);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[b][e]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // 2^(8 - exponent of amax), within fp32's normal powers
      const int ex = amax > 0.f ? min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 120) : 8;
      const float up = pow2(8 - ex);
      row_scale[i] *= pow2(ex - 8);
#pragma unroll
      for (int b = 0; b < KS / 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[2 * b + (e >> 1)][i + 2 * (e & 1)] = pack_f16x2(f[b][2 * e] * up, f[b][2 * e + 1] * up);
    }
  }

  // chunks: those of the sinks that lie before the window's first, then the
  // window's; key base of chunk c
  const int lo = a.window > 0 ? max(0, pmin - a.window + 1) : 0;
  const int c_lo = lo / kDecKeys;
  const int sink_chunks = min((min(a.sinks, lo) + kDecKeys - 1) / kDecKeys, c_lo);
  const int chunks = pmax < 0 ? 0 : sink_chunks + pmax / kDecKeys - c_lo + 1;
  auto base_of = [&](int c) { return (c < sink_chunks ? c : c - sink_chunks + c_lo) * kDecKeys; };
  const int workers = ranks * W, me = rank * W + warp;

  unsigned char* ring = dec_smem + warp * S::kWarp;
  const uint32_t ring_u = tc::smem_u32(ring);
  // the page of this lane's key of a chunk, -1 where nobody of the tile sees it
  auto page_for = [&](int c) {
    if (c >= chunks) return -1;
    const int j = base_of(c) + lane;
    const bool seen = j <= pmax && (a.window == 0 || j > pmin - a.window || j < a.sinks);
    return seen ? page_of(a.batch, a.kv, tile.b, j, a.status) : -1;
  };
  // bf16: start the copies of chunk c into a stage; keys nobody sees become zeros
  auto fetch = [&](int c, int page, uint32_t stage) {
    if (c < chunks) {
      const int row = page < 0 ? -1 : (int)pool_row(a.kv, page, kvh, base_of(c) + lane);
      constexpr int VR = D / 8;  // 16-byte vectors of a row
#pragma unroll
      for (int i = 0; i < VR; ++i) {
        const int v = lane + 32 * i, r = v / VR, cv = v - r * VR;
        const int rr = __shfl_sync(0xffffffffu, row, r);
        const long long at = ((long long)max(rr, 0) * VR + cv) * 16;
        const uint32_t dst = ring_u + stage * S::kStage + r * S::kRow + cv * 16;
        cp_async16_zfill(dst, static_cast<const char*>(a.kv.key) + at, rr >= 0);
        if (SEP) cp_async16_zfill(dst + S::kSide, static_cast<const char*>(a.kv.value) + at, rr >= 0);
      }
    }
    cp_async_commit();
  };
  // e4m3: chunk c into registers: this thread's keys (8 t .. 8 t + 7 of each 32
  // columns of keys g, g + 8, ...), its values (4 g .. 4 g + 3 of each 32 columns
  // of keys 8 i + 2 t and + 1), and the scale bytes of key `lane`; zeros for keys
  // nobody sees
  constexpr int NB = D / 32;
  uint2 kr[E4M3 ? 4 : 1][E4M3 ? NB : 1];
  uint32_t vr[E4M3 ? 8 : 1][E4M3 ? NB : 1];
  uint32_t scales = 0;
  auto row_for = [&](int c, int page) {
    return c >= chunks || page < 0 ? -1 : (int)pool_row(a.kv, page, kvh, base_of(c) + lane);
  };
  auto fetch_keys = [&](int row) {
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      const int rr = __shfl_sync(0xffffffffu, row, nt * 8 + g);
      const uint2* src = reinterpret_cast<const uint2*>(a.kv.key) + (long long)max(rr, 0) * (D / 8) + t;
#pragma unroll
      for (int b = 0; b < NB; ++b) kr[nt][b] = load_or_zero(src + 4 * b, rr >= 0);
    }
    scales = row < 0 ? (uint32_t)kScaleBias * 0x101u
                     : (uint32_t)a.kv.key_scale[row] |
                           (uint32_t)(SEP ? a.kv.value_scale : a.kv.key_scale)[row] << 8;
  };
  auto fetch_values = [&](int row) {
    const void* values = SEP ? a.kv.value : a.kv.key;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int rr = __shfl_sync(0xffffffffu, row, (i >> 1) * 8 + 2 * t + (i & 1));
      const uint32_t* src = reinterpret_cast<const uint32_t*>(values) + (long long)max(rr, 0) * (D / 4) + g;
#pragma unroll
      for (int b = 0; b < NB; ++b) vr[i][b] = rr < 0 ? 0u : src[8 * b];
    }
  };
  uint32_t* poison = reinterpret_cast<uint32_t*>(ring + S::kWarp - (E4M3 ? S::kPoison : 0));  // [row][4]
  if constexpr (E4M3) {
    poison[lane] = poison[lane + 32] = 0;
    __syncwarp();
  }
  float top_w[2] = {0.f, 0.f};        // e4m3: W of each row, 0 before its first
  float most_w[2] = {0.f, 0.f};       // the largest of this thread's weights so far, at the present maximum
  const bool two = rows > 8;          // whether rows g + 8 exist

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  int c = me, it = 0;
  int next_page = -1;
  [[maybe_unused]] int next_row = -1;
  if constexpr (E4M3) {
    const int row = row_for(c, page_for(c));
    fetch_keys(row);
    fetch_values(row);
    next_page = page_for(c + workers);
  } else {
    fetch(c, page_for(c), 0);
    next_page = page_for(c + workers);
  }
  for (; c < chunks; c += workers, ++it) {
    // scores of the 16 rows and 32 keys
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    [[maybe_unused]] uint32_t v_u = ring_u;
    [[maybe_unused]] float v_scale[4][2];  // of the keys of this thread's columns
    if constexpr (E4M3) {
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          mma_16816_f16(s[nt], qf[2 * b], e4m3x2_to_f16(kr[nt][b].x), e4m3x2_to_f16(kr[nt][b].x >> 16));
          mma_16816_f16(s[nt], qf[2 * b + 1], e4m3x2_to_f16(kr[nt][b].y), e4m3x2_to_f16(kr[nt][b].y >> 16));
        }
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t b = __shfl_sync(0xffffffffu, scales, nt * 8 + 2 * t + e);
          const float ks = __uint_as_float((b & 0xffu) << 23);
          v_scale[nt][e] = __uint_as_float((b >> 8 & 0xffu) << 23);
          s[nt][e] *= ks;
          s[nt][2 + e] *= ks;
        }
      // the next chunk's keys come while this one is worked on, its values while
      // those keys are multiplied
      next_row = row_for(c + workers, next_page);
      fetch_keys(next_row);
      next_page = page_for(c + 2 * workers);
    } else {
      const int slot = it & 1;
      fetch(c + workers, next_page, slot ^ 1);
      next_page = page_for(c + 2 * workers);
      cp_async_wait<1>();
      __syncwarp();
      const uint32_t k_u = ring_u + slot * S::kStage;
      v_u = SEP ? k_u + S::kSide : k_u;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int k2 = 0; k2 < KS / 2; ++k2) {
          uint32_t b[4];
          ldmatrix_x4(b, k_u + (nt * 8 + (lane & 7)) * S::kRow + k2 * 64 + (lane >> 3) * 16);
          mma_16816(s[nt], qf[2 * k2], b[0], b[1]);
          mma_16816(s[nt], qf[2 * k2 + 1], b[2], b[3]);
          if constexpr (F32) {
            mma_16816(s[nt], ql[2 * k2], b[0], b[1]);
            mma_16816(s[nt], ql[2 * k2 + 1], b[2], b[3]);
          }
        }
    }
    const int base = base_of(c);
    const bool whole = base + kDecKeys - 1 <= pmin &&
                       (a.window == 0 || base > pmax - a.window || base + kDecKeys <= a.sinks);
    auto sees = [&](int i, int j) {
      return j <= pos[i] && (a.window == 0 || pos[i] - j < a.window || j < a.sinks);
    };
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[nt][j] *= row_scale[j >> 1];
        if (!whole && !sees(j >> 1, base + nt * 8 + 2 * t + (j & 1))) s[nt][j] = -INFINITY;
      }
    float corr[2] = {1.f, 1.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !two) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) s[nt][2] = s[nt][3] = 0.f;
        continue;
      }
      float mx = m[i];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * i], s[nt][2 * i + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float ref = mx == -INFINITY ? 0.f : mx;
      corr[i] = exp2_fast(m[i] - ref);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_fast(s[nt][2 * i + e] - ref);
          s[nt][2 * i + e] = p;
          sum += p;
        }
      l[i] = fmaf(l[i], corr[i], sum);  // this thread's columns; the quad is summed at the end
    }
    if constexpr (E4M3) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        most_w[i] *= corr[i];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[nt][2 * i + e] *= v_scale[nt][e];
            most_w[i] = fmaxf(most_w[i], s[nt][2 * i + e]);
          }
      }
      // W is set anew where a weight reaches it or where a thread's have fallen 2^6
      // below it (the quad's need not have: then it stays)
      const bool off0 = most_w[0] >= top_w[0] || most_w[0] < top_w[0] * 0.015625f;
      const bool off1 = two && (most_w[1] >= top_w[1] || most_w[1] < top_w[1] * 0.015625f);
      if (__any_sync(0xffffffffu, off0 || off1)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float most = fmaxf(most_w[i], __shfl_xor_sync(0xffffffffu, most_w[i], 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          if (most > 0.f) {
            // the power of two above it (at least 2^-112, so that 2^14 / W is finite: below
            // every weight of p = 1)
            const float w = fmaxf(__uint_as_float((__float_as_uint(most) & 0x7f800000u) + 0x00800000u), pow2(-112));
            // most >= corr W / 2^6, so the product is below 2^6 (W / w alone may be past fp32)
            corr[i] = corr[i] * top_w[i] * __uint_as_float((254u << 23) - __float_as_uint(w));
            top_w[i] = w;
          }
        }
      }
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        o[nt][0] *= corr[0];
        o[nt][1] *= corr[0];
        o[nt][2] *= corr[1];
        o[nt][3] *= corr[1];
      }
    }
    if constexpr (E4M3) {
      if (!whole && pmin != pmax) {
        // As below: a NaN among the values is taken out, and noted for the rows
        // that see its key.
        uint32_t some = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int b = 0; b < NB; ++b) some |= e4m3_nan_bits(vr[i][b]);
        if (__any_sync(0xffffffffu, some != 0)) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              const uint32_t nan = e4m3_nan_bits(vr[i][b]);
              if (nan == 0) continue;
              const uint32_t cols = ((nan >> 7 & 1) | (nan >> 14 & 2) | (nan >> 21 & 4) | (nan >> 28 & 8)) << (4 * g);
              const int j = base + (i >> 1) * 8 + 2 * t + (i & 1);
              for (int r = 0; r < rows; ++r) {
                const int at = pos0 + map(r).x;
                if (j <= at && (a.window == 0 || at - j < a.window || j < a.sinks))
                  atomicOr(poison + r * 4 + b, cols);
              }
              vr[i][b] &= ~((nan >> 7) * 0xffu);
            }
        }
      }
      float up[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)  // 2^14 / W
        up[i] = top_w[i] > 0.f ? __uint_as_float((268u << 23) - __float_as_uint(top_w[i])) : 0.f;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int nt = 2 * kk + (j >> 1);
          p[j] = pack_f16x2(s[nt][2 * (j & 1)] * up[j & 1], s[nt][2 * (j & 1) + 1] * up[j & 1]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          // four keys' bytes of four columns, transposed
          const uint32_t w0 = vr[4 * kk][b], w1 = vr[4 * kk + 1][b], w2 = vr[4 * kk + 2][b], w3 = vr[4 * kk + 3][b];
          const uint32_t t0 = __byte_perm(w0, w1, 0x5140), t1 = __byte_perm(w0, w1, 0x7362);
          const uint32_t t2 = __byte_perm(w2, w3, 0x5140), t3 = __byte_perm(w2, w3, 0x7362);
          // t0: columns 0 (low half) and 1 of keys 0, 1; t2: of keys 2, 3
          mma_16816_f16(o[4 * b], p, e4m3x2_to_f16(t0), e4m3x2_to_f16(t2));
          mma_16816_f16(o[4 * b + 1], p, e4m3x2_to_f16(t0 >> 16), e4m3x2_to_f16(t2 >> 16));
          mma_16816_f16(o[4 * b + 2], p, e4m3x2_to_f16(t1), e4m3x2_to_f16(t3));
          mma_16816_f16(o[4 * b + 3], p, e4m3x2_to_f16(t1 >> 16), e4m3x2_to_f16(t3 >> 16));
        }
      }
      fetch_values(next_row);
    } else {
      if (!whole && pmin != pmax) {
        // A value that is not finite would reach, as 0 * NaN in the product, the
        // rows that do not see its key.  Take such numbers out of the tile and add
        // them to the rows that see them.
        unsigned bad_row = 0;
#pragma unroll 1
        for (int i = 0; i < D / 2; ++i) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(v_u + lane * S::kRow + i * 4));
          bad_row |= !finite_bf16(w) || !finite_bf16(w >> 16);
        }
        const unsigned bad = __ballot_sync(0xffffffffu, bad_row);
        if (bad) {
          for (unsigned left = bad; left; left &= left - 1) {
            const int j = __ffs(left) - 1;  // key base + j: column tile j / 8, thread (j % 8) / 2
            const int src = (lane & ~3) | ((j & 7) >> 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float p = 0.f;
#pragma unroll
              for (int nt = 0; nt < 4; ++nt)
                if (nt == j >> 3) p = j & 1 ? s[nt][2 * i + 1] : s[nt][2 * i];
              p = __shfl_sync(0xffffffffu, p, src);
              const bool vis = sees(i, base + j);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                uint32_t w;
                asm volatile("ld.shared.u32 %0, [%1];"
                             : "=r"(w)
                             : "r"(v_u + j * S::kRow + (nt * 8 + 2 * t) * 2));
                const float2 v = bf16x2_to_float2(w);
                if (vis && !finite_bf16(w)) o[nt][2 * i] = fmaf(p, v.x, o[nt][2 * i]);
                if (vis && !finite_bf16(w >> 16)) o[nt][2 * i + 1] = fmaf(p, v.y, o[nt][2 * i + 1]);
              }
            }
          }
          __syncwarp();
          if (bad_row) {
#pragma unroll 1
            for (int i = 0; i < D / 2; ++i) {
              const uint32_t at = v_u + lane * S::kRow + i * 4;
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
              if (!finite_bf16(w)) w &= 0xffff0000u;
              if (!finite_bf16(w >> 16)) w &= 0x0000ffffu;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
            }
          }
          __syncwarp();
        }
      }
      // weighted values: the probabilities rounded to bf16, as the matrix
      // instructions take them (half a step of 2^-8 relative each, unbiased)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t p[4];
        [[maybe_unused]] uint32_t pl[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int nt = 2 * kk + (j >> 1);
          if constexpr (F32) {
            const Bf16Pairs w = split_weights(s[nt][2 * (j & 1)], s[nt][2 * (j & 1) + 1]);
            p[j] = w.hi;
            pl[j] = w.lo;
          } else {
            p[j] = tc::pack_bf16x2(s[nt][2 * (j & 1)], s[nt][2 * (j & 1) + 1]);
          }
        }
#pragma unroll
        for (int n2 = 0; n2 < NT / 2; ++n2) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, v_u + (kk * 16 + (lane & 15)) * S::kRow + n2 * 32 + (lane >> 4) * 16);
          mma_16816(o[2 * n2], p, b[0], b[1]);
          mma_16816(o[2 * n2 + 1], p, b[2], b[3]);
          if constexpr (F32) {
            mma_16816(o[2 * n2], pl, b[0], b[1]);
            mma_16816(o[2 * n2 + 1], pl, b[2], b[3]);
          }
        }
      }
      __syncwarp();  // the stage may be filled again
    }
  }
  cp_async_wait<0>();
  __syncwarp();

  // ---- merge: warps of the CTA, then CTAs of the cluster -------------------
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  float* mine = reinterpret_cast<float*>(ring);  // [rows][D], then m, l
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    if constexpr (E4M3) {
      // O is relative to W 2^-14; column tiles 4 b + q hold columns 32 b + 4 n + q
      const float back = top_w[i] * pow2(-14);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float f[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f[q] = o[4 * b + q][2 * i] * back;
          f[4 + q] = o[4 * b + q][2 * i + 1] * back;
        }
        if (const uint32_t cols = poison[r * 4 + b] >> (8 * t) & 0xffu) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (cols >> q & 1) f[q] = NAN;
        }
        float4* dst = reinterpret_cast<float4*>(mine + r * D + 32 * b + 8 * t);
        dst[0] = make_float4(f[0], f[1], f[2], f[3]);
        dst[1] = make_float4(f[4], f[5], f[6], f[7]);
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        *reinterpret_cast<float2*>(mine + r * D + nt * 8 + 2 * t) =
            make_float2(o[nt][2 * i], o[nt][2 * i + 1]);
    }
    if (t == 0) {
      mine[kDecRows * D + r] = m[i];
      mine[kDecRows * D + kDecRows + r] = l[i];
    }
  }
  __syncthreads();
  float* part = reinterpret_cast<float*>(dec_smem + S::kWarp * W);
  auto write = [&](int r, int col, float4 v, float sum) {
    const int2 th = map(r);
    const float inv = row_inverse(sum, pos0 + th.x);
    const long long at = ((long long)(tile.first + th.x) * a.heads + kvh * group + th.y) * D + col;
    store_out<F32>(a, at, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
  };
  for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * W) {
    const int r = i / (D / 4), col = (i - r * (D / 4)) * 4;
    float mx = -INFINITY, sum = 0.f;
    const float* w0 = reinterpret_cast<const float*>(dec_smem);
    constexpr int kStride = S::kWarp / 4;
#pragma unroll
    for (int w = 0; w < W; ++w) mx = fmaxf(mx, w0[w * kStride + kDecRows * D + r]);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* p = w0 + w * kStride;
      const float mw = p[kDecRows * D + r];
      const float f = mw == -INFINITY ? 0.f : exp2_fast(mw - mx);
      sum = fmaf(f, p[kDecRows * D + kDecRows + r], sum);
      const float4 x = *reinterpret_cast<const float4*>(p + r * D + col);
      v.x = fmaf(f, x.x, v.x);
      v.y = fmaf(f, x.y, v.y);
      v.z = fmaf(f, x.z, v.z);
      v.w = fmaf(f, x.w, v.w);
    }
    if (ranks == 1) {
      write(r, col, v, sum);
    } else {
      *reinterpret_cast<float4*>(part + r * D + col) = v;
      if (col == 0) {
        part[kDecRows * D + r] = mx;
        part[kDecRows * D + kDecRows + r] = sum;
      }
    }
  }
  if (ranks == 1) return;
  tc::cluster_sync();
  for (int i = rank * 32 * W + threadIdx.x; i < rows * (D / 4);
       i += ranks * 32 * W) {
    const int r = i / (D / 4), col = (i - r * (D / 4)) * 4;
    float mx = -INFINITY, sum = 0.f;
    for (int k = 0; k < ranks; ++k)
      mx = fmaxf(mx, ld_cluster_f1(tc::mapa_shared(part + kDecRows * D + r, k)));
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ranks; ++k) {
      const float mk = ld_cluster_f1(tc::mapa_shared(part + kDecRows * D + r, k));
      const float f = mk == -INFINITY ? 0.f : exp2_fast(mk - mx);
      sum = fmaf(f, ld_cluster_f1(tc::mapa_shared(part + kDecRows * D + kDecRows + r, k)), sum);
      const float4 x = ld_cluster_f4(tc::mapa_shared(part + r * D + col, k));
      v.x = fmaf(f, x.x, v.x);
      v.y = fmaf(f, x.y, v.y);
      v.z = fmaf(f, x.z, v.z);
      v.w = fmaf(f, x.w, v.w);
    }
    write(r, col, v, sum);
  }
  tc::cluster_sync();  // nobody leaves while its result may be read
}

// CTAs per tile: as many as keep every warp two chunks or more of the longest
// possible context, while nineteen twentieths of the clusters that fit at once are enough
// (against three CTAs an SM, whatever fits: 24 sequences of 4096, 8-bit 13.5 us and
// 19.0, 80 of a latent 29 and 42, 8 of four heads of 128 12.6 and 23.9).
//
// A few tiles of long contexts, whose warps would go through many chunks one
// after the other, take the wide kind and clusters of up to 16, on half of the SMs
// at most (clusters of one CTA an SM fill the GPU's partitions badly: 8 tiles of 16
// CTAs run in two turns).  One sequence of a latent of 32,768 keys: 49 us with eight
// CTAs of four warps, 36 with eight of eight, 22 with sixteen; of 8192: 16, 14 and
// 11; of 4096, where the wide kind begins: 10.5 and 10.1; of 2048 it would lose: 7.6
// and 10.0.
template <int D, bool E4M3, bool SEP, bool WIDE, bool F32>
int launch_decode(PagedAttnArgs a, long long tiles, long long chunks, int most, int sms, cudaStream_t stream) {
  using S = DecodeShape<D, E4M3, SEP, WIDE>;
  auto k = paged_decode_kernel<D, E4M3, SEP, WIDE, F32>;
  static std::atomic<unsigned long long> done{0};
  if (!once_per_device(done, [&] {
        return allow_shared(k, S::kBytes) &&
               (!WIDE || cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess);
      }))
    return -2;
  static ClusterCapacity capacity;
  const long long clusters = tiles * a.kv.kv_heads;
  int ranks = 1;
  for (int r = 2; r <= most && chunks >= 2LL * r * S::kWarps; ++r)
    if (WIDE ? clusters * r * 2 <= sms
             : clusters * 20 <= 19LL * cluster_capacity(capacity, k, 32 * S::kWarps, S::kBytes, r))
      ranks = r;
  a.cluster = ranks;
  if (tiles * ranks > 0x7fffffffll) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * ranks), a.kv.kv_heads);
  cfg.blockDim = dim3(32 * S::kWarps);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)a.cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k, a) == cudaSuccess ? 0 : -2;
}

template <int D, bool E4M3, bool SEP, bool F32 = false>
int launch_decode_of(const PagedAttnArgs& a, cudaStream_t stream, int sms) {
  const long long tiles = most_tiles(a, kDecRows), all = tiles * a.kv.kv_heads;
  const long long chunks = (most_keys(a, kDecRows, kDecKeys) + kDecKeys - 1) / kDecKeys;
  if (all * 16 <= sms && chunks >= 128)
    return launch_decode<D, E4M3, SEP, true, F32>(a, tiles, chunks, 16, sms, stream);
  return launch_decode<D, E4M3, SEP, false, F32>(a, tiles, chunks, 8, sms, stream);
}

template <int D>
int launch_decode_d(const PagedAttnArgs& a, cudaStream_t stream, int sms) {
  const bool sep = a.kv.value != nullptr;
  if (a.f32) return launch_decode_of<D, false, false, true>(a, stream, sms);
  if (a.kv.key_scale != nullptr)
    return sep ? launch_decode_of<D, true, true>(a, stream, sms) : launch_decode_of<D, true, false>(a, stream, sms);
  return sep ? launch_decode_of<D, false, true>(a, stream, sms) : launch_decode_of<D, false, false>(a, stream, sms);
}

}  // namespace

// Few new tokens per sequence: the kernel above (its tile reads the keys for 16
// rows); beyond, paged_prefill.cu's (for 256 or 384).  Measured (8 heads on 2, width
// 96, a window of 2048, contexts of 4096) in bf16: 64 single tokens 26 us here and 38
// there, 32 sequences of 2 tokens 21 and 25, 8 of 2 15 and 13, 8 of 4 16 and 14, 32 of
// 4 30 and 26.  An 8-bit cache, whose tiles paged_prefill.cu's warps have to widen:
// 32 of 4 25 and 33, 8 of 8 15 and 17, 32 of 8 39 and 34.  Few rows over long contexts
// get more warps here: one piece of 8 over 16,384 keys 18 and 39, 4 of 4 of a latent
// 32 and 36.  Single tokens beside pieces go with the pieces (8 beside one of 256: 21
// us, and 29 in two launches; 64 beside 512: 58, and 64 in two).  The mean stands for
// uneven batches too, on either side of its limits (one piece among single tokens at
// 4096; here, and there with two more tokens in the piece): 255 and 256 at 2048 111 us
// and 153, 127 and 128 74 and 76, 31 and 32 21 and 27, of a latent 67 and 73; in 8 bits
// 127 and 385 74 and 115, 31 and 96 24 and 43; only 127 and 385 of an 8-bit latent lose,
// 118 and 100.
bool paged_few_queries(const PagedAttnArgs& a, int sms) {
  const long long n = a.batch.tokens, batch = a.batch.batch, rows = n * a.heads;
  if (n <= 2 * batch) return true;
  if (a.kv.key_scale != nullptr && (n <= 4 * batch || (n <= 8 * batch && rows <= 64 * kDecRows)))
    return true;
  return n <= 8 * batch && rows <= sms && most_keys(a, kDecRows, kDecKeys) >= 128 * kDecKeys;
}

int launch_paged_decode(const PagedAttnArgs& a, int sms, cudaStream_t stream) {
  switch (a.kv.head_dim) {
    case 32: return launch_decode_d<32>(a, stream, sms);
    case 64: return launch_decode_d<64>(a, stream, sms);
    case 96: return launch_decode_d<96>(a, stream, sms);
    case 128: return launch_decode_d<128>(a, stream, sms);
  }
  return -1;
}

}  // namespace parrot
