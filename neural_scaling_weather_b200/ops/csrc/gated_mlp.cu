// Gated feed-forward network on the tensor cores.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u,  y = h Wd^T + bd + residual
//   dh = dy Wd,  dg = dh * u * act'(g),  du = dh * act(g),  dx = dg Wg + du Wu
//
// act is SiLU, g / (1 + exp(-g)), or the exact GELU, g Phi(g).  Three kernel families:
//
// * gated_kernel: one persistent CTA-pair kernel (tcgen05.mma.cta_group::2, 256-row pair tiles) in five
//   forms that differ in where their operands come from and in the epilogue.  64800 x 1024 x 2736, bf16, in
//   microseconds: short runs with uniform operands (no power limit), with random ones, and in a steady state at
//   the power limit, beside the library's plain product there:
//                                   uniform          random   steady   library, steady
//     kUp, with g and u             481 (1510 TF)    584      678      610 (two projections, nothing else)
//     kDown                         224 (1623 TF)    279      328      295
//     kDh, with the column sums     364  (997 TF)    442      495      323
//     kDx                           383 (1897 TF)    509      595      562
//     kDw, three weights            597 (1825 TF)    822      941      936
//     kUp    both projections at once: the pair's B tile is 128 rows of Wg (CTA 0) and the same 128
//            rows of Wu (CTA 1), so g and u of one hidden unit land in the same TMEM lane 128 columns
//            apart and the activation and the product happen in registers; h (and, for training, g and
//            u) leave by TMA store.
//     kDown  h Wd^T + bd + residual; residual tiles arrive by TMA before the accumulator is ready.
//     kDh    dy Wd with Wd read as it is stored ([D, H], MN-major for this product, so no transposed
//            copy exists); the epilogue loads g and u tiles by TMA and writes dg and du.
//     kDx    dg Wg + du Wu as ONE product of depth 2 H: the k-loop runs through (dg, Wg), then
//            (du, Wu), into the same accumulator; the weights are again read MN-major as stored.
//     kDw    the weight gradients dg^T x, du^T x and dy^T h: both operands token-major as they are, MN-major
//            for the MMA, the depth is the tokens.  See gated_unit for the schedule.
//   The wide forms are bound by the tensor cores at the clock that the power limit leaves, at fewer tokens by the last
//   wave of 256-row tiles.  kDh reads and writes 8 bytes per hidden unit and token (g, u, dg, du) for 2 N operations:
//   neither memory (39 % busy) nor the tensor cores (46 %) are full, its epilogue warps wait for their tiles.
// * split_kernel: the four products of a few hundred rows, depth split over a cluster.  See there.
// * skinny_kernel: up to 16 tokens, where the time is that of streaming the weights once.  See there.
//
// Sums are fp32 in TMEM / registers.  Rounded to 16 bits: g, u (kept for the backward), h, dg, du,
// because the following products take 16-bit operands; the forward's h is computed from the unrounded
// g and u.  The bias gradients are fp32 sums of the rounded dg and du.  In fp16 those values overflow past 65504, as
// any 16-bit activation does.
#include <cuda.h>

#include <algorithm>
#include <cstring>

#include "attn_mma.cuh"
#include "gated.cuh"

namespace nsw {
namespace tc {

enum : int { kUp = 0, kDown = 1, kDh = 2, kDx = 3, kDw = 4 };
// Epilogue warps and 2 KB tile buffers of each.  kDh loads two tiles and stores two for each 32 columns, more
// latency than arithmetic: sixteen warps with one pair of buffers each, where the eight of the other forms took the
// same time without the column sums that sixteen do beside (kUp with sixteen: no gain).
constexpr int epi_warps(int mode) { return mode == kDh ? 16 : 8; }
constexpr int epi_bufs(int mode) { return 32 / epi_warps(mode); }
constexpr int stages(int mode) { return mode == kDh ? 4 : 5; }  // 32 KB a CTA; kDh's column sums take one

// One weight's gradient in kDw
struct DwSeg {
  int64_t end;      // tiles of this weight and those before it
  int64_t n_tiles;  // of a tile row
  int64_t M, N, ldd;
  void* D;
  int out_f32, accumulate, tma_out;  // tma_out: 16-bit rows that an output map can address
};
constexpr int kDwWeights = 3;

// Grouped form (GROUPED, the routed experts of experts.cu): the rows are sorted by expert, each expert's padded with
// zero rows to whole 256-row tiles, and the weights are stacked, [experts][rows][cols], behind tensor maps of three
// dimensions, so that a tile past an expert's last row or column reads zeros and not the next expert's.  How many tiles
// there are, and whose, is read from device memory: the grid is sized by the most there can be.
struct GroupParams {
  const int* tiles;  // [0]: row tiles, then the expert of each
  const int* rows;   // kDw: [experts + 1] first rows of the experts' groups
  int64_t experts;
};

struct GatedParams {
  CUtensorMap a0, a1, a2, b0, b1;  // operands (a1 / b1: Wu in kUp, the second half of the depth in kDx)
  CUtensorMap in0, in1;          // kDh: g, u; kDown: residual
  CUtensorMap out0, out1, out2;  // kUp: h, g, u; kDh: dg, du; kDown / kDx: the result
  int64_t M, N;                  // rows; columns of the result (hidden units in kUp / kDh)
  int kb0, kb;                   // k-blocks of the first operand pair, and in all
  const void* bias0;
  const void* bias1;
  int bias_dtype;
  int act;      // 0 SiLU, 1 GELU
  int save;     // kUp: store g and u
  int has_res;  // kDown: residual tiles by TMA
  int plain;    // kDown / kDx: rows that no tensor map can address; result and residual by plain accesses
  void* D;
  const void* res;
  int64_t ldd, ldres;
  // kDw: the weights' tiles in order; see gated_unit
  DwSeg seg[kDwWeights];  // (weight i: out_i, a_i and b_(i / 2))
  int64_t direct;
  int rem, splits;
  float* ws;  // [splits][rem][256][256]
  // kDh: column sums of the rounded dg and du over each CTA's 128 rows, [2 m_tiles][2 sums_half] (null: none)
  float* sums;
  int64_t sums_half;
  GroupParams group;
};

// A pair's i-th unit of work: a tile and its range of k-blocks.  Every form but kDw: tiles pair, pair + npairs,
// ...  kDw has few tiles and a long depth, so whole waves of tiles (`direct` of them, a multiple of the
// pairs) are worked in full, and the depth of the `rem` tiles that are left is cut into `splits` pieces, in
// piece-major order, whose fp32 partials go to the workspace and are added in piece order by dw_sum_kernel.
// Pairs that run at one time read the same tokens' slab of both operands from L2.  The grouped kDw has a tile for each
// weight, expert and part of the expert's matrix, in this order, whose depth is the expert's rows (zero for an expert
// without tokens: the tile is zeros).
struct GUnit {
  int64_t tile;
  int kb0, kb1;
  int64_t slot;  // partial's index, or -1
  int expert;
};
template <int MODE, bool GROUPED>
__device__ __forceinline__ bool gated_unit(const GatedParams& p, int64_t num_tiles, int64_t pair, int64_t npairs,
                                           int64_t i, GUnit& u) {
  const int64_t v = pair + i * npairs;
  u.slot = -1;
  u.kb0 = 0;
  u.kb1 = p.kb;
  u.tile = v;
  u.expert = 0;
  if (GROUPED) {
    if (v >= num_tiles) return false;
    if (MODE == kDw) {
      const int seg = v < p.seg[0].end ? 0 : v < p.seg[1].end ? 1 : 2;
      const int64_t t = v - (seg ? p.seg[seg - 1].end : 0), of = (p.seg[seg].M + BM2 - 1) / BM2 * p.seg[seg].n_tiles;
      u.expert = (int)(t / of);
      u.tile = v - u.expert * of;  // as if the weight had this expert's tiles alone
      u.kb0 = __ldg(p.group.rows + u.expert) / BK;
      u.kb1 = __ldg(p.group.rows + u.expert + 1) / BK;
    } else {
      u.expert = __ldg(p.group.tiles + 1 + v / ((p.N + (MODE == kUp ? 128 : 256) - 1) / (MODE == kUp ? 128 : 256)));
    }
    return true;
  }
  if (MODE != kDw || v < p.direct) return v < num_tiles;
  const int64_t w = v - p.direct;
  if (w >= (int64_t)p.rem * p.splits) return false;
  const int64_t piece = w / p.rem;
  u.tile = p.direct + (w - piece * p.rem);
  u.kb0 = (int)(piece * p.kb / p.splits);
  u.kb1 = (int)((piece + 1) * p.kb / p.splits);
  u.slot = w;
  return true;
}

struct DwPlan {
  int64_t direct;
  int rem, splits;
};

template <typename T, int MODE>
struct SmemG {
  static constexpr int EW = epi_warps(MODE), GS = stages(MODE);
  alignas(1024) T a[GS][BM * BK];
  alignas(1024) T b[GS][128 * BK];
  alignas(1024) T buf[EW][epi_bufs(MODE)][32 * kStageRow];
  float sums[MODE == kDh ? 2 : 1][MODE == kDh ? 4 : 1][MODE == kDh ? 512 : 1];  // [tile parity][32 rows][column]
  uint64_t full[GS], empty[GS];
  uint64_t tmem_full[2], tmem_empty[2];
  uint64_t in_full[EW];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
};

// f[j] += bias[nb + j] for the columns below N
__device__ __forceinline__ void add_bias32(const void* p, int dtype, int64_t nb, int64_t N, float* f) {
  if (nb + 32 <= N && (((reinterpret_cast<uintptr_t>(p)) & 15) == 0)) {
    if (dtype == kF32) {
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + nb) + v);
        f[4 * v] += b.x;
        f[4 * v + 1] += b.y;
        f[4 * v + 2] += b.z;
        f[4 * v + 3] += b.w;
      }
    } else {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float b[8];
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + nb) + v);
        if (dtype == kBF16)
          unpack8<__nv_bfloat16>(w, b);
        else
          unpack8<__half>(w, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[8 * v + j] += b[j];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (nb + j < N) f[j] += ld_bias(p, dtype, nb + j);
  }
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
__device__ __forceinline__ void bulk_wait_read_3() { asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory"); }

// named barrier that also ANDs a predicate over its threads
__device__ __forceinline__ bool bar_and(int id, int threads, bool v) {
  uint32_t out;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, %3, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(out)
      : "r"(v ? 1u : 0u), "r"(threads), "r"(id)
      : "memory");
  return out != 0;
}

// this lane's row of a 32 x 32 tile into the warp's next buffer (ring of BUFS), then one TMA store
template <typename T, int BUFS>
__device__ __forceinline__ void ring_store(const CUtensorMap* map, const float* f, T (*buf)[32 * kStageRow], int lane,
                                           int64_t nb, int64_t row_base, uint32_t& ring, int expert = -1) {
  T* b = buf[ring & (BUFS - 1)];
  if (lane == 0) {  // at most BUFS - 1 later stores pending: this buffer's has been read
    if (BUFS == 4)
      bulk_wait_read_3();
    else
      bulk_wait_read_1();
  }
  __syncwarp();
#pragma unroll
  for (int v = 0; v < 4; ++v) *reinterpret_cast<uint4*>(b + stg_off(lane, v)) = pack8<T>(&f[8 * v]);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    if (expert >= 0)
      tma_store_3d(map, b, (int)nb, (int)row_base, expert);
    else
      tma_store_2d(map, b, (int)nb, (int)row_base);
  }
  ++ring;
}

// A 32 x 32 tile of a weight gradient by plain stores: fp32 (added to what is there), or 16-bit rows that are not
// 16-byte aligned.  The lanes' rows are turned through `t` (4 KB, element (r, c) at 32 r + (c ^ r): conflict-free
// both ways), so that each store is a row segment.  What is added to is loaded first, 32 rows at once: a load behind a
// store that might alias it waits.
template <typename T>
__device__ __forceinline__ void dw_tile_store(const DwSeg& p, float* t, int64_t row_base, int64_t nb, const float* f,
                                              int lane, int expert) {
  const int64_t col = nb + lane, at = (expert * p.M + row_base) * p.ldd + col;
  const int rows = col < p.N ? (int)(p.M - row_base < 32 ? p.M - row_base : 32) : 0;
  if (lane == 0) bulk_wait_read_0();  // an earlier tile may still leave from these buffers
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) t[32 * lane + (j ^ lane)] = f[j];
  float old[32];
  if (p.out_f32) {
    float* d = reinterpret_cast<float*>(p.D) + at;
#pragma unroll
    for (int r = 0; r < 32; ++r) old[r] = p.accumulate && r < rows ? d[r * p.ldd] : 0.f;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (r < rows) d[r * p.ldd] = old[r] + t[32 * r + (lane ^ r)];
  } else {
    T* d = reinterpret_cast<T*>(p.D) + at;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (r < rows) d[r * p.ldd] = from_f<T>(t[32 * r + (lane ^ r)]);
  }
  __syncwarp();
}

// The same turn for a 16-bit result [M, N] whose rows are not 16-byte aligned, with its residual: its 32 loads leave
// before the turn, since a load behind a store that might alias it waits (20003 x 1001 x 2669: 115 us; 249 us
// with load and store row by row)
template <typename T>
__device__ __forceinline__ void plain_tile_store(const GatedParams& p, float* t, int64_t row_base, int64_t nb,
                                                 const float* f, int lane) {
  const int64_t col = nb + lane;
  const int rows = col < p.N ? (int)(p.M - row_base < 32 ? p.M - row_base : 32) : 0;
  T res[32];
  if (p.res) {
    const T* q = reinterpret_cast<const T*>(p.res) + row_base * p.ldres + col;
#pragma unroll
    for (int r = 0; r < 32; ++r) res[r] = r < rows ? q[r * p.ldres] : from_f<T>(0.f);
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) t[32 * lane + (j ^ lane)] = f[j];
  __syncwarp();
  T* d = reinterpret_cast<T*>(p.D) + row_base * p.ldd + col;
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    float v = t[32 * r + (lane ^ r)];
    if (p.res) v += to_f(res[r]);
    if (r < rows) d[r * p.ldd] = from_f<T>(v);
  }
}

// a tile of all weights' -> its weight, and the tile within it
struct DwList {
  DwSeg seg[kDwWeights];
};
template <typename P>
__device__ __forceinline__ void dw_place(const P& p, int64_t v, int& seg, int64_t& tile, int64_t& n_tiles) {
  seg = v < p.seg[0].end ? 0 : v < p.seg[1].end ? 1 : 2;
  tile = v - (seg ? p.seg[seg - 1].end : 0);
  n_tiles = p.seg[seg].n_tiles;
}

// The cut tiles' partials added in piece order: one block a tile row, one thread four columns.
template <typename T>
__global__ void dw_sum_kernel(const float* __restrict__ ws, const __grid_constant__ DwList l, int64_t first, int rem,
                              int splits) {
  const int r = blockIdx.x >> 8, row_in = blockIdx.x & 255;
  int seg;
  int64_t t, nt;
  dw_place(l, first + r, seg, t, nt);
  const DwSeg& p = l.seg[seg];
  const int64_t row = (t / nt) * BM2 + row_in, col = (t % nt) * BN2 + 4 * threadIdx.x;
  if (row >= p.M || col >= p.N) return;
  const float* src = ws + ((int64_t)r * BM2 + row_in) * BN2 + 4 * threadIdx.x;
  float4 a = __ldcs(reinterpret_cast<const float4*>(src));
  for (int k = 1; k < splits; ++k) {
    const float4 b = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)k * rem * BM2 * BN2));
    a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
  }
  const float f[4] = {a.x, a.y, a.z, a.w};
  for (int j = 0; j < 4 && col + j < p.N; ++j) {
    if (p.out_f32) {
      float* d = reinterpret_cast<float*>(p.D) + row * p.ldd + col + j;
      *d = p.accumulate ? *d + f[j] : f[j];
    } else {
      reinterpret_cast<T*>(p.D)[row * p.ldd + col + j] = from_f<T>(f[j]);
    }
  }
}

template <typename T, int MODE, bool GROUPED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * epi_warps(MODE), 1)
    gated_kernel(const __grid_constant__ GatedParams p, uint32_t idesc, int* err) {
  constexpr bool kMnA = MODE == kDw;                                // A read as stored, M contiguous
  constexpr bool kMnB = MODE == kDh || MODE == kDx || MODE == kDw;  // B read as stored, N contiguous
  constexpr int kCols = MODE == kUp ? 128 : 256;                    // result columns of a pair tile
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int EW = epi_warps(MODE), GS = stages(MODE);
  auto& S = *reinterpret_cast<SmemG<T, MODE>*>(base);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int64_t m_tiles = GROUPED && MODE != kDw ? __ldg(p.group.tiles) : (p.M + BM2 - 1) / BM2;
  const int64_t n_tiles = (p.N + kCols - 1) / kCols;
  const int64_t num_tiles = MODE == kDw ? p.direct : m_tiles * n_tiles;
  volatile int* abort_flag = &S.abort_flag;

  if (threadIdx.x == 64) {
    prefetch_map(&p.a0);
    prefetch_map(&p.b0);
    if (MODE != kDown && MODE != kDh) prefetch_map(&p.b1);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < GS; ++s) {
      mbar_init(&S.full[s], 1);
      mbar_init(&S.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&S.tmem_full[a], 1);
      mbar_init(&S.tmem_empty[a], 2 * EW);
    }
    for (int w = 0; w < EW; ++w) mbar_init(&S.in_full[w], 1);
    mbar_init(&S.done, 1);
    S.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)),
                 "r"(2 * BN2));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = S.tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      const uint32_t full_leader = map_rank(&S.full[0], 0);
      int stage = 0;
      uint32_t phase = 0;
      GUnit un;
      for (int64_t i = 0; gated_unit<MODE, GROUPED>(p, num_tiles, pair, npairs, i, un) && !*abort_flag; ++i) {
        int seg = 0;
        int64_t tile = un.tile, nt = n_tiles;
        if (MODE == kDw) dw_place(p, un.tile, seg, tile, nt);
        const int m0 = (int)((tile / nt) * BM2) + (int)rank * BM;
        const int nb0 = (int)((tile % nt) * kCols) + (MODE == kUp ? 0 : (int)rank * 128);
        for (int kb = un.kb0; kb < un.kb1; ++kb) {
          if (!mbar_wait(&S.empty[stage], phase ^ 1, abort_flag, err)) break;
          if (rank == 0) mbar_expect_tx(&S.full[stage], (uint32_t)(2 * (BM + 128) * BK * sizeof(T)));
          const uint32_t fb = full_leader + 8u * stage;
          const bool second = MODE == kDx && kb >= p.kb0;
          const int k0 = (second ? kb - p.kb0 : kb) * BK;
          const auto load_b = [&](void* dst, const CUtensorMap* m, int c0, int c1) {
            if (GROUPED && MODE != kDw)
              tma_load_3d_pair(dst, m, fb, c0, c1, un.expert);
            else
              tma_load_2d_pair(dst, m, fb, c0, c1);
          };
          if (kMnA) {
            const CUtensorMap* ma = seg == 0 ? &p.a0 : seg == 1 ? &p.a1 : &p.a2;
            tma_load_2d_pair(&S.a[stage][0], ma, fb, m0, k0);
            tma_load_2d_pair(&S.a[stage][64 * BK], ma, fb, m0 + 64, k0);
          } else {
            tma_load_2d_pair(S.a[stage], second ? &p.a1 : &p.a0, fb, k0, m0);
          }
          if (kMnB) {
            const CUtensorMap* mb = second || seg == 2 ? &p.b1 : &p.b0;
            load_b(&S.b[stage][0], mb, nb0, k0);
            load_b(&S.b[stage][64 * BK], mb, nb0 + 64, k0);
          } else {
            load_b(S.b[stage], MODE == kUp && rank ? &p.b1 : &p.b0, k0, nb0);
          }
          if (++stage == GS) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (leader)
    if (lane == 0 && rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      GUnit un;
      for (int64_t i = 0; gated_unit<MODE, GROUPED>(p, num_tiles, pair, npairs, i, un) && !*abort_flag; ++i) {
        if (!mbar_wait(&S.tmem_empty[acc], acc_phase ^ 1, abort_flag, err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN2);
        bool ok = true;
        for (int kb = un.kb0; kb < un.kb1; ++kb) {
          if (!mbar_wait(&S.full[stage], phase, abort_flag, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t db = kMnB ? smem_desc_mn(&S.b[stage][k * 16 * 64], 64 * BK * (uint32_t)sizeof(T))
                                     : smem_desc_sw128(&S.b[stage][k * 16]);
            const uint64_t da = kMnA ? smem_desc_mn(&S.a[stage][k * 16 * 64], 64 * BK * (uint32_t)sizeof(T))
                                     : smem_desc_sw128(&S.a[stage][k * 16]);
            umma2_f16(d_tmem, da, db, idesc, (kb > un.kb0 || k > 0) ? 1u : 0u);
          }
          umma2_commit_both(&S.empty[stage]);
          if (++stage == GS) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        umma2_commit_both(&S.tmem_full[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    const int ew = warp - 2;
    const int q = warp & 3;
    const int part = ew >> 2;            // which share of the result's columns this warp drains
    constexpr int kShare = kCols / (EW / 4);
    constexpr int kChunks = kShare / 32;
    T(*buf)[32 * kStageRow] = S.buf[ew];
    uint64_t* in_full = &S.in_full[ew];
    const uint32_t empty_leader = map_rank(&S.tmem_empty[0], 0);
    uint32_t ring = 0;
    uint32_t in_phase = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool pending = false;  // input tiles issued and not waited for
    bool ok = true;
    GUnit un;
    for (int64_t i = 0; ok && gated_unit<MODE, GROUPED>(p, num_tiles, pair, npairs, i, un); ++i) {
      int seg = 0;
      int64_t tile = un.tile, nt = n_tiles;
      if (MODE == kDw) dw_place(p, un.tile, seg, tile, nt);
      const int64_t M = MODE == kDw ? p.seg[seg].M : p.M, N = MODE == kDw ? p.seg[seg].N : p.N;
      const int64_t row_base = (tile / nt) * BM2 + (int64_t)rank * BM + q * 32;
      const int64_t n0 = (tile % nt) * kCols + part * kShare;
      const bool rows = row_base < M;  // warp-uniform; a tile's lower rows may be past the end
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN2 + part * kShare);
      // kDh: g and u of chunk c into the warp's two buffers
      auto issue_gu = [&](int c) {
        const int64_t nb = n0 + 32 * c;
        if (c >= kChunks || !rows || nb >= p.N) return;
        if (lane == 0) {
          bulk_wait_read_0();  // the stores that last used these buffers have read them
          mbar_expect_tx(in_full, 2 * 32 * kStageRow * sizeof(T));
          tma_load_2d(buf[0], &p.in0, in_full, (int)nb, (int)row_base);
          tma_load_2d(buf[1], &p.in1, in_full, (int)nb, (int)row_base);
        }
        pending = true;
      };
      if (MODE == kDh) issue_gu(0);
      if (MODE == kDown && p.has_res && rows && n0 < p.N) {
        if (lane == 0) {
          bulk_wait_read_0();
          uint32_t chunks = 0;
          for (int c = 0; c < kChunks; ++c) chunks += n0 + 32 * c < p.N;
          mbar_expect_tx(in_full, chunks * 32 * kStageRow * (uint32_t)sizeof(T));
          for (int c = 0; c < kChunks; ++c)
            if (n0 + 32 * c < p.N) tma_load_2d(buf[c], &p.in0, in_full, (int)(n0 + 32 * c), (int)row_base);
        }
        pending = true;
      }
      if (!mbar_wait(&S.tmem_full[acc], acc_phase, abort_flag, err)) {
        if (MODE != kDh) break;
        ok = false;  // kDh: the warps leave together, below
      }
      tc_fence_after();
      if (MODE == kUp) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int64_t nb = n0 + 32 * c;
          if (!rows || nb >= p.N) break;
          uint32_t rg[32], ru[32];
          tmem_ld32_async(t_row + (uint32_t)(32 * c), rg);
          tmem_ld32_async(t_row + (uint32_t)(128 + 32 * c), ru);
          tmem_wait_ld(rg);
          tmem_wait_ld(ru);
          float* g = reinterpret_cast<float*>(rg);
          float* u = reinterpret_cast<float*>(ru);
          if (p.bias0) add_bias32(p.bias0, p.bias_dtype, nb, p.N, g);
          if (p.bias1) add_bias32(p.bias1, p.bias_dtype, nb, p.N, u);
          if (p.save) {
            ring_store<T, epi_bufs(MODE)>(&p.out1, g, buf, lane, nb, row_base, ring);
            ring_store<T, epi_bufs(MODE)>(&p.out2, u, buf, lane, nb, row_base, ring);
          }
          if (p.act == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_parts(g[j], 0).val;
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_parts(g[j], 1).val;
          }
          ring_store<T, epi_bufs(MODE)>(&p.out0, u, buf, lane, nb, row_base, ring);
        }
      } else if (MODE == kDh) {
#pragma unroll 1
        for (int c = 0; c < kChunks && ok; ++c) {
          const int64_t nb = n0 + 32 * c;
          float* sums = &S.sums[i & 1][q][part * kShare + 32 * c];
          if (!rows || nb >= p.N) {
            if (p.sums) sums[lane] = sums[lane + 256] = 0.f;
            continue;
          }
          uint32_t r[32];
          tmem_ld32_async(t_row + (uint32_t)(32 * c), r);
          if (!mbar_wait(in_full, in_phase, abort_flag, err)) {
            ok = false;
            tmem_wait_ld(r);
            break;
          }
          in_phase ^= 1u;
          pending = false;
          tmem_wait_ld(r);
          T* bg = buf[0];
          T* bu = buf[1];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float g[8], u[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(bg + stg_off(lane, v)), g);
            unpack8<T>(*reinterpret_cast<const uint4*>(bu + stg_off(lane, v)), u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float d = __uint_as_float(r[8 * v + j]);
              const ActParts a = act_parts(g[j], p.act);
              g[j] = d * u[j] * a.slope;
              u[j] = d * a.val;
            }
            *reinterpret_cast<uint4*>(bg + stg_off(lane, v)) = pack8<T>(g);
            *reinterpret_cast<uint4*>(bu + stg_off(lane, v)) = pack8<T>(u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.out0, bg, (int)nb, (int)row_base);
            tma_store_2d(&p.out1, bu, (int)nb, (int)row_base);
          }
          if (p.sums) {
            // the tiles' column sums, of the rounded values that dx and the weights' gradients are made of too (of the
            // fp32 ones, by shuffles before they are packed: 466 us against 437 at 64800 x 1024 x 2736): lane l adds columns 2 (l % 16), 2 (l % 16) + 1 of the rows of l / 16's parity
            float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int at = stg_off(2 * k + (lane >> 4), (lane & 15) >> 2) + 2 * (lane & 3);
              float x[2];
              unpack2(*reinterpret_cast<const uint32_t*>(bg + at), x, T());
              a[0] += x[0];
              a[1] += x[1];
              unpack2(*reinterpret_cast<const uint32_t*>(bu + at), x, T());
              a[2] += x[0];
              a[3] += x[1];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] += __shfl_xor_sync(0xffffffffu, a[k], 16);
            if (lane < 16) {
              *reinterpret_cast<float2*>(sums + 2 * lane) = make_float2(a[0], a[1]);
              *reinterpret_cast<float2*>(sums + 256 + 2 * lane) = make_float2(a[2], a[3]);
            }
            __syncwarp();  // the buffers have been read: the next tiles may land in them
          }
          issue_gu(c + 1);
        }
      } else {
        if (MODE == kDown && pending) {
          if (!mbar_wait(in_full, in_phase, abort_flag, err)) break;
          in_phase ^= 1u;
          pending = false;
        }
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int64_t nb = n0 + 32 * c;
          if (!rows || nb >= N) break;
          uint32_t r[32];
          tmem_ld32(t_row + (uint32_t)(32 * c), r);
          float* f = reinterpret_cast<float*>(r);
          if (MODE == kDw && un.slot >= 0) {  // a piece's partial: this lane's row, 32 columns
            float* w = p.ws + ((un.slot * BM2 + (int64_t)rank * BM + q * 32 + lane) * BN2 + part * kShare + 32 * c);
#pragma unroll
            for (int v = 0; v < 8; ++v)
              __stcg(reinterpret_cast<float4*>(w) + v, make_float4(f[4 * v], f[4 * v + 1], f[4 * v + 2], f[4 * v + 3]));
            continue;
          }
          if (GROUPED && MODE == kDw && un.kb0 == un.kb1) {  // no product was made
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = 0.f;
          }
          if (MODE == kDw && !p.seg[seg].tma_out) {
            dw_tile_store<T>(p.seg[seg], reinterpret_cast<float*>(buf[0]), row_base, nb, f, lane, un.expert);
            continue;
          }
          if (GROUPED && MODE == kDw) {
            ring_store<T, epi_bufs(MODE)>(seg == 0 ? &p.out0 : seg == 1 ? &p.out1 : &p.out2, f, buf, lane, nb, row_base,
                                          ring, un.expert);
            continue;
          }
          if (MODE == kDown && p.bias0) add_bias32(p.bias0, p.bias_dtype, nb, p.N, f);
          if ((MODE == kDown || MODE == kDx) && p.plain) {
            plain_tile_store<T>(p, reinterpret_cast<float*>(buf[0]), row_base, nb, f, lane);
            continue;
          }
          if (MODE == kDown && p.has_res) {
            T* b = buf[c];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              float x[8];
              unpack8<T>(*reinterpret_cast<const uint4*>(b + stg_off(lane, v)), x);
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] += f[8 * v + j];
              *reinterpret_cast<uint4*>(b + stg_off(lane, v)) = pack8<T>(x);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(&p.out0, b, (int)nb, (int)row_base);
          } else {
            ring_store<T, epi_bufs(MODE)>(seg == 0 ? &p.out0 : seg == 1 ? &p.out1 : &p.out2, f, buf, lane, nb, row_base, ring);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive_cluster(empty_leader + 8u * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
      if constexpr (MODE == kDh) {
        if (!p.sums) continue;
        // the four 32-row groups of these columns; the other parity's sums are untouched until every warp has
        // been through the next tile's barrier.  A warp that gave up makes all of them leave.
        ok = bar_and(1 + part, 128, ok);
        const int t = q * 32 + lane;  // 64 columns of dg, then of du
        const int col = part * kShare + (t & 63);
        const int64_t at = (tile % n_tiles) * kCols + col;
        if (ok && at < p.N) {
          const float(*v)[512] = S.sums[i & 1];
          const int k = col + 256 * (t >> 6);
          const int64_t m = (tile / n_tiles) * 2 + rank;
          p.sums[m * 2 * p.sums_half + (t >> 6) * p.sums_half + at] = ((v[0][k] + v[1][k]) + v[2][k]) + v[3][k];
        }
      }
    }
    if (lane == 0) {
      bulk_wait_all();
      // after an abort, input loads still in flight land before the shared memory is released
      if (pending) {
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(in_full, in_phase) && globaltimer() - t0 < kWaitBudgetNs) {
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    mbar_arrive_cluster(map_rank(&S.done, rank ^ 1u));
    int never = 0;
    mbar_wait(&S.done, 0, &never, err);
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN2));
}

// Whole waves of tiles, and how to cut the tiles that are left (none if they fill a wave well).  In k-block
// steps (0.31 us a pair): a cut costs its longest pair, plus 0.26 steps a partial (256 KB written and read
// over the device) and about 15 for the second kernel and the shorter units.
static DwPlan dw_plan(int64_t tiles, int64_t K) {
  const int64_t pairs = sm_count() / 2, kb = (K + BK - 1) / BK, left = tiles % pairs;
  DwPlan best = {tiles, 0, 1};
  double best_cost = (double)kb;  // one more wave
  if (left == 0) return best;
  for (int s = 2; s <= 16 && kb / s >= 4; ++s) {
    const double cost = (double)((left * s + pairs - 1) / pairs * ((kb + s - 1) / s)) + 0.26 * left * s + 15.0;
    if (cost < best_cost) {
      best_cost = cost;
      best = {tiles - left, (int)left, s};
    }
  }
  return best;
}
static int64_t dw_tiles(const GatedDwArgs::Weight& w) {
  return w.D ? ((w.M + BM2 - 1) / BM2) * ((w.N + BN2 - 1) / BN2) : 0;
}

// launches gated_kernel for `units` tiles of work; `fill` encodes the operands (false: refused)
template <typename T, int MODE, bool GROUPED, typename Fill>
static cudaError_t launch_pairs(int64_t units, int dtype, cudaStream_t s, GatedParams& p, Fill fill) {
  const size_t smem = sizeof(SmemG<T, MODE>) + 1024;
  auto k = gated_kernel<T, MODE, GROUPED>;
  // on each call: the attribute belongs to the current device, and a runtime call has to make that device's
  // context current on this thread (an autograd thread may not have one yet) before the maps are encoded
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  memset(&p, 0, sizeof(p));
  if (!fill()) return cudaErrorInvalidValue;
  constexpr bool mn = MODE == kDh || MODE == kDx || MODE == kDw;
  const uint32_t fmt = dtype == kBF16 ? 1u : 0u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (MODE == kDw ? 1u << 15 : 0u) | (mn ? 1u << 16 : 0u) |
                         ((uint32_t)(BN2 >> 3) << 17) | ((uint32_t)(BM2 >> 4) << 24);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(64 + 32 * epi_warps(MODE), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(sm_count() & ~1, 1, 1);
  static int max_pairs = 0;
  if (!max_pairs) {
    int n = 0;
    NSW_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, k, &cfg));
    max_pairs = n > 0 ? n : 1;
  }
  const int64_t pairs = std::min<int64_t>(units, max_pairs);
  cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
  NSW_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, p, idesc, device_error_flag()));
  return cudaGetLastError();
}

template <typename T, int MODE, bool GROUPED = false>
static cudaError_t launch_gated(const GatedArgs& a, cudaStream_t s) {
  constexpr int cols = MODE == kUp ? 128 : 256;
  const int64_t tiles = ((a.M + BM2 - 1) / BM2) * ((a.N + cols - 1) / cols);
  GatedParams p;
  return launch_pairs<T, MODE, GROUPED>(tiles, a.dtype, s, p, [&]() {
    constexpr bool mn = MODE == kDh || MODE == kDx;
    bool ok = make_map(&p.a0, a.a0, a.M, a.K, a.lda, BM, a.dtype);
    if (MODE == kDx) ok = ok && make_map(&p.a1, a.a1, a.M, a.K, a.lda, BM, a.dtype);
    if (GROUPED) {
      p.group = {a.groups->tiles, a.groups->rows, a.groups->experts};
      const int64_t e = a.groups->experts, rows = mn ? a.K : a.N, cols_ = mn ? a.N : a.K;
      const int bc = 64, br = mn ? BK : 128;  // a K-major box is 64 deep, 128 rows; an MN-major one 64 by 64
      ok = ok && make_map_3d(&p.b0, a.b0, e, rows, cols_, a.ldb0, bc, br, CU_TENSOR_MAP_SWIZZLE_128B, a.dtype);
      if (MODE == kUp || MODE == kDx)
        ok = ok && make_map_3d(&p.b1, a.b1, e, rows, cols_, a.ldb1, bc, br, CU_TENSOR_MAP_SWIZZLE_128B, a.dtype);
    } else if (mn) {
      ok = ok && make_map_mn(&p.b0, a.b0, a.K, a.N, a.ldb0, a.dtype);
      if (MODE == kDx) ok = ok && make_map_mn(&p.b1, a.b1, a.K, a.N, a.ldb1, a.dtype);
    } else {
      ok = ok && make_map(&p.b0, a.b0, a.N, a.K, a.ldb0, 128, a.dtype);
      if (MODE == kUp) ok = ok && make_map(&p.b1, a.b1, a.N, a.K, a.ldb1, 128, a.dtype);
    }
    const auto odd = [](const void* q, int64_t ld) { return ld % 8 != 0 || (reinterpret_cast<uintptr_t>(q) & 15) != 0; };
    p.plain = (MODE == kDown || MODE == kDx) && (odd(a.out0, a.ldout) || (a.in0 && odd(a.in0, a.ldin)));
    if (p.plain) {
      p.D = a.out0;
      p.ldd = a.ldout;
      p.res = a.in0;
      p.ldres = a.ldin;
    }
    if (a.in0 && !p.plain) ok = ok && make_store_map(&p.in0, const_cast<void*>(a.in0), a.M, a.N, a.ldin, a.dtype);
    if (a.in1) ok = ok && make_store_map(&p.in1, const_cast<void*>(a.in1), a.M, a.N, a.ldin, a.dtype);
    if (!p.plain) ok = ok && make_store_map(&p.out0, a.out0, a.M, a.N, a.ldout, a.dtype);
    if (a.out1) ok = ok && make_store_map(&p.out1, a.out1, a.M, a.N, a.ldaux, a.dtype);
    if (a.out2) ok = ok && make_store_map(&p.out2, a.out2, a.M, a.N, a.ldaux, a.dtype);
    p.M = a.M;
    p.N = a.N;
    p.kb0 = (int)((a.K + BK - 1) / BK);
    p.kb = MODE == kDx ? 2 * p.kb0 : p.kb0;
    p.bias0 = a.bias0;
    p.bias1 = a.bias1;
    p.bias_dtype = a.bias_dtype;
    p.act = a.act;
    p.sums = MODE == kDh ? a.sums : nullptr;
    p.sums_half = a.sums_half;
    p.save = MODE == kUp && a.out1 != nullptr;
    p.has_res = MODE == kDown && a.in0 != nullptr && !p.plain;
    return ok;
  });
}

template <typename T>
static cudaError_t launch_dw(const GatedDwArgs& a, cudaStream_t s) {
  int64_t tiles = 0;
  for (const auto& w : a.w) tiles += dw_tiles(w);
  const DwPlan plan = dw_plan(tiles, a.T);
  if (plan.rem > 0 && !a.ws) return cudaErrorInvalidValue;
  GatedParams p;
  NSW_CUDA_CHECK((launch_pairs<T, kDw, false>(
      std::max<int64_t>(plan.direct, (int64_t)plan.rem * plan.splits), a.dtype, s, p, [&]() {
        // a weight without tiles has the maps of one with them: valid, and not read through
        const auto with = [&](int i, int j) -> const GatedDwArgs::Weight& {
          return a.w[i].D ? a.w[i] : a.w[j].D ? a.w[j] : a.w[3 - i - j];
        };
        const GatedDwArgs::Weight w[kDwWeights] = {with(0, 1), with(1, 0), with(2, 0)};
        bool ok = make_map_mn(&p.a0, w[0].a, a.T, w[0].M, w[0].lda, a.dtype) &&
                  make_map_mn(&p.a1, w[1].a, a.T, w[1].M, w[1].lda, a.dtype) &&
                  make_map_mn(&p.a2, w[2].a, a.T, w[2].M, w[2].lda, a.dtype) &&
                  make_map_mn(&p.b0, w[0].b, a.T, w[0].N, w[0].ldb, a.dtype) &&
                  make_map_mn(&p.b1, w[2].b, a.T, w[2].N, w[2].ldb, a.dtype);
        CUtensorMap* out[kDwWeights] = {&p.out0, &p.out1, &p.out2};
        int64_t end = 0;
        for (int i = 0; i < kDwWeights; ++i) {
          end += dw_tiles(a.w[i]);
          const bool tma = a.w[i].D && !w[i].out_f32 && w[i].N % 8 == 0 && (reinterpret_cast<uintptr_t>(w[i].D) & 15) == 0;
          p.seg[i] = {end, (w[i].N + BN2 - 1) / BN2, w[i].M, w[i].N, w[i].N, w[i].D, w[i].out_f32, w[i].accumulate, tma};
          if (tma) ok = ok && make_store_map(out[i], w[i].D, w[i].M, w[i].N, w[i].N, a.dtype);
        }
        p.kb = (int)((a.T + BK - 1) / BK);
        p.direct = plan.direct;
        p.rem = plan.rem;
        p.splits = plan.splits;
        p.ws = a.ws;
        return ok;
      })));
  if (plan.rem > 0) {
    DwList l;
    for (int i = 0; i < kDwWeights; ++i) l.seg[i] = p.seg[i];
    dw_sum_kernel<T><<<plan.rem * 256, 64, 0, s>>>(a.ws, l, plan.direct, plan.rem, plan.splits);
  }
  return cudaGetLastError();
}

// The grouped weight gradients: every expert's matrices, each a product over its own rows
template <typename T>
static cudaError_t launch_dw_grouped(const GatedDwArgs& a, cudaStream_t s) {
  const int64_t e = a.groups->experts;
  int64_t tiles = 0;
  for (const auto& w : a.w) tiles += e * dw_tiles(w);
  GatedParams p;
  return launch_pairs<T, kDw, true>(tiles, a.dtype, s, p, [&]() {
    const auto with = [&](int i, int j) -> const GatedDwArgs::Weight& {  // as in launch_dw
      return a.w[i].D ? a.w[i] : a.w[j].D ? a.w[j] : a.w[3 - i - j];
    };
    const GatedDwArgs::Weight w[kDwWeights] = {with(0, 1), with(1, 0), with(2, 0)};
    bool ok = make_map_mn(&p.a0, w[0].a, a.T, w[0].M, w[0].lda, a.dtype) &&
              make_map_mn(&p.a1, w[1].a, a.T, w[1].M, w[1].lda, a.dtype) &&
              make_map_mn(&p.a2, w[2].a, a.T, w[2].M, w[2].lda, a.dtype) &&
              make_map_mn(&p.b0, w[0].b, a.T, w[0].N, w[0].ldb, a.dtype) &&
              make_map_mn(&p.b1, w[2].b, a.T, w[2].N, w[2].ldb, a.dtype);
    CUtensorMap* out[kDwWeights] = {&p.out0, &p.out1, &p.out2};
    int64_t end = 0;
    for (int i = 0; i < kDwWeights; ++i) {
      end += e * dw_tiles(a.w[i]);
      const bool tma = a.w[i].D && !w[i].out_f32 && w[i].N % 8 == 0 && (reinterpret_cast<uintptr_t>(w[i].D) & 15) == 0;
      p.seg[i] = {end, (w[i].N + BN2 - 1) / BN2, w[i].M, w[i].N, w[i].N, w[i].D, w[i].out_f32, w[i].accumulate, tma};
      if (tma)
        ok = ok && make_map_3d(out[i], w[i].D, e, w[i].M, w[i].N, w[i].N, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B, a.dtype);
    }
    p.group = {a.groups->tiles, a.groups->rows, e};
    p.direct = end;
    return ok;
  });
}

// ============================================================================ split-depth form
// The same four products where gated_kernel would have too few tiles to fill the device (a few hundred rows,
// or few output columns with a long depth).  The weights are the MMA's M operand (128 of their rows, in kUp 64
// rows of Wg and the same 64 of Wu) and NTOK tokens its N operand, one CTA per tile and depth slice; the
// slices of a tile are the CTAs of a cluster.  Each CTA leaves its fp32 partial in its shared memory (over
// the drained pipeline stages), and after a cluster barrier every CTA adds its share of the tile over the
// slices in order (deterministic) and does the epilogue with plain, row-contiguous accesses.
//   warp 0: TMA producer; warp 1: MMA issuer; warps 2-9: TMEM to shared memory; all: the final sums.
// In a dependent launch the weight tiles of the first stages are on their way before the wait for the kernel
// that writes the tokens.
constexpr int kSplitThreads = 320;  // a multiple of a tile's quads: a thread's columns stay the same
constexpr int kMaxSlices = 8;  // the largest portable cluster

__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
  float4 o;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w)
               : "r"(at)
               : "memory");
  return o;
}

struct SplitParams {
  CUtensorMap w0, w1, x0, x1;
  int64_t M, N;
  int kb0, kb;
  const void *bias0, *bias1, *in0, *in1;
  void *out0, *out1, *out2;
  int64_t ldin, ldout, ldaux;
  int bias_dtype, act, dependent;
  const int* tiles;  // grouped: the number of token tiles, then each one's expert
};

template <typename T, int NTOK, int STAGES>
struct SmemS {
  union {
    struct {
      alignas(1024) T w[STAGES][BM * BK];
      alignas(1024) T x[STAGES][NTOK * BK];
    };
    float part[NTOK][BM];  // [token][weight row]
  };
  uint64_t full[STAGES], empty[STAGES];
  uint64_t tmem_full;
  uint32_t tmem_base;
  int abort_flag;
};

// four consecutive 16-bit columns of a row, those of the first `left` (zeros after)
__device__ __forceinline__ uint2 load4(const uint16_t* p, int64_t left, bool vec) {
  if (vec && left >= 4) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  return make_uint2(w[0], w[1]);
}
template <typename T>
__device__ __forceinline__ void unpack4(uint2 w, float* f) {
  unpack2(w.x, f, T());
  unpack2(w.y, f + 2, T());
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t left, bool vec, const float* f) {
  if (vec && left >= 4) {
    T h[4] = {from_f<T>(f[0]), from_f<T>(f[1]), from_f<T>(f[2]), from_f<T>(f[3])};
    uint2 w;
    memcpy(&w, h, 8);
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = from_f<T>(f[j]);
  }
}

template <typename T, int MODE, int NTOK, int STAGES>
__global__ void __launch_bounds__(kSplitThreads, NTOK <= 64 ? 2 : 1) split_kernel(const __grid_constant__ SplitParams p, uint32_t idesc,
                                                              int* err) {
  constexpr bool kMn = MODE == kDh || MODE == kDx;
  constexpr int kUnits = MODE == kUp ? 64 : 128;  // output columns of a tile
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using Smem = SmemS<T, NTOK, STAGES>;
  auto& S = *reinterpret_cast<Smem*>(base);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = blockIdx.y, slices = gridDim.y;
  const int64_t n0 = (int64_t)blockIdx.x * kUnits, m0 = (int64_t)blockIdx.z * NTOK;
  const int kb_begin = (int)((int64_t)slice * p.kb / slices), kb_end = (int)((int64_t)(slice + 1) * p.kb / slices);
  const int nkb = kb_end - kb_begin;
  volatile int* abort_flag = &S.abort_flag;
  int w_row = 0;  // the expert's first row of the weights
  if (MODE == kUp || MODE == kDown)
    if (p.tiles) {
      // (written two kernels ago: by way of L2, past what an L1 may hold of its earlier contents)
      if ((int)blockIdx.z >= __ldcg(p.tiles)) {  // the whole cluster; nobody overtakes the kernel before
        if (p.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
      }
      w_row = __ldcg(p.tiles + 1 + blockIdx.z) * (int)p.N;
    }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 64) {
    prefetch_map(&p.w0);
    prefetch_map(&p.x0);
    if (MODE == kUp || MODE == kDx) prefetch_map(&p.w1);
    if (MODE == kDx) prefetch_map(&p.x1);
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&S.full[s], 1);
      mbar_init(&S.empty[s], 1);
    }
    mbar_init(&S.tmem_full, 1);
    S.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&S.tmem_base)),
                 "r"(NTOK));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = S.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      auto load_w = [&](int i) {
        const int kb = kb_begin + i, st = i % STAGES;
        const bool second = MODE == kDx && kb >= p.kb0;
        const int k0 = (second ? kb - p.kb0 : kb) * BK;
        const CUtensorMap* m = second ? &p.w1 : &p.w0;
        if (kMn) {
          tma_load_2d(&S.w[st][0], m, &S.full[st], (int)n0, k0);
          tma_load_2d(&S.w[st][64 * BK], m, &S.full[st], (int)n0 + 64, k0);
        } else if (MODE == kUp) {
          tma_load_2d(&S.w[st][0], &p.w0, &S.full[st], k0, w_row + (int)n0);
          tma_load_2d(&S.w[st][64 * BK], &p.w1, &S.full[st], k0, w_row + (int)n0);
        } else {
          tma_load_2d(&S.w[st][0], m, &S.full[st], k0, w_row + (int)n0);
        }
      };
      auto load_x = [&](int i) {
        const int kb = kb_begin + i, st = i % STAGES;
        const bool second = MODE == kDx && kb >= p.kb0;
        tma_load_2d(&S.x[st][0], second ? &p.x1 : &p.x0, &S.full[st], (second ? kb - p.kb0 : kb) * BK, (int)m0);
      };
      constexpr uint32_t kBytes = (BM + NTOK) * BK * sizeof(T);
      const int first = nkb < STAGES ? nkb : STAGES;
      for (int i = 0; i < first; ++i) {
        mbar_expect_tx(&S.full[i], kBytes);
        load_w(i);
      }
      if (p.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int i = 0; i < first; ++i) load_x(i);
      int issued = first;
      for (; issued < nkb; ++issued) {
        const int st = issued % STAGES;
        if (!mbar_wait(&S.empty[st], (uint32_t)((issued / STAGES - 1) & 1), abort_flag, err)) break;
        mbar_expect_tx(&S.full[st], kBytes);
        load_w(issued);
        load_x(issued);
      }
      // every load has landed before the stages are reused (bounded; at once unless something gave up)
      for (int i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i) {
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(&S.full[i % STAGES], (uint32_t)((i / STAGES) & 1)) && globaltimer() - t0 < kWaitBudgetNs) {
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int i = 0; i < nkb; ++i) {
        const int st = i % STAGES;
        if (!mbar_wait(&S.full[st], (uint32_t)((i / STAGES) & 1), abort_flag, err)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          const uint64_t da = kMn ? smem_desc_mn(&S.w[st][k * 16 * 64], 64 * BK * (uint32_t)sizeof(T))
                                  : smem_desc_sw128(&S.w[st][k * 16]);
          umma_f16(tmem_base, da, smem_desc_sw128(&S.x[st][k * 16]), idesc, (i > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&S.empty[st]);
      }
      if (ok) umma_commit(&S.tmem_full);
    }
  }
  __syncwarp();
  // what the epilogue reads from global memory is on its way while the products run
  constexpr int kQuads = kUnits / 4;
  constexpr int kBatch = MODE == kUp ? 2 : 4;  // items whose loads are in flight together
  static_assert(kSplitThreads % kQuads == 0, "a thread's columns");
  const int tokens = (int)(p.M - m0 < NTOK ? p.M - m0 : NTOK);
  const int64_t col = n0 + 4 * (threadIdx.x % kQuads), left = p.N - col;
  const bool vec = ((p.ldout | p.ldaux | p.ldin) & 3) == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.out0) | reinterpret_cast<uintptr_t>(p.out1) |
                     reinterpret_cast<uintptr_t>(p.out2) | reinterpret_cast<uintptr_t>(p.in0) |
                     reinterpret_cast<uintptr_t>(p.in1)) & 7) == 0;
  const int step = slices * (kSplitThreads / kQuads);
  int t0 = (slice * kSplitThreads + threadIdx.x) / kQuads;
  if (p.dependent) asm volatile("griddepcontrol.wait;" ::: "memory");
  float b0[4] = {0.f, 0.f, 0.f, 0.f}, b1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (p.bias0 && j < left) b0[j] = ld_bias(p.bias0, p.bias_dtype, col + j);
    if (MODE == kUp && p.bias1 && j < left) b1[j] = ld_bias(p.bias1, p.bias_dtype, col + j);
  }
  uint2 in0[kBatch], in1[kBatch];
  auto fetch = [&](int first) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int tok = first + b * step;
      in0[b] = in1[b] = make_uint2(0, 0);
      if (tok >= tokens || left <= 0 || !p.in0) continue;
      const int64_t at = (m0 + tok) * p.ldin + col;
      in0[b] = load4(reinterpret_cast<const uint16_t*>(p.in0) + at, left, vec);
      if (MODE == kDh) in1[b] = load4(reinterpret_cast<const uint16_t*>(p.in1) + at, left, vec);
    }
  };
  fetch(t0);
  if (warp >= 2) {
    // the accumulator is complete, so every stage has landed and been read: they become `part`
    mbar_wait(&S.tmem_full, 0, abort_flag, err);
    tc_fence_after();
    const int q = warp & 3;
#pragma unroll 1
    for (int c = 32 * ((warp - 2) >> 2); c < NTOK; c += 64) {
      uint32_t r[32];
      tmem_ld32(tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)c, r);
#pragma unroll
      for (int j = 0; j < 32; ++j) S.part[c + j][q * 32 + lane] = __uint_as_float(r[j]);
    }
    tc_fence_before();
  }
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(NTOK));

  const float* mine = &S.part[0][4 * (threadIdx.x % kQuads)];
  for (; t0 < tokens && left > 0; t0 += step * kBatch) {
    float f[kBatch][4], u[kBatch][4];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[b][j] = b0[j], u[b][j] = b1[j];
      if (MODE == kDown) {
        unpack4<T>(in0[b], u[b]);  // the residual (zeros without one)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[b][j] += u[b][j];
      }
      if (MODE == kDh) {
        float g[4];
        unpack4<T>(in0[b], g);
        unpack4<T>(in1[b], u[b]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const ActParts a = act_parts(g[j], p.act);
          f[b][j] = u[b][j] * a.slope;
          u[b][j] = a.val;
        }
      }
    }
    const int now = t0;
    if (p.in0) fetch(t0 + step * kBatch);
    // every slice's partials, in slice order
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int tok = now + b * step;
      if (tok >= tokens) continue;
      float4 o[kMaxSlices], o2[MODE == kUp ? kMaxSlices : 1];
#pragma unroll
      for (int c = 0; c < kMaxSlices; ++c) {
        o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (MODE == kUp) o2[c] = o[c];
        if (c < slices) {
          const uint32_t at = map_rank(mine + tok * BM, (uint32_t)c);
          o[c] = ld_cluster4(at);
          if (MODE == kUp) o2[c] = ld_cluster4(at + 256u);
        }
      }
      float a[4] = {o[0].x, o[0].y, o[0].z, o[0].w};
#pragma unroll
      for (int c = 1; c < kMaxSlices; ++c) a[0] += o[c].x, a[1] += o[c].y, a[2] += o[c].z, a[3] += o[c].w;
      if (MODE == kUp) {
        float w[4] = {o2[0].x, o2[0].y, o2[0].z, o2[0].w};
#pragma unroll
        for (int c = 1; c < kMaxSlices; ++c) w[0] += o2[c].x, w[1] += o2[c].y, w[2] += o2[c].z, w[3] += o2[c].w;
#pragma unroll
        for (int j = 0; j < 4; ++j) u[b][j] += w[j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (MODE == kDh) {
          f[b][j] *= a[j];
          u[b][j] *= a[j];
        } else {
          f[b][j] += a[j];
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int tok = now + b * step;
      if (tok >= tokens) continue;
      const int64_t row = m0 + tok;
      if (MODE == kUp && p.out1) {
        store4<T>(reinterpret_cast<T*>(p.out1) + row * p.ldaux + col, left, vec, f[b]);
        store4<T>(reinterpret_cast<T*>(p.out2) + row * p.ldaux + col, left, vec, u[b]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (MODE == kUp) f[b][j] = act_parts(f[b][j], p.act).val * u[b][j];
      }
      if (MODE == kDh) store4<T>(reinterpret_cast<T*>(p.out1) + row * p.ldaux + col, left, vec, u[b]);
      store4<T>(reinterpret_cast<T*>(p.out0) + row * p.ldout + col, left, vec, f[b]);
    }
  }
  // the peers have read this CTA's partials (their loads have returned: nothing needs to be released)
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, int MODE, int NTOK, int STAGES>
static cudaError_t launch_split(const GatedArgs& a, int slices, bool dependent, cudaStream_t s) {
  constexpr bool mn = MODE == kDh || MODE == kDx;
  auto k = split_kernel<T, MODE, NTOK, STAGES>;
  const size_t smem = sizeof(SmemS<T, NTOK, STAGES>) + 1024;
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  SplitParams p;
  memset(&p, 0, sizeof(p));
  const int rows = MODE == kUp ? 64 : 128;
  const int64_t w_rows = (a.groups ? a.groups->experts : 1) * a.N;
  bool ok = make_map(&p.x0, a.a0, a.M, a.K, a.lda, NTOK, a.dtype);
  if (MODE == kDx) ok = ok && make_map(&p.x1, a.a1, a.M, a.K, a.lda, NTOK, a.dtype);
  ok = ok && (mn ? make_map_mn(&p.w0, a.b0, a.K, a.N, a.ldb0, a.dtype)
                 : make_map(&p.w0, a.b0, w_rows, a.K, a.ldb0, rows, a.dtype));
  if (MODE == kUp) ok = ok && make_map(&p.w1, a.b1, w_rows, a.K, a.ldb1, rows, a.dtype);
  if (MODE == kDx) ok = ok && make_map_mn(&p.w1, a.b1, a.K, a.N, a.ldb1, a.dtype);
  if (!ok) return cudaErrorInvalidValue;
  p.M = a.M;
  p.N = a.N;
  p.kb0 = (int)((a.K + BK - 1) / BK);
  p.kb = MODE == kDx ? 2 * p.kb0 : p.kb0;
  p.bias0 = a.bias0;
  p.bias1 = a.bias1;
  p.bias_dtype = a.bias_dtype;
  p.in0 = a.in0;
  p.in1 = a.in1;
  p.out0 = a.out0;
  p.out1 = a.out1;
  p.out2 = a.out2;
  p.ldin = a.ldin;
  p.ldout = a.ldout;
  p.ldaux = a.ldaux;
  p.act = a.act;
  p.dependent = dependent;
  if (a.groups) p.tiles = a.groups->tiles;
  const uint32_t fmt = a.dtype == kBF16 ? 1u : 0u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (mn ? 1u << 15 : 0u) |
                         ((uint32_t)(NTOK >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = (unsigned)slices;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((a.N + rows - 1) / rows), (unsigned)slices, (unsigned)((a.M + NTOK - 1) / NTOK));
  cfg.blockDim = dim3(kSplitThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, p, idesc, device_error_flag());
}

// CTAs of clusters of `slices` that the device holds at once, one a SM (clusters do not cross the groups of
// SMs they are placed in, so the larger ones leave some SMs idle)
static int64_t split_room(int slices) {
  static int64_t room[kMaxSlices + 1] = {};
  if (!room[slices]) {
    auto k = split_kernel<__nv_bfloat16, kDown, 256, 4>;
    const size_t smem = sizeof(SmemS<__nv_bfloat16, 256, 4>) + 1024;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)slices;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(1, (unsigned)slices, 64);
    cfg.blockDim = dim3(kSplitThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess || n < 1)
      n = 1;
    room[slices] = (int64_t)n * slices;
  }
  return room[slices];
}

// Tokens a tile and depth slices of the split form, and whether it beats gated_kernel.  Both forms' times are
// modelled in microseconds, launch to launch: waves of CTAs times (k-blocks, final sums, fixed part), and for
// the split form the operands' way from L2.  The constants were fitted to 1500 timings of both forms over the
// four products at 17 to 2048 rows and widths 128 x 344 to 2048 x 5464; the plan's choice is on average 2% (at
// most 25%) above the best of them, the general form alone 66%.  For example, 256 rows of h [.., 2736] times Wd
// [1024, ..]: 18.9 us in gated_kernel (4 tiles), 8.8 us as 64 x 4.
struct SplitPlan {
  int ntok, slices;
  bool use;
};
static SplitPlan plan_split(const GatedArgs& a) {
  const int64_t units = a.mode == kGatedUp ? 64 : 128, cols = a.mode == kGatedUp ? 128 : 256;
  const int64_t kb = (a.K + BK - 1) / BK * (a.mode == kGatedDx ? 2 : 1);
  const double tail = a.mode == kGatedUp || a.mode == kGatedDh ? 0.042 : 0.028;  // final sums of a token
  SplitPlan best = {0, 1, false};
  double best_cost = 1e30;
  for (int ntok = 32; ntok <= 256; ntok *= 2) {
    const double step = ntok == 32 ? 0.22 : ntok == 64 ? 0.25 : ntok == 128 ? 0.28 : 0.40;
    const int64_t tiles = (a.M + ntok - 1) / ntok * ((a.N + units - 1) / units);
    const double l2 = 0.019 * 1e-6 * (double)(tiles * kb * (BM + ntok) * BK * 2);  // 0.019 us a megabyte
    for (int slices = 1, log2 = 0; slices <= kMaxSlices && slices <= kb; slices *= 2, ++log2) {
      const int64_t one = split_room(slices), room = one * (ntok <= 64 ? 2 : 1);  // 64 tokens: two CTAs a SM
      const int64_t ctas = tiles * slices, waves = (ctas + room - 1) / room;
      const double cost = 1.0 + l2 + (room > one && ctas > one ? 1.3 : 0.0) + 0.45 * log2 +
                          waves * ((double)((kb + slices - 1) / slices) * step +
                                   tail * std::min<int64_t>(a.M, ntok) / slices + 2.85);
      if (cost < best_cost) {
        best_cost = cost;
        best.ntok = ntok;
        best.slices = slices;
      }
    }
  }
  const int64_t tiles = ((a.M + BM2 - 1) / BM2) * ((a.N + cols - 1) / cols), pairs = sm_count() / 2;
  const double fixed = a.mode == kGatedUp ? 0.85 : a.mode == kGatedDown ? 1.65 : a.mode == kGatedDh ? 6.0 : 0.0;
  const double general = 4.9 + (double)((tiles + pairs - 1) / pairs) * (0.314 * kb + fixed);
  best.use = best_cost < general && (a.M + best.ntok - 1) / best.ntok <= 65535;
  return best;
}

// Grouped, a few rows an expert: these products are bound by reading every expert's weights once, so the depth is split
// until there are about as many CTAs as the device holds, two an SM (8 experts of 2736 x 1024, 74 rows: the down
// projection's 64 CTAs times four, the call 57 us, with one slice 65; the up projection has 344: with one slice 65 us,
// with two 66, with four 76).
static int few_rows_slices(const GatedArgs& a) {
  const int64_t units = a.mode == kGatedUp ? 64 : 128, kb = (a.K + BK - 1) / BK;
  const int64_t ctas = a.M / a.groups->tile * ((a.N + units - 1) / units);
  int slices = 1;
  while (2 * slices <= std::min<int64_t>(kb, 4) && 2 * slices * ctas <= 2 * sm_count()) slices *= 2;
  return slices;
}

template <typename T, int MODE>
static cudaError_t launch_any(const GatedArgs& a, bool dependent, cudaStream_t s) {
  if constexpr (MODE == kUp || MODE == kDown) {
    if (a.groups && a.groups->tile < kExpertTile) {
      const int slices = few_rows_slices(a);
      if (a.groups->tile == 32) return launch_split<T, MODE, 32, 5>(a, slices, dependent, s);
      if (a.groups->tile == 64) return launch_split<T, MODE, 64, 4>(a, slices, dependent, s);
      return cudaErrorInvalidValue;
    }
  }
  if (a.groups) return launch_gated<T, MODE, true>(a, s);
  const SplitPlan plan = plan_split(a);
  if (!plan.use) return launch_gated<T, MODE>(a, s);
  switch (plan.ntok) {
    case 32: return launch_split<T, MODE, 32, 5>(a, plan.slices, dependent, s);
    case 64: return launch_split<T, MODE, 64, 4>(a, plan.slices, dependent, s);
    case 128: return launch_split<T, MODE, 128, 6>(a, plan.slices, dependent, s);
    default: return launch_split<T, MODE, 256, 4>(a, plan.slices, dependent, s);
  }
}

template <typename T>
static cudaError_t launch_gated_mode(const GatedArgs& a, bool dependent, cudaStream_t s) {
  switch (a.mode) {
    case kGatedUp: return launch_any<T, kUp>(a, dependent, s);
    case kGatedDown: return launch_any<T, kDown>(a, dependent, s);
    case kGatedDh: return launch_any<T, kDh>(a, dependent, s);
    case kGatedDx: return launch_any<T, kDx>(a, dependent, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tc

// ============================================================================ few tokens
// Up to 16 tokens: the products are bound by moving the weights into the SMs once, and the tokens as often
// as there are blocks.  A tile is the 16 rows of one mma.sync m16n8k16: 16 output rows, or, in the DUAL form,
// the rows of Wg and of Wu of 8 hidden units, so that g and u of a unit end in one thread.  A block takes one
// tile of a K slice, its warps split the slice in steps of 32: lane (r, t) reads
// 16 contiguous bytes, k = k0 + 8 t .. 8 t + 7, of weight row r, and of token row r for the other operand.
// Which four of those values meet in which MMA is a permutation of k that both operands share, so the sum is
// unchanged and every load is a full 16-byte vector.  The K slices are the CTAs of a cluster.  Partials are
// added in warp order through shared memory, then in slice order through the cluster's shared memory
// (deterministic).  Larger blocks, whose tiles share the token loads, measured slower at up to 16 tokens: what
// counts is how many loads are in flight (1 token, 1024 x 2736, up: 3.5 us with one tile a block, 5.2 with four;
// 11.2 MB of weights from L2, 3.2 TB/s).
namespace gated {

constexpr int SK_WARPS = 8;

struct SkinnyParams {
  const void* x;
  const void* w0;
  const void* w1;
  const void* bias0;
  const void* bias1;
  const void* res;
  void* out;
  int64_t ldx, ldw0, ldw1, ldres, ldout;
  int M, N, K, k_slice;
  int bias_dtype, act;
  int dependent;  // launched as a programmatic dependent of the kernel that writes x
};

// eight values at p (those below `left` of them, zeros after); NC: through the read-only path
template <bool VEC, bool NC>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int left) {
  if (left <= 0) return make_uint4(0, 0, 0, 0);
  if (VEC && left >= 8) {
    if (NC) return __ldg(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const uint4*>(p);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// (DUAL: two steps' loads in flight and five blocks an SM, so that a projection's many blocks are resident at once;
// 16 tokens, 2048 x 5464: 13.2 us against 15.9 with four steps and four blocks.  The down projection has few
// blocks, which take four steps: 1 token, 1024 x 2736: 3.9 against 4.1 us)
template <typename T, int NT, bool DUAL, bool VEC>
__global__ void __launch_bounds__(32 * SK_WARPS, DUAL ? 5 : 1) skinny_kernel(const SkinnyParams p) {
  constexpr int U = DUAL ? 2 : 4;  // steps whose weight loads are in flight together
  constexpr int R = DUAL ? 8 : 16;  // output rows of a tile
  __shared__ float red[SK_WARPS][NT][32][4];
  __shared__ float part[NT][32][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, slices = gridDim.y;
  const int k_begin = slice * p.k_slice;
  const int k_end = min(p.K, k_begin + p.k_slice);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x);
  const int64_t row = (int64_t)blockIdx.x * R + r, row1 = DUAL ? row : row + 8;
  const bool ok0 = row < p.N, ok1 = row1 < p.N;
  const uint16_t* w0 = reinterpret_cast<const uint16_t*>(p.w0) + row * p.ldw0;
  const uint16_t* w1 = DUAL ? reinterpret_cast<const uint16_t*>(p.w1) + row * p.ldw1
                            : reinterpret_cast<const uint16_t*>(p.w0) + row1 * p.ldw0;
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  bool waited = !p.dependent;
  for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += SK_WARPS * 32 * U) {
    uint4 wa[U], wb[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int kk = k0 + i * SK_WARPS * 32 + 8 * t;
      wa[i] = load8<VEC, true>(w0 + kk, ok0 ? k_end - kk : 0);
      wb[i] = load8<VEC, true>(w1 + kk, ok1 ? k_end - kk : 0);
    }
    if (!waited) {  // the weights do not depend on the kernel before; x does
      asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int kk = k0 + i * SK_WARPS * 32 + 8 * t;
      uint4 xv[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int tok = 8 * n + r;
        xv[n] = load8<VEC, false>(x + tok * p.ldx + kk, tok < p.M ? k_end - kk : 0);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t lo[4] = {wa[i].x, wb[i].x, wa[i].y, wb[i].y}, hi[4] = {wa[i].z, wb[i].z, wa[i].w, wb[i].w};
        attn::mma16816<T>(acc[n], lo, xv[n].x, xv[n].y);
        attn::mma16816<T>(acc[n], hi, xv[n].z, xv[n].w);
      }
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int n = 0; n < NT; ++n)
    *reinterpret_cast<float4*>(red[warp][n][lane]) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 32; i += 32 * SK_WARPS) {
    const int n = i >> 5, l = i & 31;
    float4 v = *reinterpret_cast<const float4*>(red[0][n][l]);
#pragma unroll
    for (int w = 1; w < SK_WARPS; ++w) {
      const float4 o = *reinterpret_cast<const float4*>(red[w][n][l]);
      v.x += o.x;
      v.y += o.y;
      v.z += o.z;
      v.w += o.w;
    }
    *reinterpret_cast<float4*>(part[n][l]) = v;
  }
  if (slices > 1)
    tc::cluster_sync_all();
  else
    __syncthreads();
  // this CTA's share of the (token group, lane) entries: the slices' partials in order, then the epilogue
  constexpr int entries = NT * 32;
  const int share = (entries + slices - 1) / slices;
  for (int i = slice * share + threadIdx.x; i < min(entries, (slice + 1) * share); i += 32 * SK_WARPS) {
    const int n = i >> 5, l = i & 31;
    float4 v;
    if (slices == 1) {
      v = *reinterpret_cast<const float4*>(part[n][l]);
    } else {
      v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < slices; ++c) {
        const float4 o = tc::ld_cluster4(tc::map_rank(part[n][l], (uint32_t)c));
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
    }
    const int64_t col = (int64_t)blockIdx.x * R + (l >> 2);
    const int tok = 8 * n + 2 * (l & 3);
#pragma unroll
    for (int half = 0; half < (DUAL ? 1 : 2); ++half) {
      const int64_t c = col + 8 * half;
      if (c >= p.N) break;
      const float b0 = p.bias0 ? tc::ld_bias(p.bias0, p.bias_dtype, c) : 0.f;
      float f[2] = {(half ? v.z : v.x) + b0, (half ? v.w : v.y) + b0};
      if (DUAL) {
        const float b1 = p.bias1 ? tc::ld_bias(p.bias1, p.bias_dtype, c) : 0.f;
        f[0] = tc::act_parts(f[0], p.act).val * (v.z + b1);
        f[1] = tc::act_parts(f[1], p.act).val * (v.w + b1);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (tok + j >= p.M) break;
        if (!DUAL && p.res) f[j] += to_f(reinterpret_cast<const T*>(p.res)[(tok + j) * p.ldres + c]);
        reinterpret_cast<T*>(p.out)[(tok + j) * p.ldout + c] = from_f<T>(f[j]);
      }
    }
  }
  if (slices > 1) tc::cluster_sync_all();  // the peers have read this CTA's partials
}

template <typename T, int NT, bool DUAL>
static cudaError_t launch_skinny_nt(SkinnyParams p, bool vec, cudaStream_t s) {
  constexpr int rows = DUAL ? 8 : 16;
  // depth slices while there are fewer tiles than two an SM and every warp keeps a step
  // (1 token, h [2736] times Wd [1024, 2736]: 5.4 us in one slice, 3.7 in four)
  const int tiles = (p.N + rows - 1) / rows;
  int slices = 1;
  while (slices < 4 && 2 * slices * tiles <= 2 * tc::sm_count() && p.K / (2 * slices) >= 32 * SK_WARPS) slices *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (slices > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1;
    attr[n].val.clusterDim.y = (unsigned)slices;
    attr[n++].val.clusterDim.z = 1;
  }
  p.k_slice = (p.K + 32 * slices - 1) / (32 * slices) * 32;
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)slices, 1);
  cfg.blockDim = dim3(32 * SK_WARPS, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (vec) return cudaLaunchKernelEx(&cfg, skinny_kernel<T, NT, DUAL, true>, p);
  return cudaLaunchKernelEx(&cfg, skinny_kernel<T, NT, DUAL, false>, p);
}

template <typename T, bool DUAL>
static cudaError_t launch_skinny(const SkinnyParams& p, bool vec, cudaStream_t s) {
  return p.M <= 8 ? launch_skinny_nt<T, 1, DUAL>(p, vec, s) : launch_skinny_nt<T, 2, DUAL>(p, vec, s);
}

// dst[i, j] = src[i s0 + j s1] (16-bit) for several matrices: operands whose rows are not 16-byte aligned, into rows
// that are.  A group is eight elements of a row, one 16-byte store; a thread copies kPadGroups of them, all loads
// before the stores, and a matrix has blocks of its own (20003 x 1001 and three weights: 30 us; 41 with a group a
// thread and as many blocks for each matrix as for the longest).  Where the elements are adjacent, the two aligned
// groups that hold them are read and shifted; at a tensor's ends, past which nothing is read, single elements.
constexpr int kPadGroups = 4;
struct PadCopies {
  PadCopy v[kPadCopies];
  int64_t first[kPadCopies + 1];  // a matrix's first block
};
__device__ __forceinline__ uint4 pad_group(const PadCopy& a, int64_t i, int64_t groups) {
  const int64_t m = i < ((int64_t)1 << 32) ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups;
  const int64_t c = 8 * (i - m * groups), s1 = a.s1;
  const uint16_t* p = reinterpret_cast<const uint16_t*>(a.src) + m * a.s0 + c * s1;
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const uintptr_t at = reinterpret_cast<uintptr_t>(p), lo = at & ~(uintptr_t)15;
  const uintptr_t first = reinterpret_cast<uintptr_t>(a.src), end = first + 2 * ((a.rows - 1) * a.s0 + a.cols);
  if (s1 == 1 && c + 8 <= a.cols && lo >= first && lo + 32 <= end) {
    const uint4 u = *reinterpret_cast<const uint4*>(lo), v = *reinterpret_cast<const uint4*>(lo + 16);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w, w[4] = v.x, w[5] = v.y, w[6] = v.z, w[7] = v.w;
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = at & 8 ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = at & 4 ? w[j + 1] : w[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 8 * (int)(at & 2));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < a.cols) w[j >> 1] |= (uint32_t)p[j * s1] << (16 * (j & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__global__ void __launch_bounds__(256) pad_copy_kernel(const __grid_constant__ PadCopies l) {
  int k = 0;
#pragma unroll
  for (int i = 1; i < kPadCopies; ++i)
    if (blockIdx.x >= l.first[i]) k = i;
  const PadCopy& a = l.v[k];
  const int64_t groups = a.ld / 8, total = a.rows * groups;
  const int64_t i0 = (blockIdx.x - l.first[k]) * (256 * kPadGroups) + threadIdx.x;
  uint4 u[kPadGroups];
#pragma unroll
  for (int g = 0; g < kPadGroups; ++g)
    if (i0 + 256 * g < total) u[g] = pad_group(a, i0 + 256 * g, groups);
#pragma unroll
  for (int g = 0; g < kPadGroups; ++g)
    if (i0 + 256 * g < total) reinterpret_cast<uint4*>(a.dst)[i0 + 256 * g] = u[g];
}

// Column sums of up to two 16-bit [rows, n] matrices (rows 16-byte aligned, ld >= n rounded up to 8; blockIdx.z):
// partial[y][c] over the y-th slice of the rows; a warp takes 256 columns of a row, 16 bytes a lane.
struct ColSources {
  ColSource v[2];
};
template <typename T>
__global__ void __launch_bounds__(256) col_partial_kernel(const __grid_constant__ ColSources p) {
  const ColSource& s = p.v[blockIdx.z];
  const int64_t rows = s.rows, n = s.n, ld = s.ld, step = 8 * s.parts;
  if ((int64_t)blockIdx.x * 256 >= n || (int64_t)blockIdx.y >= s.parts) return;
  __shared__ float red[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8;
  const T* x = reinterpret_cast<const T*>(s.x) + c;
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int64_t r = (int64_t)blockIdx.y * 8 + warp; r < rows; r += step) {
      float f[8];
      unpack8<T>(__ldg(reinterpret_cast<const uint4*>(x + r * ld)), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += f[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) red[warp][lane * 8 + j] = a[j];
  __syncthreads();
  float v = red[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < 8; ++w) v += red[w][threadIdx.x];
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col < n) s.partial[(int64_t)blockIdx.y * n + col] = v;
}

// out[c] (+)= sum over the parts of partial[.][first + c], in a fixed order; blockIdx.y: which sum
struct ColSums {
  ColSum v[kColSums];
};
template <typename T>
__global__ void __launch_bounds__(1024) col_finish_kernel(const __grid_constant__ ColSums p) {
  __shared__ float red[32][33];
  const ColSum& s = p.v[blockIdx.y];
  if (!s.out || (int64_t)blockIdx.x * 32 >= s.n) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < s.n)
    for (int64_t r = w; r < s.parts; r += 32) a += s.partial[r * s.stride + s.first + c];
  red[w][lane] = a;
  __syncthreads();
  if (w || c >= s.n) return;
  for (int i = 1; i < 32; ++i) a += red[i][lane];
  if (s.f32) {
    float* o = reinterpret_cast<float*>(s.out) + c;
    *o = s.accumulate ? *o + a : a;
  } else {
    reinterpret_cast<T*>(s.out)[c] = from_f<T>(a);
  }
}

}  // namespace gated

int col_sum_parts(int64_t rows, int64_t n) {
  const int64_t cols = (n + 255) / 256;
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + 31) / 32, 4 * (int64_t)tc::sm_count() / cols));
}
cudaError_t col_partial(const ColSource* src, int count, int dtype, cudaStream_t s) {
  if (count < 1 || count > 2) return cudaErrorInvalidValue;
  const ColSource &a = src[0], &b = src[count - 1];
  const gated::ColSources p = {{a, b}};
  const dim3 grid((unsigned)((std::max(a.n, b.n) + 255) / 256), (unsigned)std::max(a.parts, b.parts), (unsigned)count);
  if (dtype == kBF16)
    gated::col_partial_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  else
    gated::col_partial_kernel<__half><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}
cudaError_t col_finish(const ColSum* v, int dtype, cudaStream_t s) {
  gated::ColSums p;
  int64_t n = 1;
  for (int i = 0; i < kColSums; ++i) {
    p.v[i] = v[i];
    if (v[i].out) n = std::max(n, v[i].n);
  }
  const dim3 grid((unsigned)((n + 31) / 32), kColSums, 1);
  if (dtype == kBF16)
    gated::col_finish_kernel<__nv_bfloat16><<<grid, 1024, 0, s>>>(p);
  else
    gated::col_finish_kernel<__half><<<grid, 1024, 0, s>>>(p);
  return cudaGetLastError();
}

int64_t gated_dw_workspace(const GatedDwArgs& a) {
  int64_t tiles = 0;
  for (const auto& w : a.w) tiles += tc::dw_tiles(w);
  const tc::DwPlan p = tc::dw_plan(tiles, a.T);
  return (int64_t)p.rem * p.splits * tc::BM2 * tc::BN2;
}

cudaError_t gated_dw(const GatedDwArgs& a, cudaStream_t s) {
  if ((a.dtype != kBF16 && a.dtype != kF16) || a.T <= 0) return cudaErrorInvalidValue;
  if (!a.w[0].D && !a.w[1].D && !a.w[2].D) return cudaErrorInvalidValue;
  for (const auto& w : a.w)
    if (w.D && (!w.a || !w.b || w.M <= 0 || w.N <= 0 || (w.accumulate && !w.out_f32))) return cudaErrorInvalidValue;
  if (a.groups) return a.dtype == kBF16 ? tc::launch_dw_grouped<__nv_bfloat16>(a, s) : tc::launch_dw_grouped<__half>(a, s);
  return a.dtype == kBF16 ? tc::launch_dw<__nv_bfloat16>(a, s) : tc::launch_dw<__half>(a, s);
}

int64_t gated_sum_rows(const GatedArgs& a) {
  return a.mode == kGatedDh && !tc::plan_split(a).use ? 2 * ((a.M + tc::BM2 - 1) / tc::BM2) : 0;
}

cudaError_t gated_product(const GatedArgs& a, bool dependent, cudaStream_t s) {
  if ((a.dtype != kBF16 && a.dtype != kF16) || a.M <= 0 || a.N <= 0 || a.K <= 0) return cudaErrorInvalidValue;
  if (a.dtype == kBF16) return tc::launch_gated_mode<__nv_bfloat16>(a, dependent, s);
  return tc::launch_gated_mode<__half>(a, dependent, s);
}

cudaError_t gated_skinny(const GatedArgs& a, bool dependent, cudaStream_t s) {
  if ((a.dtype != kBF16 && a.dtype != kF16) || a.M <= 0 || a.M > kGatedSkinnyTokens || a.N <= 0 || a.K <= 0 ||
      a.N > (int64_t)1 << 30 || a.K > (int64_t)1 << 30)
    return cudaErrorInvalidValue;
  gated::SkinnyParams p;
  p.x = a.a0;
  p.w0 = a.b0;
  p.w1 = a.b1;
  p.bias0 = a.bias0;
  p.bias1 = a.bias1;
  p.res = a.in0;
  p.out = a.out0;
  p.ldx = a.lda;
  p.ldw0 = a.ldb0;
  p.ldw1 = a.ldb1;
  p.ldres = a.ldin;
  p.ldout = a.ldout;
  p.M = (int)a.M;
  p.N = (int)a.N;
  p.K = (int)a.K;
  p.bias_dtype = a.bias_dtype;
  p.act = a.act;
  p.dependent = dependent ? 1 : 0;
  const bool dual = a.mode == kGatedUp;
  const bool vec = (a.lda | a.ldb0 | (dual ? a.ldb1 : 0)) % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.a0) | reinterpret_cast<uintptr_t>(a.b0) |
                     (dual ? reinterpret_cast<uintptr_t>(a.b1) : 0)) & 15) == 0;
  if (a.dtype == kBF16)
    return dual ? gated::launch_skinny<__nv_bfloat16, true>(p, vec, s)
                : gated::launch_skinny<__nv_bfloat16, false>(p, vec, s);
  return dual ? gated::launch_skinny<__half, true>(p, vec, s) : gated::launch_skinny<__half, false>(p, vec, s);
}

cudaError_t pad_copy(const PadCopy* v, int count, cudaStream_t s) {
  gated::PadCopies l;
  int64_t blocks = 0;
  if (count > kPadCopies) return cudaErrorInvalidValue;
  for (int i = 0; i <= kPadCopies; ++i) {
    l.first[i] = i <= count ? blocks : INT64_MAX;
    if (i >= count) continue;
    if (v[i].ld % 8 || (reinterpret_cast<uintptr_t>(v[i].dst) & 15)) return cudaErrorInvalidValue;
    l.v[i] = v[i];
    blocks += (v[i].rows * (v[i].ld / 8) + 256 * gated::kPadGroups - 1) / (256 * gated::kPadGroups);
  }
  if (blocks == 0) return cudaSuccess;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  gated::pad_copy_kernel<<<(unsigned)blocks, 256, 0, s>>>(l);
  return cudaGetLastError();
}

}  // namespace nsw
