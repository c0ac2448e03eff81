// Gated feed-forward network on the tensor cores.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) * u,  y = h Wd^T + bd + residual
//   dh = dy Wd,  dg = dh * u * act'(g),  du = dh * act(g),  dx = dg Wg + du Wu
//
// act is SiLU, g / (1 + exp(-g)), or the exact GELU, g Phi(g).  Two kernel families:
//
// * gated_kernel: one persistent CTA-pair kernel (tcgen05.mma.cta_group::2, 256-row pair tiles) in four
//   forms that differ in where their operands come from and in the epilogue:
//     kUp    both projections at once: the pair's B tile is 128 rows of Wg (CTA 0) and the same 128
//            rows of Wu (CTA 1), so g and u of one hidden unit land in the same TMEM lane 128 columns
//            apart and the activation and the product happen in registers; h (and, for training, g and
//            u) leave by TMA store.
//     kDown  h Wd^T + bd + residual; residual tiles arrive by TMA before the accumulator is ready.
//     kDh    dy Wd with Wd read as it is stored ([D, H], MN-major for this product, so no transposed
//            copy exists); the epilogue loads g and u tiles by TMA and writes dg and du.
//     kDx    dg Wg + du Wu as ONE product of depth 2 H: the k-loop runs through (dg, Wg), then
//            (du, Wu), into the same accumulator; the weights are again read MN-major as stored.
// * skinny_kernel: up to 64 tokens, where the time is that of streaming the weights once.  See there.
//
// Sums are fp32 in TMEM / registers.  Rounded to 16 bits: g, u (kept for the backward), h, dg, du,
// because the following products take 16-bit operands; the forward's h is computed from the unrounded
// g and u.
#include <cuda.h>

#include <algorithm>
#include <cstring>

#include "tcgen05.cuh"

namespace nsw {
namespace tc {

constexpr int GS = 5;        // pipeline stages (32 KB a CTA)
constexpr int GBUFS = 4;     // 2 KB tile buffers per epilogue warp
enum : int { kUp = 0, kDown = 1, kDh = 2, kDx = 3 };

struct GatedParams {
  CUtensorMap a0, a1, b0, b1;    // operands (a1 / b1: Wu in kUp, the second half of the depth in kDx)
  CUtensorMap in0, in1;          // kDh: g, u; kDown: residual
  CUtensorMap out0, out1, out2;  // kUp: h, g, u; kDh: dg, du; kDown / kDx: the result
  int64_t M, N;                  // rows; columns of the result (hidden units in kUp / kDh)
  int kb0, kb;                   // k-blocks of the first operand pair, and in all
  const void* bias0;
  const void* bias1;
  int bias_dtype;
  int act;      // 0 SiLU, 1 GELU
  int save;     // kUp: store g and u
  int has_res;  // kDown
};

template <typename T>
struct SmemG {
  alignas(1024) T a[GS][BM * BK];
  alignas(1024) T b[GS][128 * BK];
  alignas(1024) T buf[kEpiWarps][GBUFS][32 * kStageRow];
  uint64_t full[GS], empty[GS];
  uint64_t tmem_full[2], tmem_empty[2];
  uint64_t in_full[kEpiWarps][2];
  uint64_t done;
  uint32_t tmem_base;
  int abort_flag;
};

// act(g) and act'(g).  The exponential and the reciprocal are the hardware approximations (2 ulp):
// their error is far below the 16-bit rounding of every result.  exp(-g) = inf gives sig = 0.
struct ActParts {
  float val, slope;
};
__device__ __forceinline__ ActParts act_parts(float g, int act) {
  ActParts r;
  if (act == 0) {
    float e, sig;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.44269504088896340736f * g));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(sig) : "f"(1.0f + e));
    r.val = g * sig;
    r.slope = fmaf(r.val, 1.0f - sig, sig);
  } else {
    const GeluParts p = gelu_parts_fast(g);
    r.val = g * p.cdf;
    r.slope = fmaf(g, p.pdf, p.cdf);
  }
  return r;
}

__device__ __forceinline__ float ld_bias(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dtype == kBF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(reinterpret_cast<const __half*>(p)[i]);
}
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

__device__ __forceinline__ void bulk_wait_read_3() { asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory"); }

// this lane's row of a 32 x 32 tile into the warp's next buffer (ring of GBUFS), then one TMA store
template <typename T>
__device__ __forceinline__ void ring_store(const CUtensorMap* map, const float* f, T (*buf)[32 * kStageRow], int lane,
                                           int64_t nb, int64_t row_base, uint32_t& ring) {
  T* b = buf[ring & (GBUFS - 1)];
  if (lane == 0) bulk_wait_read_3();  // at most three later stores pending: this buffer's has been read
  __syncwarp();
#pragma unroll
  for (int v = 0; v < 4; ++v) *reinterpret_cast<uint4*>(b + stg_off(lane, v)) = pack8<T>(&f[8 * v]);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) tma_store_2d(map, b, (int)nb, (int)row_base);
  ++ring;
}

template <typename T, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gated_kernel(const __grid_constant__ GatedParams p, uint32_t idesc, int* err) {
  constexpr bool kMnB = MODE == kDh || MODE == kDx;  // B read as stored, N contiguous
  constexpr int kCols = MODE == kUp ? 128 : 256;     // result columns of a pair tile
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto& S = *reinterpret_cast<SmemG<T>*>(base);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int64_t m_tiles = (p.M + BM2 - 1) / BM2;
  const int64_t n_tiles = (p.N + kCols - 1) / kCols;
  const int64_t num_tiles = m_tiles * n_tiles;
  volatile int* abort_flag = &S.abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < GS; ++s) {
      mbar_init(&S.full[s], 1);
      mbar_init(&S.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&S.tmem_full[a], 1);
      mbar_init(&S.tmem_empty[a], 2 * kEpiWarps);
      for (int w = 0; w < kEpiWarps; ++w) mbar_init(&S.in_full[w][a], 1);
    }
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
      for (int64_t tile = pair; tile < num_tiles && !*abort_flag; tile += npairs) {
        const int m0 = (int)((tile / n_tiles) * BM2) + (int)rank * BM;
        const int nb0 = (int)((tile % n_tiles) * kCols) + (MODE == kUp ? 0 : (int)rank * 128);
        for (int kb = 0; kb < p.kb; ++kb) {
          if (!mbar_wait(&S.empty[stage], phase ^ 1, abort_flag, err)) break;
          if (rank == 0) mbar_expect_tx(&S.full[stage], (uint32_t)(2 * (BM + 128) * BK * sizeof(T)));
          const uint32_t fb = full_leader + 8u * stage;
          const bool second = MODE == kDx && kb >= p.kb0;
          const int k0 = (second ? kb - p.kb0 : kb) * BK;
          tma_load_2d_pair(S.a[stage], second ? &p.a1 : &p.a0, fb, k0, m0);
          if (kMnB) {
            const CUtensorMap* mb = second ? &p.b1 : &p.b0;
            tma_load_2d_pair(&S.b[stage][0], mb, fb, nb0, k0);
            tma_load_2d_pair(&S.b[stage][64 * BK], mb, fb, nb0 + 64, k0);
          } else {
            tma_load_2d_pair(S.b[stage], MODE == kUp && rank ? &p.b1 : &p.b0, fb, k0, nb0);
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
      for (int64_t tile = pair; tile < num_tiles && !*abort_flag; tile += npairs) {
        if (!mbar_wait(&S.tmem_empty[acc], acc_phase ^ 1, abort_flag, err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN2);
        bool ok = true;
        for (int kb = 0; kb < p.kb; ++kb) {
          if (!mbar_wait(&S.full[stage], phase, abort_flag, err)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t db = kMnB ? smem_desc_mn(&S.b[stage][k * 16 * 64], 64 * BK * (uint32_t)sizeof(T))
                                     : smem_desc_sw128(&S.b[stage][k * 16]);
            umma2_f16(d_tmem, smem_desc_sw128(&S.a[stage][k * 16]), db, idesc, (kb > 0 || k > 0) ? 1u : 0u);
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
    const int half = ew >> 2;
    T(*buf)[32 * kStageRow] = S.buf[ew];
    uint64_t* in_full = S.in_full[ew];
    const uint32_t empty_leader = map_rank(&S.tmem_empty[0], 0);
    uint32_t ring = 0;
    uint32_t in_phase = 0;  // parity of each in_full barrier, one bit each
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t pending = 0;  // input loads issued and not waited for, one bit per in_full barrier
    bool ok = true;
    for (int64_t tile = pair; tile < num_tiles && ok; tile += npairs) {
      const int64_t row_base = (tile / n_tiles) * BM2 + (int64_t)rank * BM + q * 32;
      const int64_t n0 = (tile % n_tiles) * kCols + half * (kCols / 2);
      const bool rows = row_base < p.M;  // warp-uniform; a tile's lower rows may be past the end
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN2);
      // kDh: g and u of chunk c into buffers 2 (c & 1), 2 (c & 1) + 1
      auto issue_gu = [&](int c) {
        const int64_t nb = n0 + 32 * c;
        if (!rows || nb >= p.N) return;
        if (lane == 0) {
          bulk_wait_read_0();  // the stores that last used these buffers have read them
          uint64_t* bar = &in_full[c & 1];
          mbar_expect_tx(bar, 2 * 32 * kStageRow * sizeof(T));
          tma_load_2d(buf[2 * (c & 1)], &p.in0, bar, (int)nb, (int)row_base);
          tma_load_2d(buf[2 * (c & 1) + 1], &p.in1, bar, (int)nb, (int)row_base);
        }
        pending |= 1u << (c & 1);
      };
      if (MODE == kDh) issue_gu(0);
      if (MODE == kDown && p.has_res && rows && n0 < p.N) {
        if (lane == 0) {
          bulk_wait_read_0();
          uint32_t chunks = 0;
          for (int c = 0; c < 4; ++c) chunks += n0 + 32 * c < p.N;
          mbar_expect_tx(&in_full[0], chunks * 32 * kStageRow * (uint32_t)sizeof(T));
          for (int c = 0; c < 4; ++c)
            if (n0 + 32 * c < p.N) tma_load_2d(buf[c], &p.in0, &in_full[0], (int)(n0 + 32 * c), (int)row_base);
        }
        pending |= 1u;
      }
      if (!mbar_wait(&S.tmem_full[acc], acc_phase, abort_flag, err)) break;
      tc_fence_after();
      if (MODE == kUp) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int64_t nb = n0 + 32 * c;
          if (!rows || nb >= p.N) break;
          uint32_t rg[32], ru[32];
          tmem_ld32_async(t_row + (uint32_t)(64 * half + 32 * c), rg);
          tmem_ld32_async(t_row + (uint32_t)(128 + 64 * half + 32 * c), ru);
          tmem_wait_ld(rg);
          tmem_wait_ld(ru);
          float* g = reinterpret_cast<float*>(rg);
          float* u = reinterpret_cast<float*>(ru);
          if (p.bias0) add_bias32(p.bias0, p.bias_dtype, nb, p.N, g);
          if (p.bias1) add_bias32(p.bias1, p.bias_dtype, nb, p.N, u);
          if (p.save) {
            ring_store<T>(&p.out1, g, buf, lane, nb, row_base, ring);
            ring_store<T>(&p.out2, u, buf, lane, nb, row_base, ring);
          }
          if (p.act == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_parts(g[j], 0).val;
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_parts(g[j], 1).val;
          }
          ring_store<T>(&p.out0, u, buf, lane, nb, row_base, ring);
        }
      } else if (MODE == kDh) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int64_t nb = n0 + 32 * c;
          if (!rows || nb >= p.N) break;
          uint32_t r[32];
          tmem_ld32_async(t_row + (uint32_t)(128 * half + 32 * c), r);
          if (c + 1 < 4) issue_gu(c + 1);
          if (!mbar_wait(&in_full[c & 1], (in_phase >> (c & 1)) & 1u, abort_flag, err)) {
            ok = false;
            tmem_wait_ld(r);
            break;
          }
          in_phase ^= 1u << (c & 1);
          pending &= ~(1u << (c & 1));
          tmem_wait_ld(r);
          T* bg = buf[2 * (c & 1)];
          T* bu = buf[2 * (c & 1) + 1];
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
        }
      } else {
        if (MODE == kDown && (pending & 1u)) {
          if (!mbar_wait(&in_full[0], in_phase & 1u, abort_flag, err)) break;
          in_phase ^= 1u;
          pending = 0;
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          const int64_t nb = n0 + 32 * c;
          if (!rows || nb >= p.N) break;
          uint32_t r[32];
          tmem_ld32(t_row + (uint32_t)(128 * half + 32 * c), r);
          float* f = reinterpret_cast<float*>(r);
          if (MODE == kDown && p.bias0) add_bias32(p.bias0, p.bias_dtype, nb, p.N, f);
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
            ring_store<T>(&p.out0, f, buf, lane, nb, row_base, ring);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(empty_leader + 8u * acc);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) {
      bulk_wait_all();
      // after an abort, input loads still in flight land before the shared memory is released
      for (int b = 0; b < 2; ++b) {
        if (!(pending & (1u << b))) continue;
        const unsigned long long t0 = globaltimer();
        while (!mbar_try_wait(&in_full[b], (in_phase >> b) & 1u) && globaltimer() - t0 < kWaitBudgetNs) {
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

template <typename T, int MODE>
static cudaError_t launch_gated(const GatedArgs& a, cudaStream_t s) {
  const size_t smem = sizeof(SmemG<T>) + 1024;
  auto k = gated_kernel<T, MODE>;
  // on each call: the attribute belongs to the current device, and a runtime call has to make that device's
  // context current on this thread (an autograd thread may not have one yet) before the maps are encoded
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  GatedParams p;
  memset(&p, 0, sizeof(p));
  const bool mn = MODE == kDh || MODE == kDx;
  bool ok = make_map(&p.a0, a.a0, a.M, a.K, a.lda, BM, a.dtype);
  if (MODE == kDx) ok = ok && make_map(&p.a1, a.a1, a.M, a.K, a.lda, BM, a.dtype);
  if (mn) {
    ok = ok && make_map_mn(&p.b0, a.b0, a.K, a.N, a.ldb0, a.dtype);
    if (MODE == kDx) ok = ok && make_map_mn(&p.b1, a.b1, a.K, a.N, a.ldb1, a.dtype);
  } else {
    ok = ok && make_map(&p.b0, a.b0, a.N, a.K, a.ldb0, 128, a.dtype);
    if (MODE == kUp) ok = ok && make_map(&p.b1, a.b1, a.N, a.K, a.ldb1, 128, a.dtype);
  }
  if (a.in0) ok = ok && make_store_map(&p.in0, const_cast<void*>(a.in0), a.M, a.N, a.ldin, a.dtype);
  if (a.in1) ok = ok && make_store_map(&p.in1, const_cast<void*>(a.in1), a.M, a.N, a.ldin, a.dtype);
  ok = ok && make_store_map(&p.out0, a.out0, a.M, a.N, a.ldout, a.dtype);
  if (a.out1) ok = ok && make_store_map(&p.out1, a.out1, a.M, a.N, a.ldaux, a.dtype);
  if (a.out2) ok = ok && make_store_map(&p.out2, a.out2, a.M, a.N, a.ldaux, a.dtype);
  if (!ok) return cudaErrorInvalidValue;
  p.M = a.M;
  p.N = a.N;
  p.kb0 = (int)((a.K + BK - 1) / BK);
  p.kb = MODE == kDx ? 2 * p.kb0 : p.kb0;
  p.bias0 = a.bias0;
  p.bias1 = a.bias1;
  p.bias_dtype = a.bias_dtype;
  p.act = a.act;
  p.save = MODE == kUp && a.out1 != nullptr;
  p.has_res = MODE == kDown && a.in0 != nullptr;
  const uint32_t fmt = a.dtype == kBF16 ? 1u : 0u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (mn ? 1u << 16 : 0u) | ((uint32_t)(BN2 >> 3) << 17) |
                         ((uint32_t)(BM2 >> 4) << 24);
  const int cols = MODE == kUp ? 128 : 256;
  const int64_t tiles = ((a.M + BM2 - 1) / BM2) * ((a.N + cols - 1) / cols);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kThreads, 1, 1);
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
  const int pairs = tiles < max_pairs ? (int)tiles : max_pairs;
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  NSW_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, p, idesc, device_error_flag()));
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_gated_mode(const GatedArgs& a, cudaStream_t s) {
  switch (a.mode) {
    case kGatedUp: return launch_gated<T, kUp>(a, s);
    case kGatedDown: return launch_gated<T, kDown>(a, s);
    case kGatedDh: return launch_gated<T, kDh>(a, s);
    case kGatedDx: return launch_gated<T, kDx>(a, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tc

// ============================================================================ few tokens
// Up to 64 tokens: the products are bound by moving the weights into the SMs once, and the tokens as often
// as there are blocks.  A tile is the 16 rows of one mma.sync m16n8k16: 16 output rows, or, in the DUAL form,
// the rows of Wg and of Wu of 8 hidden units, so that g and u of a unit end in one thread.  A block takes G
// tiles (they share each token load) of a K slice, its warps split the slice in steps of 32: lane (r, t) reads
// 16 contiguous bytes, k = k0 + 8 t .. 8 t + 7, of weight row r, and of token row r for the other operand.
// Which four of those values meet in which MMA is a permutation of k that both operands share, so the sum is
// unchanged and every load is a full 16-byte vector.  The K slices are the CTAs of a cluster.  Partials are
// added in warp order through shared memory, then in slice order through the cluster's shared memory
// (deterministic).  plan_skinny picks G and the number of slices.
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

template <typename T>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

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

template <typename T, int NT, int G, bool DUAL, bool VEC>
__global__ void __launch_bounds__(32 * SK_WARPS) skinny_kernel(const SkinnyParams p) {
  constexpr int U = 4 / G;  // steps whose weight loads are in flight together
  constexpr int R = DUAL ? 8 : 16;  // output rows of a tile
  __shared__ float red[SK_WARPS][NT][32][4];
  __shared__ float part[G][NT][32][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int slice = blockIdx.y, slices = gridDim.y;
  const int k_begin = slice * p.k_slice;
  const int k_end = min(p.K, k_begin + p.k_slice);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x);
  const uint16_t *w0[G], *w1[G];
  bool ok0[G], ok1[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int64_t row = ((int64_t)blockIdx.x * G + g) * R + r;
    const int64_t row1 = DUAL ? row : row + 8;
    ok0[g] = row < p.N;
    ok1[g] = row1 < p.N;
    w0[g] = reinterpret_cast<const uint16_t*>(p.w0) + row * p.ldw0;
    w1[g] = DUAL ? reinterpret_cast<const uint16_t*>(p.w1) + row * p.ldw1
                 : reinterpret_cast<const uint16_t*>(p.w0) + row1 * p.ldw0;
  }
  float acc[G][NT][4];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[g][i][j] = 0.f;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  bool waited = !p.dependent;
  for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += SK_WARPS * 32 * U) {
    uint4 wa[U][G], wb[U][G];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int kk = k0 + i * SK_WARPS * 32 + 8 * t;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        wa[i][g] = load8<VEC, true>(w0[g] + kk, ok0[g] ? k_end - kk : 0);
        wb[i][g] = load8<VEC, true>(w1[g] + kk, ok1[g] ? k_end - kk : 0);
      }
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
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          mma16816<T>(acc[g][n], wa[i][g].x, wb[i][g].x, wa[i][g].y, wb[i][g].y, xv[n].x, xv[n].y);
          mma16816<T>(acc[g][n], wa[i][g].z, wb[i][g].z, wa[i][g].w, wb[i][g].w, xv[n].z, xv[n].w);
        }
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (g) __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
      *reinterpret_cast<float4*>(red[warp][n][lane]) =
          make_float4(acc[g][n][0], acc[g][n][1], acc[g][n][2], acc[g][n][3]);
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
      *reinterpret_cast<float4*>(part[g][n][l]) = v;
    }
  }
  if (slices > 1)
    tc::cluster_sync_all();
  else
    __syncthreads();
  // this CTA's share of the (tile, token group, lane) entries: the slices' partials in order, then the epilogue
  const int entries = G * NT * 32;
  for (int i = slice * (32 * SK_WARPS) + threadIdx.x; i < entries; i += slices * (32 * SK_WARPS)) {
    const int g = i / (NT * 32), n = (i >> 5) % NT, l = i & 31;
    float4 v;
    if (slices == 1) {
      v = *reinterpret_cast<const float4*>(part[g][n][l]);
    } else {
      v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = 0; c < slices; ++c) {
        float4 o;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w)
                     : "r"(tc::map_rank(part[g][n][l], (uint32_t)c))
                     : "memory");
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
    }
    const int64_t col = ((int64_t)blockIdx.x * G + g) * R + (l >> 2);
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

// G tiles a block and `slices` K slices that move the fewest bytes through the busiest SM: blocks per SM times
// (tokens' slice + weights' slice).  A slice's exchange through the cluster's shared memory costs about as
// much as 16 KB more (a cluster launch and two barriers; fitted at 1 and 37 tokens).
struct SkinnyPlan {
  int g, slices;
};
static SkinnyPlan plan_skinny(int64_t M, int64_t N, int64_t K, bool dual) {
  const int64_t sms = tc::sm_count(), tiles = (N + (dual ? 7 : 15)) / (dual ? 8 : 16);
  SkinnyPlan best = {1, 1};
  int64_t best_cost = INT64_MAX;
  for (int slices = 1; slices <= 8; slices *= 2) {
    if (slices > 1 && K / slices < 32 * SK_WARPS) break;  // a step for every warp
    for (int g = 1; g <= 4; g *= 2) {
      if (g > 1 && (tiles + g - 1) / g * slices < sms / 2) break;
      const int64_t blocks = (tiles + g - 1) / g * slices;
      const int64_t bytes = 2 * (K / slices) * (M + 16 * g) + (slices > 1 ? 16384 : 0);
      const int64_t cost = (blocks + sms - 1) / sms * bytes;
      if (cost < best_cost) {
        best_cost = cost;
        best = {g, slices};
      }
    }
  }
  return best;
}

template <typename T, int NT, int G, bool DUAL>
static cudaError_t launch_skinny_g(SkinnyParams p, int slices, bool vec, cudaStream_t s) {
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
  constexpr int rows = (DUAL ? 8 : 16) * G;
  p.k_slice = (p.K + 32 * slices - 1) / (32 * slices) * 32;
  cfg.gridDim = dim3((unsigned)((p.N + rows - 1) / rows), (unsigned)slices, 1);
  cfg.blockDim = dim3(32 * SK_WARPS, 1, 1);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (vec) return cudaLaunchKernelEx(&cfg, skinny_kernel<T, NT, G, DUAL, true>, p);
  return cudaLaunchKernelEx(&cfg, skinny_kernel<T, NT, G, DUAL, false>, p);
}

template <typename T, int NT, bool DUAL>
static cudaError_t launch_skinny_nt(const SkinnyParams& p, bool vec, cudaStream_t s) {
  const SkinnyPlan plan = plan_skinny(p.M, p.N, p.K, DUAL);
  if (plan.g == 1) return launch_skinny_g<T, NT, 1, DUAL>(p, plan.slices, vec, s);
  if (plan.g == 2) return launch_skinny_g<T, NT, 2, DUAL>(p, plan.slices, vec, s);
  return launch_skinny_g<T, NT, 4, DUAL>(p, plan.slices, vec, s);
}

template <typename T, bool DUAL>
static cudaError_t launch_skinny(const SkinnyParams& p, bool vec, cudaStream_t s) {
  if (p.M <= 8) return launch_skinny_nt<T, 1, DUAL>(p, vec, s);
  if (p.M <= 16) return launch_skinny_nt<T, 2, DUAL>(p, vec, s);
  if (p.M <= 32) return launch_skinny_nt<T, 4, DUAL>(p, vec, s);
  return launch_skinny_nt<T, 8, DUAL>(p, vec, s);
}

// dst[i, j] = src[i s0 + j s1] (16-bit), rows of ld elements: operands whose rows are not 16-byte aligned
__global__ void pad_copy_kernel(const uint16_t* __restrict__ src, int64_t s0, int64_t s1, uint16_t* __restrict__ dst,
                                int64_t ld, int64_t rows, int64_t cols) {
  const int64_t total = rows * ld;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / ld, c = i - m * ld;
    if (c < cols) dst[i] = src[m * s0 + c * s1];
  }
}

}  // namespace gated

cudaError_t gated_product(const GatedArgs& a, cudaStream_t s) {
  if ((a.dtype != kBF16 && a.dtype != kF16) || a.M <= 0 || a.N <= 0 || a.K <= 0) return cudaErrorInvalidValue;
  if (a.dtype == kBF16) return tc::launch_gated_mode<__nv_bfloat16>(a, s);
  return tc::launch_gated_mode<__half>(a, s);
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

cudaError_t pad_copy(const void* src, int64_t s0, int64_t s1, void* dst, int64_t ld, int64_t rows, int64_t cols,
                     cudaStream_t s) {
  const int64_t total = rows * ld;
  if (total <= 0) return cudaSuccess;
  const int blocks = (int)std::min<int64_t>((total + 255) / 256, 16 * tc::sm_count());
  gated::pad_copy_kernel<<<blocks, 256, 0, s>>>(reinterpret_cast<const uint16_t*>(src), s0, s1,
                                                reinterpret_cast<uint16_t*>(dst), ld, rows, cols);
  return cudaGetLastError();
}

}  // namespace nsw
