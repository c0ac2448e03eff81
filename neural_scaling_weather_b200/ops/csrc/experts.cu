// Routed experts: y_t = sum_j w_tj MLP_e(t,j)(x_t) + residual_t over the experts that a router chose for each token.
//
// The products run grouped by expert (gated_mlp.cu, the GROUPED forms of its pair kernel, and its split kernel for few
// rows an expert) on rows sorted by expert.
// Here is what stands around them:
//   plan     a stable counting sort of the assignments (token t's j-th expert) by expert, each expert's rows padded to
//            whole tiles (256 rows, or fewer: expert_tile), so that a tile belongs to one expert and needs no bounds;
//   gather   the sorted rows of x; in the backward those of dy times their weights, and with the same read of dy the
//            weights' gradients, the dot products with the experts' outputs;
//   combine  a token's rows of the experts' outputs, weighted, plus the residual; in the backward those of dx;
//   few      the whole network for a few assignments, which reads the chosen experts' weights and nothing else.
// Padding rows are zeros: the products make zeros of them, and the weights' gradients add zeros.
// Rounded to 16 bits: the experts' outputs (before their weighted sum in fp32) and, in the backward, the weighted dy,
// as operands of the next product and because wider ones would double the traffic here; each adds half a step beside
// the products' own roundings (gated_mlp.cu).  In fp16 that holds from 6e-5 to 65504: a weight of 1e-3 times a dy of 1e-3
// keeps four bits, less than 3e-8 is zero, as it is for dg and du, in the dense network too.  A loss scale moves all
// of them together; bf16 has fp32's range.
#include <algorithm>

#include "gated.cuh"

namespace nsw {
namespace experts {

// ------------------------------------------------------------------------------------------------------- plan
// A block sorts a chunk of assignments, each of its warps `share` of them in order, 32 at once; equal experts among the 32
// find one another by match_any.  One block does it all in one launch up to kOneChunk, where that takes as long as the three
// launches for chunks of kChunk (8 experts: 4000 assignments 7.5 us; 8100 in one block 14.1, in chunks 9.8 and two gaps).
constexpr int kWarps = 16, kThreads = 32 * kWarps, kChunk = 2048, kOneChunk = 4096;

__device__ __forceinline__ int expert_at(const ExpertPlan& p, int64_t i) {
  if (i >= p.count) return -1;
  const int64_t e = p.experts[i];
  return e >= 0 && e < p.num_experts ? (int)e : -1;
}

// f(assignment, expert) of a warp's share from `first`, eight steps' loads together; `share` is a multiple of 32
template <typename F>
__device__ __forceinline__ void each_assignment(const ExpertPlan& p, int64_t first, int share, F f) {
  const int64_t end = min(first + share, p.count);
  for (int64_t i0 = first; i0 < end; i0 += 256) {
    int e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t i = i0 + 32 * u + (threadIdx.x & 31);
      e[u] = i < end ? expert_at(p, i) : -1;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + 32 * u < end) f(i0 + 32 * u + (threadIdx.x & 31), e[u]);
  }
}

// count[warp][e] of this block's chunk
__device__ __forceinline__ void count_chunk(const ExpertPlan& p, int64_t first, int share, int (*count)[kMaxExperts]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = lane; e < p.num_experts; e += 32) count[warp][e] = 0;
  __syncwarp();
  each_assignment(p, first + warp * share, share, [&](int64_t, int e) {
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && (same & ((1u << lane) - 1)) == 0) count[warp][e] += __popc(same);
    __syncwarp();
  });
}

// rows, tiles and the padding's sources from every expert's number of assignments; one block, thread e has expert e's
__device__ __forceinline__ void place_experts(const ExpertPlan& p, int count, int* start) {
  __shared__ int warp_sum[kWarps];
  __shared__ int2 pad[kMaxExperts];
  const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
  const int padded = (count + p.tile - 1) / p.tile * p.tile;
  int upto = padded;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += warp_sum[w];
  const int first = upto - padded;
  if (e < p.num_experts) {
    start[e] = first;
    p.rows[e] = first;
    for (int t = first / p.tile; t < upto / p.tile; ++t) p.tiles[1 + t] = e;
    if (e == p.num_experts - 1) {
      p.rows[e + 1] = upto;
      p.tiles[0] = upto / p.tile;
    }
  }
  // the padding: a warp takes an expert
  if (e < p.num_experts) pad[e] = make_int2(first + count, upto);
  __syncthreads();
  for (int x = warp; x < p.num_experts; x += kWarps)
    for (int r = pad[x].x + lane; r < pad[x].y; r += 32) p.src_of[r] = -1;
  __syncthreads();
}

// base[e]: the chunk's first row of expert e; count[warp][e] becomes the warp's
__device__ __forceinline__ void scatter_chunk(const ExpertPlan& p, int64_t first, int share, int (*count)[kMaxExperts],
                                              const int* base) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.num_experts; e += kThreads) {
    int at = base[e];
    for (int w = 0; w < kWarps; ++w) {
      const int c = count[w][e];
      count[w][e] = at;
      at += c;
    }
  }
  __syncthreads();
  each_assignment(p, first + warp * share, share, [&](int64_t a, int e) {
    const unsigned same = __match_any_sync(0xffffffffu, e), before = same & ((1u << lane) - 1);
    int row = -1;
    if (e >= 0) row = count[warp][e] + __popc(before);
    __syncwarp();
    if (e >= 0 && before == 0) count[warp][e] += __popc(same);
    __syncwarp();
    if (a < p.count) {
      p.row_of[a] = row;
      if (row >= 0) p.src_of[row] = (int)a;
    }
  });
}

// one chunk: all of it in one launch
__global__ void __launch_bounds__(kThreads) plan_one_kernel(const ExpertPlan p) {
  __shared__ int count[kWarps][kMaxExperts], start[kMaxExperts];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int share = (int)((p.count + 32 * kWarps - 1) / (32 * kWarps)) * 32;
  count_chunk(p, 0, share, count);
  __syncthreads();
  int n = 0;
  if (threadIdx.x < p.num_experts)
    for (int w = 0; w < kWarps; ++w) n += count[w][threadIdx.x];
  place_experts(p, n, start);
  scatter_chunk(p, 0, share, count, start);
}

__global__ void __launch_bounds__(kThreads) plan_count_kernel(const ExpertPlan p) {
  __shared__ int count[kWarps][kMaxExperts];
  count_chunk(p, (int64_t)blockIdx.x * kChunk, kChunk / kWarps, count);
  __syncthreads();
  if (threadIdx.x >= p.num_experts) return;
  int n = 0;
  for (int w = 0; w < kWarps; ++w) n += count[w][threadIdx.x];
  p.hist[(int64_t)blockIdx.x * p.num_experts + threadIdx.x] = n;
}
// hist becomes every chunk's first row of every expert
__global__ void __launch_bounds__(kThreads) plan_place_kernel(const ExpertPlan p, int chunks) {
  __shared__ int start[kMaxExperts];
  const int e = threadIdx.x;
  int* hist = p.hist + e;
  // eight chunks' loads leave together: one behind a store that might alias it waits
  const auto load8 = [&](int c, int* m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = c + i < chunks ? hist[(int64_t)(c + i) * p.num_experts] : 0;
  };
  int n = 0, m[8];
  if (e < p.num_experts)
    for (int c = 0; c < chunks; c += 8) {
      load8(c, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) n += m[i];
    }
  place_experts(p, n, start);
  if (e >= p.num_experts) return;
  int at = start[e];
  for (int c = 0; c < chunks; c += 8) {
    load8(c, m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i < chunks) hist[(int64_t)(c + i) * p.num_experts] = at;
      at += m[i];
    }
  }
}
__global__ void __launch_bounds__(kThreads) plan_scatter_kernel(const ExpertPlan p) {
  __shared__ int count[kWarps][kMaxExperts];
  count_chunk(p, (int64_t)blockIdx.x * kChunk, kChunk / kWarps, count);
  __syncthreads();
  scatter_chunk(p, (int64_t)blockIdx.x * kChunk, kChunk / kWarps, count, p.hist + (int64_t)blockIdx.x * p.num_experts);
}

// ------------------------------------------------------------------------------------------- gather and combine
// eight elements at p of which `left` are the row's; NC: by the read-only path, which stores do not hold up.  That path
// is for what was complete before the first of a chain of programmatic dependents began (the caller's tensors): a kernel
// that is resident while the one before it still writes takes what that one leaves by ordinary loads, behind its wait.
template <bool VEC, bool NC>
__device__ __forceinline__ uint4 row8(const uint16_t* p, int64_t left) {
  if (VEC && NC) return __ldg(reinterpret_cast<const uint4*>(p));
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp takes a token, 16 bytes a lane and step.  The loads of a step (kSpan column groups of it, two of its rows) leave
// together and know of no branch: at 1024 columns and two experts a token that alone took the combining sum of 64800
// tokens from 118 to 81 us, the weighted gather from 140 to 113 and the plain one from 81 to 65.  With the rows by
// ordinary loads (see row8) the combining sum takes 91 us (5.8 TB/s), that of dx 69.
constexpr int kRowWarps = 8, kSpan = 2;
template <typename T, bool WEIGHTED, bool VEC>
__global__ void __launch_bounds__(32 * kRowWarps, 4) gather_kernel(const ExpertPlan plan, const ExpertGather a) {
  const int lane = threadIdx.x & 31, k = (int)a.k;
  const int64_t warp = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5), warps = (int64_t)gridDim.x * kRowWarps;
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.dst);
  // (in this order: what follows this kernel may read the plan before it waits)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint16_t* other = reinterpret_cast<const uint16_t*>(a.other);
  const int64_t tokens = plan.count / k;
  for (int64_t t = warp; t < tokens; t += warps) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(a.rows) + t * a.ld_rows;
    // lane i holds the token's i-th row and weight (kMaxChosen <= 32), and the dot product that is its weight's gradient
    const int my_row = lane < k ? plan.row_of[t * k + lane] : -1;
    const float my_weight = WEIGHTED && lane < k ? load_any(a.weights, a.weight_dtype, t * k + lane) : 1.f;
    float my_dot = 0.f;
    for (int64_t c0 = 8 * lane; c0 - 8 * lane < a.n; c0 += 256 * kSpan) {
      uint4 in[kSpan];
#pragma unroll
      for (int j = 0; j < kSpan; ++j) {
        const int64_t c = c0 + 256 * j;
        in[j] = c < a.n ? row8<VEC, true>(p + c, a.n - c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll 2
      for (int i = 0; i < k; ++i) {
        const int row = __shfl_sync(0xffffffffu, my_row, i);
        const float w = __shfl_sync(0xffffffffu, my_weight, i);
        uint4 o[kSpan];
        if (WEIGHTED && a.dweights) {
#pragma unroll
          for (int j = 0; j < kSpan; ++j) {
            const int64_t c = c0 + 256 * j;
            o[j] = c < a.n && row >= 0 ? row8<true, true>(other + row * a.ld_other + c, 8) : make_uint4(0, 0, 0, 0);
          }
        }
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < kSpan; ++j) {
          const int64_t c = c0 + 256 * j;
          if (c >= a.n || row < 0) continue;
          uint4* d = reinterpret_cast<uint4*>(dst + row * a.ld_dst + c);
          if (!WEIGHTED) {
            *d = in[j];
            continue;
          }
          float f[8], g[8];
          unpack8<T>(in[j], f);
          if (a.dweights) {
            unpack8<T>(o[j], g);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (VEC || c + x < a.n) dot = fmaf(f[x], g[x], dot);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] *= w;
          *d = pack8<T>(f);
        }
        if (WEIGHTED && a.dweights) {
          dot = warp_sum(dot);
          if (lane == i) my_dot += dot;
        }
      }
    }
    if (WEIGHTED && a.dweights && lane < k) store_any(a.dweights, a.weight_dtype, t * k + lane, my_dot);
  }
  // the padding's zeros; lane i looks at the warp's i-th row of 32
  const int64_t rows = (int64_t)*plan.tiles * plan.tile;
  for (int64_t r0 = warp; r0 < rows; r0 += 32 * warps) {
    const int64_t mine = r0 + lane * warps;
    unsigned empty = __ballot_sync(0xffffffffu, mine < rows && plan.src_of[mine] < 0);
    for (; empty; empty &= empty - 1) {
      uint16_t* d = dst + (r0 + (__ffs(empty) - 1) * warps) * a.ld_dst;
      for (int64_t c = 8 * lane; c < a.n; c += 256) *reinterpret_cast<uint4*>(d + c) = make_uint4(0, 0, 0, 0);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * kRowWarps, 4) combine_kernel(const ExpertCombine a) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5), warps = (int64_t)gridDim.x * kRowWarps;
  const int k = (int)a.k;
  const uint16_t* rows = reinterpret_cast<const uint16_t*>(a.rows);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t t = warp; t < a.tokens; t += warps) {
    const uint16_t* res = reinterpret_cast<const uint16_t*>(a.residual) + t * a.ld_res;
    T* out = reinterpret_cast<T*>(a.out) + t * a.ld_out;
    // lane i holds the token's i-th row and weight (kMaxChosen <= 32)
    const int my_row = lane < k ? a.row_of[t * k + lane] : -1;
    const float my_weight = lane < k && a.weights ? load_any(a.weights, a.weight_dtype, t * k + lane) : 1.f;
    for (int64_t c0 = 8 * lane; c0 - 8 * lane < a.n; c0 += 256 * kSpan) {
      float f[kSpan][8];
#pragma unroll
      for (int j = 0; j < kSpan; ++j) {
        const int64_t c = c0 + 256 * j;
        unpack8<T>(a.residual && c < a.n ? row8<VEC, true>(res + c, a.n - c) : make_uint4(0, 0, 0, 0), f[j]);
      }
      for (int i0 = 0; i0 < k; i0 += 2) {
        uint4 in[2][kSpan];
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = i0 + i < k ? __shfl_sync(0xffffffffu, my_row, i0 + i) : -1;
          w[i] = __shfl_sync(0xffffffffu, my_weight, i0 + i);
          if (row < 0) w[i] = 0.f;  // (its row counts as zeros, whatever the weight)
#pragma unroll
          for (int j = 0; j < kSpan; ++j) {
            const int64_t c = c0 + 256 * j;
            in[i][j] = row >= 0 && c < a.n ? row8<true, false>(rows + row * a.ld_rows + c, 8) : make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < kSpan; ++j) {
            float g[8];
            unpack8<T>(in[i][j], g);
#pragma unroll
            for (int x = 0; x < 8; ++x) f[j][x] = fmaf(w[i], g[x], f[j][x]);
          }
      }
#pragma unroll
      for (int j = 0; j < kSpan; ++j) {
        const int64_t c = c0 + 256 * j;
        if (c >= a.n) continue;
        if (VEC) {
          *reinterpret_cast<uint4*>(out + c) = pack8<T>(f[j]);
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (c + x < a.n) out[c + x] = from_f<T>(f[j][x]);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ few assignments
// Bound by reading the chosen experts' weights once.  A warp takes a row of a matrix (of Wg and of Wu at once), 16
// bytes a lane and step; there are rows enough that all of them are in flight together.
//   up    block (8 hidden units, assignment s): if s is the first assignment of its expert, h of the expert's every
//         assignment, four at a time; other blocks end at once.
//   down  block (8 outputs, token): the weighted sum over the token's experts in one warp's registers; the weights are
//         on their way to L2 before the wait for the kernel that writes h.
constexpr int kFewGroup = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) few_up_kernel(const ExpertFew a) {
  __shared__ int list[kExpertFewRows];
  __shared__ int listed;
  const int lane = threadIdx.x & 31, total = a.tokens * a.k, s = blockIdx.y;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t e = a.experts[s];
  if (e < 0 || e >= a.num_experts) return;
  if (threadIdx.x < 32) {  // (kExpertFewRows <= 32)
    const bool same = lane < total && a.experts[lane] == e;
    const unsigned m = __ballot_sync(0xffffffffu, same);
    if (same) list[__popc(m & ((1u << lane) - 1))] = lane;
    if (lane == 0) listed = (m & ((1u << s) - 1)) ? 0 : __popc(m);
  }
  __syncthreads();
  if (listed == 0 || unit >= a.H) return;
  const uint16_t* wg = reinterpret_cast<const uint16_t*>(a.wg) + (e * a.H + unit) * a.ldwg;
  const uint16_t* wu = reinterpret_cast<const uint16_t*>(a.wu) + (e * a.H + unit) * a.ldwu;
  for (int i0 = 0; i0 < listed; i0 += kFewGroup) {
    float g[kFewGroup], u[kFewGroup];
    const uint16_t* x[kFewGroup];
#pragma unroll
    for (int i = 0; i < kFewGroup; ++i) {
      g[i] = u[i] = 0.f;
      x[i] = reinterpret_cast<const uint16_t*>(a.x) + (int64_t)(list[min(i0 + i, listed - 1)] / a.k) * a.ldx;
    }
#pragma unroll 4
    for (int c = 8 * lane; c < a.K; c += 256) {
      float fg[8], fu[8];
      unpack8<T>(row8<VEC, true>(wg + c, a.K - c), fg);
      unpack8<T>(row8<VEC, true>(wu + c, a.K - c), fu);
#pragma unroll
      for (int i = 0; i < kFewGroup; ++i) {
        if (i > 0 && i0 + i >= listed) continue;
        float f[8];
        unpack8<T>(row8<VEC, true>(x[i] + c, a.K - c), f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[i] = fmaf(f[j], fg[j], g[i]);
          u[i] = fmaf(f[j], fu[j], u[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kFewGroup; ++i) {
      if (i0 + i >= listed) break;
      g[i] = warp_sum(g[i]);
      u[i] = warp_sum(u[i]);
      if (lane == 0)
        reinterpret_cast<T*>(a.h)[list[i0 + i] * a.ldh + unit] = from_f<T>(tc::act_parts(g[i], a.act).val * u[i]);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) few_down_kernel(const ExpertFew a) {
  const int lane = threadIdx.x & 31, t = blockIdx.y;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n < a.N)
    for (int j = 0; j < a.k; ++j) {
      const int64_t e = a.experts[t * a.k + j];
      if (e < 0 || e >= a.num_experts) continue;
      const uint16_t* w = reinterpret_cast<const uint16_t*>(a.wd) + (e * a.N + n) * a.ldwd;
      for (int c = 64 * lane; c < a.H; c += 2048) asm volatile("prefetch.global.L2 [%0];" ::"l"(w + c));
    }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n >= a.N) return;
  float y = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int64_t e = a.experts[t * a.k + j];
    if (e < 0 || e >= a.num_experts) continue;
    const uint16_t* w = reinterpret_cast<const uint16_t*>(a.wd) + (e * a.N + n) * a.ldwd;
    const uint16_t* h = reinterpret_cast<const uint16_t*>(a.h) + (t * a.k + j) * a.ldh;
    float dot = 0.f;
#pragma unroll 4
    for (int c = 8 * lane; c < a.H; c += 256) {
      float f[8], g[8];
      unpack8<T>(row8<VEC, true>(w + c, a.H - c), f);
      unpack8<T>(row8<VEC, false>(h + c, a.H - c), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(f[i], g[i], dot);
    }
    y = fmaf(load_any(a.weights, a.weight_dtype, t * a.k + j), dot, y);
  }
  y = warp_sum(y);
  if (lane == 0) {
    if (a.residual) y += to_f(reinterpret_cast<const T*>(a.residual)[t * a.ldres + n]);
    reinterpret_cast<T*>(a.y)[(int64_t)t * a.N + n] = from_f<T>(y);
  }
}

template <typename T, bool VEC>
static cudaError_t launch_few(const ExpertFew& a, cudaStream_t s) {
  few_up_kernel<T, VEC><<<dim3((a.H + 7) / 8, a.tokens * a.k), 256, 0, s>>>(a);
  NSW_CUDA_CHECK(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((a.N + 7) / 8, a.tokens);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few_down_kernel<T, VEC>, a);
}

// dependent: a programmatic dependent of the kernel before it on the stream
template <typename... P, typename... A>
static cudaError_t launch(void (*k)(P...), int blocks, bool dependent, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(32 * kRowWarps);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, args...);
}

static bool aligned(const void* p, int64_t ld) { return ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace experts

int64_t expert_tiles(int64_t count, int64_t experts, int tile) {
  return (count + (tile - 1) * std::min(count, experts)) / tile;
}
// Up to 48 rows an expert on average (in every expert) the split products, whose tiles are 32 or 64 rows, read the
// weights about as fast as gated_kernel with its 256-row tiles and start and end sooner; so they do up to 512 rows while
// their blocks are few, three an SM, or five where most experts have one tile yet.  Microseconds of a call without gradients, in a
// graph, weights not in L2, tiles of 32 / 64 / 256 rows, and 64-row tiles' blocks of the up projection:
//   2 experts of 768 x 1024:    512 rows 43 / 35 / 39 (272),  1024 - / 51 / 43 (528)
//   2 of 1024 x 4096:           128 rows 47 / 41 / 57 (320),  192 59 / 51 / 57 (448),  384 96 / 68 / 66 (832)
//   8 of 1024 x 2736:           8 rows 55 / 59 / 72,  32 57 / 62 / 70,  64 76 / 66 / 72 (645),  96 84 / 78 / 72 (817)
//   32 of 768 x 512:            48 rows 57 / 49 / 57,  64 64 / 55 / 58 (504),  96 79 / 68 / 61 (632)
//   64 of 1024 x 1368:          16 rows 140 / 152 / 162,  48 201 / 162 / 168 (2442),  64 236 / 195 / 172 (2794)
//   4 of 128 x 344:             16 rows 21 / 21 / 31,  512 33 / 30 / 33 (210),  1024 - / 39 / 37 (402)
//   128 of 256 x 344:           8 rows 51 / 53 / 64,  48 82 / 70 / 74 (1332),  64 94 / 82 / 74 (1524)
int expert_tile(int64_t count, int64_t experts, int64_t H, int64_t N) {
  if (experts * std::max(H, N) >= INT32_MAX) return kExpertTile;  // (the split products' rows of all experts' weights)
  if (count <= 24 * experts) return 32;
  if (count <= 48 * experts) return 64;
  const int64_t blocks = expert_tiles(count, experts, 64) * ((H + 63) / 64);
  return count <= 512 * experts && blocks <= (count <= 64 * experts ? 5 : 3) * tc::sm_count() ? 64 : kExpertTile;
}
static int64_t plan_chunks(int64_t count) {
  return count <= experts::kOneChunk ? 1 : (count + experts::kChunk - 1) / experts::kChunk;
}
int64_t expert_plan_hist(int64_t count, int64_t num_experts) {
  const int64_t chunks = plan_chunks(count);
  return chunks > 1 ? chunks * num_experts : 0;
}

cudaError_t expert_plan(const ExpertPlan& p, cudaStream_t s) {
  if (p.num_experts < 1 || p.num_experts > kMaxExperts || p.count < 1 || p.tile < 1) return cudaErrorInvalidValue;
  const int chunks = (int)plan_chunks(p.count);
  if (chunks == 1) {
    experts::plan_one_kernel<<<1, experts::kThreads, 0, s>>>(p);
    return cudaGetLastError();
  }
  experts::plan_count_kernel<<<chunks, experts::kThreads, 0, s>>>(p);
  experts::plan_place_kernel<<<1, experts::kThreads, 0, s>>>(p, chunks);
  experts::plan_scatter_kernel<<<chunks, experts::kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t expert_gather(const ExpertGather& a, bool dependent, cudaStream_t s) {
  const int64_t rows = a.plan->tile * expert_tiles(a.plan->count, a.plan->num_experts, a.plan->tile);
  const int blocks = (int)std::min<int64_t>((rows + experts::kRowWarps - 1) / experts::kRowWarps, 4 * tc::sm_count());
  if (!experts::aligned(a.dst, a.ld_dst) || (a.dweights && !experts::aligned(a.other, a.ld_other)))
    return cudaErrorInvalidValue;
  const bool vec = experts::aligned(a.rows, a.ld_rows) && a.n % 8 == 0;
#define NSW_GATHER(T, W, V) return experts::launch(experts::gather_kernel<T, W, V>, blocks, dependent, s, *a.plan, a)
  if (!a.weights) {  // a copy: either 16-bit type
    if (vec)
      NSW_GATHER(__half, false, true);
    else
      NSW_GATHER(__half, false, false);
  } else if (a.dtype == kBF16) {
    if (vec)
      NSW_GATHER(__nv_bfloat16, true, true);
    else
      NSW_GATHER(__nv_bfloat16, true, false);
  } else {
    if (vec)
      NSW_GATHER(__half, true, true);
    else
      NSW_GATHER(__half, true, false);
  }
#undef NSW_GATHER
}

cudaError_t expert_combine(const ExpertCombine& a, bool dependent, cudaStream_t s) {
  if (!experts::aligned(a.rows, a.ld_rows)) return cudaErrorInvalidValue;
  const int blocks = (int)std::min<int64_t>((a.tokens + experts::kRowWarps - 1) / experts::kRowWarps, 4 * tc::sm_count());
  const bool vec = a.n % 8 == 0 && experts::aligned(a.out, a.ld_out) &&
                   (!a.residual || experts::aligned(a.residual, a.ld_res));
#define NSW_COMBINE(T, V) return experts::launch(experts::combine_kernel<T, V>, blocks, dependent, s, a)
  if (a.dtype == kBF16) {
    if (vec)
      NSW_COMBINE(__nv_bfloat16, true);
    else
      NSW_COMBINE(__nv_bfloat16, false);
  } else {
    if (vec)
      NSW_COMBINE(__half, true);
    else
      NSW_COMBINE(__half, false);
  }
#undef NSW_COMBINE
}

// The kernels for a few assignments read an expert's weights for each of them, the others once; from 64 MB of them on that
// costs more than sorting.  Microseconds as above, here and by tiles of 32 rows: 2 experts of 768 x 1024 (4.7 MB): 4
// assignments 14 / 24, 12 21 / 24, 24 33 / 24; 8 of 1024 x 2736 (16.8 MB): 4 39 / 37, 12 53 / 45; 64 of 512 x 680 (2.1 MB):
// 4 14 / 23, 32 31 / 35; 4 of 128 x 344: 4 10 / 20, 32 14 / 18.
bool expert_few_pays(int64_t count, int64_t H, int64_t K, int64_t N) {
  return count <= kExpertFewRows && count * H * (2 * K + N) <= (int64_t)32 << 20;
}

cudaError_t expert_few(const ExpertFew& a, cudaStream_t s) {
  if (a.tokens < 1 || a.k < 1 || a.tokens * a.k > kExpertFewRows) return cudaErrorInvalidValue;
  const bool vec = a.K % 8 == 0 && a.H % 8 == 0 && experts::aligned(a.x, a.ldx) && experts::aligned(a.wg, a.ldwg) &&
                   experts::aligned(a.wu, a.ldwu) && experts::aligned(a.wd, a.ldwd) && experts::aligned(a.h, a.ldh);
  if (a.dtype == kBF16)
    return vec ? experts::launch_few<__nv_bfloat16, true>(a, s) : experts::launch_few<__nv_bfloat16, false>(a, s);
  return vec ? experts::launch_few<__half, true>(a, s) : experts::launch_few<__half, false>(a, s);
}

}  // namespace nsw
