// The router of a block with routed experts: for each token the k largest of E logits, their weights, and the balance
// of the choices over the experts.
//
//   p = softmax(z);  chosen = top k of z, equal values in the order of their indices
//   w_j = exp(z_cj - z_c0) / sum_i exp(z_ci - z_c0) (normalized), or p_cj
//   share_e = E count_e / (k M);  balance = sum_e share_e mean_t p_te
//   dz_e = [e = c_j] w_j (dw_j - sum_i w_i dw_i)                        (normalized)
//          p_e ([e = c_j] dw_j - sum_i p_ci dw_i)                       (not)
//        + dbalance / M p_e (share_e - sum_f p_f share_f)
//
// A token is a group of 8, 16 or 32 lanes, G, whose lane l holds the experts l, l + G, ..., so that a warp's loads are
// contiguous.  The order of two logits is that of their 64-bit keys: the value as an unsigned number of the same order
// (-0 as 0, NaN above all), then the index, inverted; a round of the selection is a maximum over the group's keys.
// Groups walk the tokens in strides of the grid; a lane sums its experts' probabilities in registers, a block adds its
// groups' sums in order and the blocks' rows are added in order by a second kernel, so results repeat bit for bit
// (counts are integers, in any order).  A row that is -inf throughout has weights and probabilities of zero.
//
// Floor: reading the logits once (64800 x 64 bf16: 8.3 MB, 1.3 us).  There the forward takes 16.4 us, the balance's sum 5.8
// and the backward 12: 2.2 and 2.0 instructions a cycle of 4 with a quarter and under half of the warps, which wait for the
// results of their own shuffles and comparisons and for their loads.  A few tokens are bound by the launch.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace nsw {
namespace route {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float load(const void* p, int64_t i) {
  return to_f(reinterpret_cast<const T*>(p)[i]);
}

__device__ __forceinline__ unsigned long long key_of(float z, int index) {
  uint32_t u = __float_as_uint(z + 0.0f);
  if (z != z) u = 0x7fffffffu;
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)u << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)~(uint32_t)key; }

template <int G>
__device__ __forceinline__ unsigned long long group_max(unsigned long long v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exp(z - m), zero for a row without a finite value
__device__ __forceinline__ float shifted_exp(float z, float m) { return m == -INFINITY ? 0.f : expf(z - m); }

// share and balance of one block's own sums (of all of them: a few tokens take one block and one launch)
__device__ __forceinline__ void finish_block(const RouteArgs& a, const float* psum, const int* count, int groups,
                                             float* red) {
  const int E = a.experts;
  float term = 0.f;
  for (int e = threadIdx.x; e < E; e += kThreads) {
    float p = 0.f;
    for (int i = 0; i < groups; ++i) p += psum[i * E + e];
    const float share = a.tokens > 0 ? (float)count[e] * (float)((double)E / ((double)a.tokens * a.k)) : 0.f;
    a.share[e] = share;
    term += a.tokens > 0 ? share * p / (float)a.tokens : 0.f;
  }
  term = warp_sum(term);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) term += red[w];
    *a.balance = term;
  }
}

// All lanes of a warp run the same number of rounds; groups past the last token take part with nothing.
template <typename T, int G, int V>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const RouteArgs a) {
  extern __shared__ float sums[];  // [kThreads / G][experts] probabilities, then [experts] counts
  __shared__ float red[kThreads / 32];
  constexpr int kGroups = kThreads / G;
  const int E = a.experts, k = a.k, l = threadIdx.x % G, group = threadIdx.x / G;
  int* count = reinterpret_cast<int*>(sums + kGroups * E);
  for (int i = threadIdx.x; i < E; i += kThreads) count[i] = 0;
  __syncthreads();
  float psum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) psum[i] = 0.f;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  for (int64_t t0 = (int64_t)blockIdx.x * kGroups; t0 < a.tokens; t0 += step) {
    const int64_t t = t0 + group;
    const bool live = t < a.tokens;
    unsigned long long key[V];
    float z[V];
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = l + G * i;
      key[i] = 0;  // below every logit's
      z[i] = -INFINITY;
      if (live && e < E) {
        z[i] = load<T>(a.logits, t * a.ld + e);
        key[i] = key_of(z[i], e);
      }
      best = key[i] > best ? key[i] : best;
    }
    best = group_max<G>(best);
    const float m = live ? key_value(best) : 0.f;
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      z[i] = live && l + G * i < E ? shifted_exp(z[i], m) : 0.f;
      total += z[i];
    }
    total = group_sum<G>(total);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < V; ++i) psum[i] += z[i] * inv;
    // k rounds; the j-th choice stays with lane j % G (two at most: k <= 16)
    unsigned long long mine[2] = {0, 0};
    float chosen_sum = 0.f;
    for (int j = 0; j < k; ++j) {
      if (j > 0) {
        best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) best = key[i] > best ? key[i] : best;
        best = group_max<G>(best);
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (key[i] == best) key[i] = 0;
      if (l == j % G) {
        if (j < G)
          mine[0] = best;
        else
          mine[1] = best;
      }
      chosen_sum += shifted_exp(key_value(best), m);
    }
    const float scale = !a.normalize ? inv : chosen_sum == 0.f ? 0.f : 1.0f / chosen_sum;
    if (live) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = l + G * i;
        if (j >= k) break;
        const int e = key_index(mine[i]);
        a.weights[t * k + j] = shifted_exp(key_value(mine[i]), m) * scale;
        a.chosen[t * k + j] = e;
        atomicAdd(&count[e], 1);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (l + G * i < E) sums[group * E + l + G * i] = psum[i];
  __syncthreads();
  if (gridDim.x == 1) return finish_block(a, sums, count, kGroups, red);
  float* psums = reinterpret_cast<float*>(a.partial);
  int* counts = reinterpret_cast<int*>(psums + (int64_t)gridDim.x * E);
  for (int e = threadIdx.x; e < E; e += kThreads) {
    float s = 0.f;
    for (int i = 0; i < kGroups; ++i) s += sums[i * E + e];
    psums[(int64_t)blockIdx.x * E + e] = s;
    counts[(int64_t)blockIdx.x * E + e] = count[e];
  }
}

// The blocks' sums, in order: slices of the blocks for each expert, then the slices; then over the experts
__global__ void __launch_bounds__(1024) balance_kernel(const RouteArgs a, int blocks) {
  __shared__ float ps[1024];
  __shared__ int cs[1024];
  const int E = a.experts, slices = 1024 / E, e = threadIdx.x % E, slice = threadIdx.x / E;
  const float* psums = reinterpret_cast<const float*>(a.partial);
  const int* counts = reinterpret_cast<const int*>(psums + (int64_t)blocks * E);
  float p = 0.f;
  int c = 0;
  if (slice < slices)
#pragma unroll 8
    for (int b = slice; b < blocks; b += slices) {
      p += psums[(int64_t)b * E + e];
      c += counts[(int64_t)b * E + e];
    }
  ps[threadIdx.x] = p;
  cs[threadIdx.x] = c;
  __syncthreads();
  float term = 0.f;
  if (threadIdx.x < E) {
    for (int s = 1; s < slices; ++s) {
      p += ps[s * E + e];
      c += cs[s * E + e];
    }
    const float share = a.tokens > 0 ? (float)c * (float)((double)E / ((double)a.tokens * a.k)) : 0.f;
    a.share[e] = share;
    term = a.tokens > 0 ? share * p / (float)a.tokens : 0.f;
  }
  __syncthreads();
  ps[threadIdx.x] = term;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) ps[threadIdx.x] += ps[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *a.balance = ps[0];
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const RouteArgs a) {
  constexpr int kGroups = kThreads / G;
  const int E = a.experts, k = a.k, l = threadIdx.x % G, group = threadIdx.x / G;
  const float db = a.dbalance ? *a.dbalance / (float)a.tokens : 0.f;
  float share[V];
#pragma unroll
  for (int i = 0; i < V; ++i) share[i] = l + G * i < E ? a.share[l + G * i] : 0.f;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  for (int64_t t0 = (int64_t)blockIdx.x * kGroups; t0 < a.tokens; t0 += step) {
    const int64_t t = t0 + group;
    const bool live = t < a.tokens;
    float z[V];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = l + G * i;
      z[i] = live && e < E ? load<T>(a.logits, t * a.ld + e) : -INFINITY;
      m = fmaxf(m, z[i]);
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float total = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      z[i] = shifted_exp(z[i], m);
      total += z[i];
    }
    total = group_sum<G>(total);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      z[i] *= inv;
      dot = fmaf(z[i], share[i], dot);
    }
    dot = group_sum<G>(dot);
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = db * z[i] * (share[i] - dot);
    if (a.dweights) {
      float wd = 0.f;
      if (live)
        for (int j = 0; j < k; ++j) wd = fmaf(a.weights[t * k + j], a.dweights[t * k + j], wd);
      if (!a.normalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = fmaf(-z[i], wd, d[i]);
      }
      if (live)
        for (int j = 0; j < k; ++j) {
          const int e = (int)a.chosen[t * k + j];
          const float g = a.weights[t * k + j] * (a.dweights[t * k + j] - (a.normalize ? wd : 0.f));
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (e == l + G * i) d[i] += g;
        }
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (l + G * i < E) reinterpret_cast<T*>(a.dlogits)[t * E + l + G * i] = from_f<T>(d[i]);
    }
  }
}

// As few lanes a token as hold its logits in 16 registers each: fewer shuffles for more tokens at once.  Forward and backward
// of 64800 tokens, us: 64 experts 16.5 + 12.3 by 8 lanes, 35.0 + 20.4 by 32; 128 experts 25.2 + 20.9 by 8, 42.2 + 25.9 by 32;
// 150 experts 46.6 + 34.7 by 16, 59.4 + 35.3 by 32.  (100 tokens of 128: 4.6 by 8, 3.1 by 32.)
template <typename F>
cudaError_t by_width(int experts, F f) {
  if (experts <= 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
  if (experts <= 16) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 2>());
  if (experts <= 32) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 4>());
  if (experts <= 64) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  if (experts <= 128) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 16>());
  if (experts <= 256) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>(), std::integral_constant<int, 16>());
}
template <typename F>
cudaError_t by_type(int dtype, F f) {
  if (dtype == kBF16) return f(__nv_bfloat16());
  if (dtype == kF16) return f(__half());
  return f(float());
}
int groups(int experts) { return kThreads / (experts <= 128 ? 8 : experts <= 256 ? 16 : 32); }

}  // namespace route

// Two blocks an SM: 64800 x 64 with the balance's sum 25.7 us a call, with one 33.9, with four 25.6, with eight 29.8
int route_blocks(int64_t tokens, int experts, int sms) {
  const int64_t need = (tokens + route::groups(experts) - 1) / route::groups(experts);
  return (int)(need < 1 ? 1 : need < 2 * sms ? need : 2 * sms);
}

static bool route_ok(const RouteArgs& a) {
  return a.experts >= 1 && a.experts <= kMaxExperts && a.k >= 1 && a.k <= kMaxChosen && a.k <= a.experts &&
         (a.dtype == kBF16 || a.dtype == kF16 || a.dtype == kF32);
}

cudaError_t route_fwd(const RouteArgs& a, int blocks, cudaStream_t s) {
  if (!route_ok(a)) return cudaErrorInvalidValue;
  NSW_CUDA_CHECK(route::by_type(a.dtype, [&](auto t) {
    return route::by_width(a.experts, [&](auto g, auto v) {
      const size_t smem = (size_t)(route::kThreads / g() + 1) * a.experts * 4;
      route::fwd_kernel<decltype(t), g(), v()><<<blocks, route::kThreads, smem, s>>>(a);
      return cudaGetLastError();
    });
  }));
  if (blocks > 1) route::balance_kernel<<<1, 1024, 0, s>>>(a, blocks);
  return cudaGetLastError();
}

cudaError_t route_bwd(const RouteArgs& a, int sms, cudaStream_t s) {
  if (!route_ok(a) || a.tokens <= 0) return cudaErrorInvalidValue;
  const int64_t need = (a.tokens + route::groups(a.experts) - 1) / route::groups(a.experts);
  const int blocks = (int)(need < 8 * sms ? need : 8 * sms);
  return route::by_type(a.dtype, [&](auto t) {
    return route::by_width(a.experts, [&](auto g, auto v) {
      route::bwd_kernel<decltype(t), g(), v()><<<blocks, route::kThreads, 0, s>>>(a);
      return cudaGetLastError();
    });
  });
}

}  // namespace nsw
