// Device helpers shared by the gated feed-forward networks' kernels, dense and routed: the activations and their
// slopes, biases of any type, cluster reads, and the warp-level products of a few tokens.
#pragma once

#include "tcgen05.cuh"

namespace nsw {
namespace tc {

// act(g) and act'(g), whose exponential and reciprocal are the hardware approximations (2 ulp); exp(-g) = inf gives
// sig = 0.  GELU is g Phi(g) with the tail Phi(-a) = exp(-a^2 / 2) H(a), a = |g|, taken as it is for g < 0: as
// 1 - (1 - tail) it would keep only what fp32 holds beside 1, nothing of it below -5.5.  H(a) = exp(a^2 / 2) Phi(-a),
// which falls from 1/2 like 1 / a, is a polynomial in t = 1 / (1 + p a) without constant term, fitted to it over
// 0 <= a <= 13.5 (where the tail leaves fp32's normal numbers) for the smallest largest relative error, 3.7e-6.  With
// fp32's roundings, act and act' have relative errors below 1e-5 at any g (act' around its zero at -0.75: 1e-6 of
// one), a fiftieth of fp16's half spacing.
struct ActParts {
  float val, slope;
};
__device__ __forceinline__ ActParts act_parts(float g, int act) {
  ActParts r;
  float e;
  if (act == 0) {
    float sig;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.44269504088896340736f * g));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(sig) : "f"(1.0f + e));
    r.val = g * sig;
    r.slope = fmaf(r.val, 1.0f - sig, sig);
  } else {
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(fabsf(g), 0.30764427f, 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-g * g * 0.72134752044448170368f));
    float h = fmaf(t, -0.0758030088f, 0.19158072f);
    h = fmaf(t, h, 0.00538051427f);
    h = fmaf(t, h, 0.137291841f);
    h = fmaf(t, h, 0.118551773f);
    h = fmaf(t, h, 0.122996339f);
    const float tail = t * h * e;
    const float cdf = g < 0.f ? tail : 1.0f - tail;
    r.val = g * cdf;
    r.slope = fmaf(g, e * 0.39894228040143267794f, cdf);
  }
  return r;
}

__device__ __forceinline__ float ld_bias(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dtype == kBF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
  float4 o;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w)
               : "r"(at)
               : "memory");
  return o;
}

}  // namespace tc

namespace gated {

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

}  // namespace gated
}  // namespace nsw
