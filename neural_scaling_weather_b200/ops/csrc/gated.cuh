// Device helpers shared by the gated feed-forward networks' kernels, dense and routed: the activations and their slopes,
// and biases of any type.
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

}  // namespace tc
}  // namespace nsw
