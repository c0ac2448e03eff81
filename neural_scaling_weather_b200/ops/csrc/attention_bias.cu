// The learned relative position bias of window attention: the entries as the attention kernels read them, and its
// gradient from their partial sums.
//
//   logit_ij += table[head, bucket(i, j)],
//   bucket = ((t_i - t_j + T - 1) (2 wh - 1) + y_i - y_j + wh - 1) (2 ww - 1) + x_i - x_j + ww - 1
//
// A head's entries (at most 1155 for windows of up to 192 tokens) are kept in shared memory, where a row's entry for a
// key is at off(row) - off(key), off linear in the token's place.  Rows of a warp are consecutive tokens; where there is
// room the pitch of a latitude is raised until it is ww modulo 32, so that they read consecutive banks.
#include <float.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace nsw {
namespace attn_bias {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == kBF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(reinterpret_cast<const __half*>(p)[i]);
}

// One block a head, and one for the norms' weights.  Entries are less the head's largest, so that an offset of all of them
// costs no precision, unless that is beyond 2^40: a head of the lowest value throughout, say, absorbs the logits, as it
// does in 64 bits, and its rows are even.  A finite entry stays finite.
__global__ void __launch_bounds__(256) prepare_kernel(const AnyMatrix table, const AnyMatrix qw, const AnyMatrix kw, int heads,
                                                      int hd, int nx, int rows, int pitch, int stride,
                                                      float* __restrict__ tab) {
  __shared__ float hi_w[8], lo_w[8];
  const int h = blockIdx.x, n = rows * nx;
  float* out = tab + (int64_t)h * stride;
  if (h == heads) {
    for (int i = threadIdx.x; i < hd; i += 256) {
      out[i] = load_any(qw.p, qw.dtype, i * qw.s0);
      out[hd + i] = load_any(kw.p, kw.dtype, i * kw.s0);
    }
    return;
  }
  float hi = -INFINITY, lo = INFINITY;
  for (int i = threadIdx.x; i < n; i += 256) {
    const float v = load_any(table.p, table.dtype, h * table.s0 + i * table.s1);
    hi = fmaxf(hi, v);
    lo = fminf(lo, v);
  }
  hi = warp_max(hi);
  lo = -warp_max(-lo);
  if ((threadIdx.x & 31) == 0) hi_w[threadIdx.x >> 5] = hi, lo_w[threadIdx.x >> 5] = lo;
  __syncthreads();
  for (int w = 0; w < 8; ++w) hi = fmaxf(hi, hi_w[w]), lo = fminf(lo, lo_w[w]);
  const bool shifted = fabsf(hi) <= 1099511627776.f;
  const float shift = shifted ? hi : 0.f;
  const auto entry = [&](float v) {
    const float e = (v - shift) * kLog2e;
    return isinf(e) && !isinf(v) ? copysignf(FLT_MAX, e) : e;
  };
  for (int i = threadIdx.x; i < stride; i += 256) {
    const int at = i - 4, row = at / pitch, x = at - row * pitch;
    float v = 0.f;
    if (i == 0)
      v = shifted ? -entry(lo) : INFINITY;  // (the forward's bound on the logits needs the largest to be 0)
    else if (at >= 0 && row < rows && x < nx)
      v = entry(load_any(table.p, table.dtype, h * table.s0 + (row * nx + x) * table.s1));
    out[i] = v;
  }
}

// Sums of columns of partial rows, in order: blockIdx.y is a head of the bias, or q's or k's norm weights.  tc: block c of
// `grid` walked items [n c / grid, n (c + 1) / grid) of the head-major list and left its sums for head h in row c + h;
// otherwise each (head, window) has a row.
struct Grads {
  AttnGrad bias, q, k;
  int64_t windows, qk_rows;
  int heads, grid, buckets, hd;
  float unit;
};
__global__ void __launch_bounds__(1024) grad_kernel(const Grads p) {
  __shared__ float red[32][33];
  const int h = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const bool head = h < p.heads;
  const AttnGrad& t = head ? p.bias : h == p.heads ? p.q : p.k;
  const int n = head ? p.buckets : p.hd;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  if (!t.out || (int64_t)blockIdx.x * 32 >= n) return;
  int64_t first = 0, last = p.qk_rows - 1;
  if (head) {
    const int64_t items = p.windows * p.heads;
    first = h * p.windows;
    last = first + p.windows - 1;
    if (p.grid > 0) {
      first = ((first + 1) * p.grid - 1) / items + h;
      last = ((last + 1) * p.grid - 1) / items + h;
    }
  }
  float a = 0.f;
  if (c < n) {
#pragma unroll 4
    for (int64_t r = first + w; r <= last; r += 32) a += t.part[r * n + c];
  }
  red[w][lane] = a;
  __syncthreads();
  if (w || c >= n) return;
  for (int i = 1; i < 32; ++i) a += red[i][lane];
  if (head) a /= p.unit;
  const int64_t at = (head ? (int64_t)h * n : 0) + c;
  if (t.add) a += reinterpret_cast<const float*>(t.out)[at];
  if (t.dtype == kF32)
    reinterpret_cast<float*>(t.out)[at] = a;
  else if (t.dtype == kBF16)
    reinterpret_cast<__nv_bfloat16*>(t.out)[at] = from_f<__nv_bfloat16>(a);
  else
    reinterpret_cast<__half*>(t.out)[at] = from_f<__half>(a);
}

}  // namespace attn_bias

static int bias_rows(const AttnGeom& g) { return (2 * g.T - 1) * (2 * g.wh - 1); }

AttnBias attn_bias_layout(const AttnGeom& g) {
  const int nx = 2 * g.ww - 1, rows = bias_rows(g);
  int pitch = nx;
  while (pitch % 32 != g.ww % 32) ++pitch;
  if (4 + rows * pitch > kAttnBiasRow) pitch = nx;
  return {nullptr, (4 + rows * pitch + 3) / 4 * 4, pitch};
}

cudaError_t attn_bias_prepare(const AnyMatrix& table, const AnyMatrix& qw, const AnyMatrix& kw, const AttnGeom& g,
                              const AttnBias& b, float* tab, cudaStream_t s) {
  if (b.stride > kAttnBiasRow) return cudaErrorInvalidValue;
  attn_bias::prepare_kernel<<<g.nh + 1, 256, 0, s>>>(table, qw, kw, g.nh, g.hd, 2 * g.ww - 1, bias_rows(g), b.pitch,
                                                     b.stride, tab);
  return cudaGetLastError();
}

int64_t attn_bias_rows(const AttnGeom& g, bool tc, int sms) {
  const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
  return tc ? std::min<int64_t>(items, sms) + g.nh - 1 : items;
}

cudaError_t attn_bias_grads(const AttnGrad& bias, const AttnGrad& q, const AttnGrad& k, int64_t qk_rows, const AttnGeom& g,
                            bool tc, int sms, cudaStream_t s) {
  attn_bias::Grads p{};
  p.bias = bias;
  p.q = q;
  p.k = k;
  p.windows = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww);
  p.qk_rows = qk_rows;
  p.heads = g.nh;
  p.grid = tc ? (int)std::min<int64_t>(p.windows * g.nh, sms) : 0;
  p.buckets = bias_rows(g) * (2 * g.ww - 1);
  p.hd = g.hd;
  p.unit = tc ? g.scale : 1.f;  // the tcgen05 kernel sums dS times the scale, as its products take it
  attn_bias::grad_kernel<<<dim3((std::max(p.buckets, g.hd) + 31) / 32, g.nh + 2), 1024, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace nsw
