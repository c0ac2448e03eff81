// Window attention with a learned relative position bias, forward and backward, on mma.sync.
//
//   s_ij = scale <rms(q_i) qw, rms(k_j) kw> + table[head, bucket(i, j)] - 100 [i and j on different sides of the wrap]
//   p = softmax(s);  o = p v
//   dv = p^T do;  dp = do v^T;  ds = p (dp - <do, o>);  dq = scale ds k;  dk = scale ds^T q;  dtable[c] = sum of ds in c
//   bucket = ((t_i - t_j + T - 1) (2 wh - 1) + y_i - y_j + wh - 1) (2 ww - 1) + x_i - x_j + ww - 1
//
// A window is at most 192 tokens of one head, so its products are short: what counts is how few instructions stand around
// them, and that several windows are worked on at once on an SM.  64800 tokens of 16 heads of 64 in windows of 9 x 18, bf16:
// forward 322 us a call (134 TFLOP/s, 1.7 TB/s), with the backward 1195 (backward 126 TFLOP/s); bound by shared memory, whose
// data path is two thirds busy (a 16 x 16 block of logits takes 32 wavefronts for the fragments of K and V and 25 for its
// entries and their offsets), and by latencies at four warps a scheduler, not by products or memory.  The tcgen05
// kernels of the plain attention with the entries added to their logits took 463 and 1798.
#include <float.h>
#include <limits.h>

#include <algorithm>

#include "attn_mma.cuh"
#include "kernels.h"

namespace nsw {
namespace attn_bias {

using attn::cp_async16;
using attn::cp_async_wait_all;
using attn::fast_exp2;
using attn::kAbsorbs;
using attn::kLog2e;
using attn::ldsm_x4;
using attn::ldsm_x4_t;
using attn::mma16816;
using attn::mma16816_from;
using attn::pack2;
using attn::stsm_x4;
using attn::stsm_x4_t;

// arrays one behind the other in shared memory, each 16-byte aligned
struct Carve {
  unsigned char* base;
  size_t at;
  template <typename U>
  __host__ __device__ U* take(int n) {
    U* p = reinterpret_cast<U*>(base + at);
    at += ((size_t)n * sizeof(U) + 15) / 16 * 16;
    return p;
  }
};

// One block a head, and one for the norms' weights.  Entries are less the head's largest, so that an offset of all of them
// costs no precision, unless that is beyond 2^40: a head of the lowest value throughout, say, absorbs the logits, as it
// does in 64 bits, and its rows are even.  A finite entry stays finite.
__global__ void __launch_bounds__(256) prepare_kernel(const AnyMatrix table, const AnyMatrix qw, const AnyMatrix kw, const AttnBias b,
                                                      int heads, int hd, int n, float scale, float* __restrict__ tab) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float hi_w[8], held[1160];  // (windows of 192 tokens have at most 1155 displacements)
  const int h = blockIdx.x;
  float* out = tab + (int64_t)h * b.stride;
  if (h == heads) {
    for (int i = threadIdx.x; i < hd; i += 256) {
      out[i] = load_any(qw.p, qw.dtype, i * qw.s0);
      out[hd + i] = load_any(kw.p, kw.dtype, i * kw.s0);
    }
    return;
  }
  float hi = -INFINITY, most = 0.f;
  for (int i = threadIdx.x & 31; i < hd; i += 32)
    most = fmaxf(most, fabsf(load_any(qw.p, qw.dtype, i * qw.s0) * load_any(kw.p, kw.dtype, i * kw.s0)));
  for (int i = threadIdx.x; i < n; i += 256) {
    const float v = load_any(table.p, table.dtype, h * table.s0 + i * table.s1);
    held[i] = v;
    hi = fmaxf(hi, v);
  }
  hi = warp_max(hi);
  if ((threadIdx.x & 31) == 0) hi_w[threadIdx.x >> 5] = hi;
  __syncthreads();
  for (int w = 0; w < 8; ++w) hi = fmaxf(hi, hi_w[w]);
  const bool shifted = fabsf(hi) <= kAbsorbs;
  const float shift = shifted ? hi : 0.f;
  const auto entry = [&](float v) {
    const float e = (v - shift) * kLog2e;
    return isinf(e) && !isinf(v) ? copysignf(FLT_MAX, e) : e;
  };
  // (a margin for the roundings of q and k)
  most = warp_max(most) * fabsf(scale) * (1.01f * kLog2e * (float)hd);
  for (int i = threadIdx.x; i < b.stride; i += 256) {
    float v = 0.f;
    if (i == 0)
      v = shifted ? most : INFINITY;  // (the bound needs the largest entry to be 0)
    else if (i >= 4 && i - 4 < n)
      v = entry(held[i - 4]);
    out[i] = v;
  }
}

// Sums of columns of partial rows, in order: blockIdx.y is a head of the bias, or q's or k's norm weights.  Block c of
// `grid` walked items [n c / grid, n (c + 1) / grid) of the head-major list and left its sums for head h in row c + h; with
// no grid each (head, window) has a row.
struct Grads {
  AttnGrad bias, q, k;
  int64_t windows, qk_rows;
  int heads, grid, buckets, hd;
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
  const int64_t at = (head ? (int64_t)h * n : 0) + c;
  if (t.add) a += reinterpret_cast<const float*>(t.out)[at];
  store_any(t.out, t.dtype, at, a);
}

// ------------------------------------------------------------------------------------------------------ layout
// Tokens of a window: longitude fastest (extent nf), latitude (ns) next, time slowest.
struct Order {
  int nf, ns, nt, length, tiles;  // tiles of 16 tokens
  int entries;                    // entry of query i and key j: center + off(i) - off(j)
  int center;
  int nww, nwh;                   // windows across and down
  int sh, sw;                     // the shifts, in [0, H) and [0, W)
  int far;                        // rows of the shifted grid from here on are beyond the wrap
};
static Order order_of(const AttnGeom& g) {
  const auto wrapped = [](int v, int n) { return (v % n + n) % n; };
  Order o;
  o.nf = g.ww;
  o.ns = g.wh;
  o.nt = g.T;
  o.length = g.T * g.wh * g.ww;
  o.tiles = (o.length + 15) / 16;
  o.entries = (2 * g.T - 1) * (2 * o.ns - 1) * (2 * o.nf - 1);
  o.center = o.entries / 2;
  o.nww = g.W / g.ww;
  o.nwh = g.H / g.wh;
  o.sh = wrapped(g.sh, g.H);
  o.sw = wrapped(g.sw, g.W);
  o.far = g.mask && g.mask_shift > 0 ? g.h_global - g.mask_shift - g.row_offset : INT_MAX;
  return o;
}
// A window's corner on the shifted grid (0 <= shift < extent) and on the grid of the wrap's mask
struct Window {
  int x, y, image;  // image: b T
};
__device__ __forceinline__ Window window_of(const AttnGeom& g, const Order& o, int win) {
  const int row = win / o.nww, b = row / o.nwh;
  return {(win - row * o.nww) * g.ww, (row - b * o.nwh) * g.wh, b * g.T};
}
// the next window of the list
__device__ __forceinline__ void next_window(const AttnGeom& g, Window& w) {
  w.x += g.ww;
  if (w.x < g.W) return;
  w.x = 0;
  w.y += g.wh;
  if (w.y < g.H) return;
  w.y = 0;
  w.image = w.image + g.T == g.B * g.T ? 0 : w.image + g.T;
}
// Token i of the order: time, row and column in the window (i < 2^16; a quotient of halves is never close to a whole)
__device__ __forceinline__ int3 place_of(const Order& o, int i) {
  const int r = (int)__fdividef(i + 0.5f, (float)o.nf), f = i - r * o.nf;
  const int t = (int)__fdividef(r + 0.5f, (float)o.ns), s = r - t * o.ns;
  return make_int3(t, s, f);
}
__device__ __forceinline__ int off_of(const Order& o, const int3& p) {
  return (p.x * (2 * o.ns - 1) + p.y) * (2 * o.nf - 1) + p.z;
}
// Grid token of a window's token
__device__ __forceinline__ int token_of(const AttnGeom& g, const Order& o, const Window& w, const int3& p) {
  int y = w.y + p.y + o.sh, x = w.x + p.z + o.sw;
  if (y >= g.H) y -= g.H;
  if (x >= g.W) x -= g.W;
  return ((w.image + p.x) * g.H + y) * g.W + x;
}
// The entries of a head into shared memory; REVERSED: last entry first.  They lie in rows of 2 nf - 1.  Measured beside it on
// 64800 tokens of 16 heads, us of the forward and with the backward: rows padded so that consecutive tokens fall on consecutive
// banks 294 and 960 for 274 and 921 (windows of 9 x 9); two copies, one shifted by an entry, so that any two neighbours are an
// aligned pair, 313 and 1202 for 317 and 1173 (9 x 18).
template <bool REVERSED>
__device__ __forceinline__ void load_table(float* tab, const AttnBias& b, int entries, int head, float less) {
  const float* src = b.tab + (int64_t)head * b.stride + 4;
#pragma unroll 4
  for (int i = threadIdx.x; i < entries; i += blockDim.x)  // (no read-only load: the forward may have begun before it was written)
    tab[REVERSED ? entries - 1 - i : i] = src[i] - less;
}

__device__ __forceinline__ int2 lds_i2(uint32_t at) {
  int2 v;
  asm volatile("ld.shared.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ void lds_f2(uint32_t at, float& a, float& b) {
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(a), "=f"(b) : "r"(at));
}
__device__ __forceinline__ void lds_f(uint32_t at, float& a) {
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a) : "r"(at));
}

// The eight entries of a 16 x 16 block of logits that a lane has, in the layout of mma's results: c[j][e] for row r0 (e < 2)
// or r0 + 8 and column 8 j + 2 tq + (e & 1).  row0 / row1: addresses of the rows' entries for offset 0; off: address of the
// offsets (in bytes) of this lane's columns of the block.  A row of queries walks its entries backwards, so the forward has
// them reversed.
__device__ __forceinline__ void load_block(float (&c)[2][4], uint32_t row0, uint32_t row1, uint32_t off) {
  const int2 o[2] = {lds_i2(off), lds_i2(off + 8)};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    lds_f(row0 + o[j].x, c[j][0]);
    lds_f(row0 + o[j].y, c[j][1]);
    lds_f(row1 + o[j].x, c[j][2]);
    lds_f(row1 + o[j].y, c[j][3]);
  }
}
constexpr uint32_t kOffBytes = 16, kOffTile = 4 * kOffBytes;  // a lane's four offsets of a tile; a tile's
// the offset of token i (4 off) to where its block's lanes look for it
__device__ __forceinline__ void put_off(int* offs, int i, int off4) {
  const int tile = i >> 4, c = i & 15, j = c >> 3, tq = (c & 7) >> 1;
  offs[(tile * 4 + tq) * 4 + 2 * j + (c & 1)] = off4;
}
// The latitude-wrap mask: side is 0 or 1 of each token, s0 / s1 of the rows
__device__ __forceinline__ void mask_block(float (&c)[2][4], const float* side, float s0, float s1, int col, int tq) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 t = *reinterpret_cast<const float2*>(side + col + 8 * j + 2 * tq);
    const float d[4] = {s0 - t.x, s0 - t.y, s1 - t.x, s1 - t.y};
#pragma unroll
    for (int e = 0; e < 4; ++e) c[j][e] = fmaf(d[e] * d[e], -100.f * kLog2e, c[j][e]);
  }
}

__device__ __forceinline__ uint32_t ld32(const void* p) { return __ldg(reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// 16 raw rows in the layout of an operand's fragments (element pairs of rows r0 and r0 + 8), zeros past the window
template <typename T, int HD>
__device__ __forceinline__ void raw_rows(uint32_t (&raw)[HD / 16][4], const T* base, int64_t stride, const int* tok, int row,
                                         int length, int lane) {
  const int r0 = row + (lane >> 2), r1 = r0 + 8;
  const T* p0 = base + (int64_t)tok[r0] * stride + 2 * (lane & 3);
  const T* p1 = base + (int64_t)tok[r1] * stride + 2 * (lane & 3);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    raw[ks][0] = r0 < length ? ld32(p0 + ks * 16) : 0u;
    raw[ks][1] = r1 < length ? ld32(p1 + ks * 16) : 0u;
    raw[ks][2] = r0 < length ? ld32(p0 + ks * 16 + 8) : 0u;
    raw[ks][3] = r1 < length ? ld32(p1 + ks * 16 + 8) : 0u;
  }
}
// Lane's addresses of 16 rows in shared memory (row stride RS) as the second operand: of A B^T (the rows are B's), and of
// P V (the rows are V's)
template <typename T, int RS>
__device__ __forceinline__ uint32_t rows_nt(const T* rows, int lane) {
  return smem_u32(rows + ((lane & 7) + (lane >> 4) * 8) * RS + ((lane >> 3) & 1) * 8);
}
template <typename T, int RS>
__device__ __forceinline__ uint32_t rows_nn(const T* rows, int lane) {
  return smem_u32(rows + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8);
}
// c (+)= a 16 x 16 block of A B^T, from `from` at first
template <typename T, int HD>
__device__ __forceinline__ void block_product(float (&c)[2][4], const float (&from)[2][4], const uint32_t (&a)[HD / 16][4],
                                              uint32_t at) {
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint32_t b0, b1, b2, b3;
    ldsm_x4(at + ks * 32, b0, b1, b2, b3);
    mma16816_from<T>(c[0], ks == 0 ? from[0] : c[0], a[ks], b0, b1);
    mma16816_from<T>(c[1], ks == 0 ? from[1] : c[1], a[ks], b2, b3);
  }
}
// Two such products side by side: four chains of instructions, of which each waits for the one before it, instead of two
template <typename T, int HD>
__device__ __forceinline__ void block_products(float (&c)[2][4], const float (&from)[2][4], const uint32_t (&a)[HD / 16][4],
                                               uint32_t at, float (&c2)[2][4], const float (&from2)[2][4],
                                               const uint32_t (&a2)[HD / 16][4], uint32_t at2) {
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint32_t b[4], b2[4];
    ldsm_x4(at + ks * 32, b[0], b[1], b[2], b[3]);
    ldsm_x4(at2 + ks * 32, b2[0], b2[1], b2[2], b2[3]);
    mma16816_from<T>(c[0], ks == 0 ? from[0] : c[0], a[ks], b[0], b[1]);
    mma16816_from<T>(c[1], ks == 0 ? from[1] : c[1], a[ks], b[2], b[3]);
    mma16816_from<T>(c2[0], ks == 0 ? from2[0] : c2[0], a2[ks], b2[0], b2[1]);
    mma16816_from<T>(c2[1], ks == 0 ? from2[1] : c2[1], a2[ks], b2[2], b2[3]);
  }
}
// o += P V for 16 rows of P (one fragment) and 16 rows of V
template <typename T, int HD>
__device__ __forceinline__ void block_add(float (&o)[HD / 8][4], const uint32_t (&p)[4], uint32_t at) {
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) {
    uint32_t b0, b1, b2, b3;
    ldsm_x4_t(at + d * 32, b0, b1, b2, b3);
    mma16816<T>(o[2 * d], p, b0, b1);
    mma16816<T>(o[2 * d + 1], p, b2, b3);
  }
}
// fragments of 16 rows at `rows`
template <typename T, int HD, int RS>
__device__ __forceinline__ void load_frags(uint32_t (&a)[HD / 16][4], const T* rows, int lane) {
  const uint32_t at = smem_u32(rows + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) ldsm_x4(at + ks * 32, a[ks][0], a[ks][1], a[ks][2], a[ks][3]);
}
// results (rows r0, r0 + 8) as 16-bit rows at `rows`
template <typename T, int HD, int RS>
__device__ __forceinline__ void stage_rows(T* rows, const float (&o)[HD / 8][4], int lane) {
  const uint32_t at = smem_u32(rows + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8);
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
    stsm_x4(at + d * 32, pack2<T>(o[2 * d][0], o[2 * d][1]), pack2<T>(o[2 * d][2], o[2 * d][3]),
            pack2<T>(o[2 * d + 1][0], o[2 * d + 1][1]), pack2<T>(o[2 * d + 1][2], o[2 * d + 1][3]));
}
// 16 staged rows to their tokens, 16 bytes a lane
template <typename T, int HD, int RS>
__device__ __forceinline__ void store_rows(const T* rows, T* dst, int64_t stride, const int* tok, int row, int length,
                                           int lane) {
  constexpr int CH = HD / 8;
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) {
    const int r = (lane + 32 * i) / CH, c = (lane + 32 * i) % CH;
    if (row + r < length)
      *reinterpret_cast<uint4*>(dst + (int64_t)tok[row + r] * stride + 8 * c) =
          *reinterpret_cast<const uint4*>(rows + r * RS + 8 * c);
  }
}

// two fp32 numbers in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 c, a, b;\n"
      " mov.b64 {%0, %1}, c;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 c, a, b, c;\n mov.b64 {%0, %1}, c;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  float f[2];
  unpack2(w, f, T());
  return make_float2(f[0], f[1]);
}
// RMSNorm of one row by HD / 8 lanes, eight elements each: x * rs * w (w in shared memory); rs of the row
template <typename T, int HD>
__device__ __forceinline__ float norm_chunk(const uint4& raw, const float* w, uint4& out) {
  const float2 f[4] = {unpack_pair<T>(raw.x), unpack_pair<T>(raw.y), unpack_pair<T>(raw.z), unpack_pair<T>(raw.w)};
  const float4 w0 = *reinterpret_cast<const float4*>(w), w1 = *reinterpret_cast<const float4*>(w + 4);
  const float2 we[4] = {{w0.x, w0.y}, {w0.z, w0.w}, {w1.x, w1.y}, {w1.z, w1.w}};
  float2 s2 = mul2(f[0], f[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s2 = fma2(f[i], f[i], s2);
  float ss = s2.x + s2.y;
#pragma unroll
  for (int o = 1; o < HD / 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float rs = rsqrtf(ss * (1.f / HD) + FLT_EPSILON);
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = mul2(mul2(f[i], we[i]), make_float2(rs, rs));
    y[i] = pack2<T>(v.x, v.y);
  }
  out = make_uint4(y[0], y[1], y[2], y[3]);
  return rs;
}

// The exponentials are taken less a bound on the window's logits, less `top`: with the largest entry 0, no logit is above
// head_dim max_i |qw_i kw_i| scale (Cauchy and Schwarz, in the norm that the weights' products give), which the preparation
// has left in the head's header.  So they are at most 2^top, the bound is in the entries before the products begin, and
// nothing is looked up or subtracted for a row.  Rows far below the bound lose precision to their type's smallest numbers:
// those whose sum is below `least` (in fp16, 192 numbers that are each off by at most 2^-25 are off by less than 2^-17 of
// it) make their tile begin again with every row less its own largest logit, for one more product of q and k.  In bf16 the
// weights meet V in fp32's range: a tile also begins again where a sum of P V is not finite (|V| above 2^(120 - top) at
// weights of 2^top), and where a row's weights add up to less than one and one of its sums is below 2^-100, where what
// 192 products lost below 2^-126 might show.  The second way's weights are at most 2^-drop, so that 192 of them times
// any value of the type stay below fp32's largest number.
// top: a product is no further below zero than the bound is above it, so twice the bound, and 24 for a row's entries below
// the head's largest, leave few tiles to do again; 110 at most, where such weights still meet V of some hundreds.  From
// there rows may be 154 below the bound, 1.44 head_dim^1/2 times the largest product of two norm weights (16 heads of 64: up
// to weights of 3 or so a call takes the first way, 323 us, the second 573).
template <typename T>
struct Bound;
template <>
struct Bound<__nv_bfloat16> {
  static constexpr float least = 5.6843419e-14f, drop = 8.f;  // 2^-44
  static __device__ __forceinline__ float top(float bound) { return fminf(2.f * bound + 24.f, 110.f); }
};
template <>
struct Bound<__half> {
  static constexpr float least = 1.f, drop = 0.f;  // (65504 2^14 192 is far from fp32's limit)
  static __device__ __forceinline__ float top(float) { return 14.f; }
};
constexpr float kMostBound = 1e4f;  // beyond it (or NaN): the second way at once

// ----------------------------------------------------------------------------------------------------- forward
// A block takes a window and head, a warp 16 queries at a time.  K is normalised into shared memory, V copied there; the
// queries' fragments come straight from global memory and are normalised in registers, with scale and log2 e, so that
// the first product, which begins with the entries less the bound, ends in the exponents themselves.  P goes from
// registers into the second product.  Nothing waits for a row's maximum, and several blocks share an SM, so that one's
// loads and norms run beside the others' products.
constexpr int kFwdWarps = 6;
template <typename T, int HD>
struct FwdSmem {
  float *tab, *qw, *kw;
  T *k, *v, *stage;
  int *tok, *off4, *offs;
  float* side;
  __host__ __device__ size_t carve(unsigned char* base, const Order& o) {
    const int rows = o.tiles * 16, RS = HD + 8;
    Carve c{base, 0};
    k = c.take<T>(rows * RS);
    v = c.take<T>(rows * RS);
    stage = c.take<T>(16 * kFwdWarps * RS);
    tok = c.take<int>(rows);
    off4 = c.take<int>(rows);
    offs = c.take<int>(rows);
    qw = c.take<float>(HD);  // with scale and log2 e
    kw = c.take<float>(HD);
    side = c.take<float>(rows);
    tab = c.take<float>(o.entries);
    return c.at;
  }
};
template <typename T, int HD>
__global__ void __launch_bounds__(32 * kFwdWarps, HD <= 64 ? 3 : 2)
    fwd_kernel(const T* __restrict__ qkv, const AttnBias bias, const float* norms, T* __restrict__ out,
               float2* __restrict__ lse, const __grid_constant__ AttnGeom g, const __grid_constant__ Order o) {
  constexpr int RS = HD + 8, KS = HD / 16, CH = HD / 8;
  constexpr uint32_t kTile = 16 * RS * sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  const int L = o.length, rows = o.tiles * 16, nthreads = blockDim.x, nw = nthreads / 32;
  FwdSmem<T, HD> S;
  S.carve(smem, o);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int win = blockIdx.x / g.nh, head = blockIdx.x - win * g.nh;
  const int64_t C = (int64_t)g.nh * HD;
  const T* base = qkv + (int64_t)head * HD;

  asm volatile("griddepcontrol.wait;" ::: "memory");  // (for the table and the norms' weights)
  const float bound = bias.tab[(int64_t)head * bias.stride];
  const bool exact = !(bound <= kMostBound);
  const float less = exact ? 0.f : bound - Bound<T>::top(bound);  // in the entries
  const Window window = window_of(g, o, win);
  const bool mixed = window.y < o.far && window.y + g.wh > o.far;
  for (int i = threadIdx.x; i < rows; i += nthreads) {
    const int3 p = place_of(o, i);
    const int off4 = i < L ? 4 * off_of(o, p) : 0;
    S.tok[i] = i < L ? token_of(g, o, window, p) : 0;
    S.off4[i] = off4;
    put_off(S.offs, i, off4);
    S.side[i] = window.y + p.y >= o.far ? 1.f : 0.f;
  }
  for (int i = threadIdx.x; i < HD; i += nthreads) {
    S.qw[i] = norms[i] * (g.scale * kLog2e);
    S.kw[i] = norms[HD + i];
  }
  __syncthreads();
  uint32_t raw[KS][4];
  const int first = blockIdx.y * nw + warp;
  if (first < o.tiles)  // the first tile's raw queries, on their way under what follows
    raw_rows<T, HD>(raw, base, g.qkv_stride, S.tok, first * 16, L, lane);
  for (int i = threadIdx.x; i < rows * CH; i += nthreads) {
    const int r = i / CH, c = i % CH;
    T* dst = S.v + r * RS + 8 * c;
    if (r < L)
      cp_async16(dst, base + (int64_t)S.tok[r] * g.qkv_stride + 2 * C + 8 * c);
    else
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
  }
  // keys: the lanes of a row are neighbours, and a warp's rows are whole (32 is a multiple of CH)
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < rows * CH; i0 += kAhead * nthreads) {
    uint4 x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * nthreads + threadIdx.x, r = i / CH;
      x[u] = i < rows * CH && r < L
                 ? __ldg(reinterpret_cast<const uint4*>(base + (int64_t)S.tok[r] * g.qkv_stride + C + 8 * (i % CH)))
                 : make_uint4(0, 0, 0, 0);
    }
    if (i0 == 0) load_table<true>(S.tab, bias, o.entries, head, less);  // (while the first keys arrive)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * nthreads + threadIdx.x;
      if (i0 + u * nthreads >= rows * CH) break;
      uint4 y;
      norm_chunk<T, HD>(x[u], S.kw + 8 * (i % CH), y);
      if (i < rows * CH) *reinterpret_cast<uint4*>(S.k + (i / CH) * RS + 8 * (i % CH)) = y;
    }
  }
  cp_async_wait_all();
  __syncthreads();

  const uint32_t k_at = rows_nt<T, RS>(S.k, lane), v_at = rows_nn<T, RS>(S.v, lane);
  const uint32_t off_at = smem_u32(S.offs) + tq * kOffBytes;
  const int whole = mixed ? 0 : L / 16;  // tiles of keys without a mask
  for (int qt = first; qt < o.tiles; qt += nw * gridDim.y) {
    if (qt != first) raw_rows<T, HD>(raw, base, g.qkv_stride, S.tok, qt * 16, L, lane);
    const int r0 = qt * 16 + gq, r1 = r0 + 8;
    uint32_t qa[KS][4];
    {
      float2 x[KS][4], s0 = {0.f, 0.f}, s1 = {0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[ks][e] = unpack_pair<T>(raw[ks][e]);
          float2& s = e & 1 ? s1 : s0;
          s = fma2(x[ks][e], x[ks][e], s);
        }
      const float rs0 = rsqrtf(quad_sum(s0.x + s0.y) * (1.f / HD) + FLT_EPSILON);
      const float rs1 = rsqrtf(quad_sum(s1.x + s1.y) * (1.f / HD) + FLT_EPSILON);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 w = *reinterpret_cast<const float2*>(S.qw + ks * 16 + (e >> 1) * 8 + 2 * tq);
          const float rs = e & 1 ? rs1 : rs0;
          const float2 v = mul2(mul2(x[ks][e], w), make_float2(rs, rs));
          qa[ks][e] = pack2<T>(v.x, v.y);
        }
    }
    const int last = o.entries - 1 - o.center;
    const uint32_t row0 = smem_u32(S.tab + last - (S.off4[r0] >> 2));
    const uint32_t row1 = smem_u32(S.tab + last - (S.off4[r1] >> 2));
    // f(logits less m0 / m1 of their rows, key tile) for all key tiles; late: subtracted after the product
    const auto each_tile = [&](float m0, float m1, bool late, auto shifted, auto f) {
      const auto subtract = [&](float (&c)[2][4]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          c[j][0] -= m0;
          c[j][1] -= m0;
          c[j][2] -= m1;
          c[j][3] -= m1;
        }
      };
      const auto before = [&](float (&c)[2][4], int kb, auto masked) {
        load_block(c, row0, row1, off_at + kb * kOffTile);
        if (masked()) {
          if (mixed) mask_block(c, S.side, S.side[r0], S.side[r1], kb * 16, tq);
          if (kb * 16 + 16 > L) {  // padding keys
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (kb * 16 + 8 * j + 2 * tq + (e & 1) >= L) c[j][e] = -INFINITY;
          }
        }
        if (shifted() && !late) subtract(c);
      };
      int kb = 0;
#pragma unroll 1
      for (; kb + 1 < whole; kb += 2) {
        float c[2][4], d[2][4];
        before(c, kb, std::false_type());
        before(d, kb + 1, std::false_type());
        block_products<T, HD>(c, c, qa, k_at + kb * kTile, d, d, qa, k_at + (kb + 1) * kTile);
        if (shifted() && late) subtract(c), subtract(d);
        f(c, kb);
        f(d, kb + 1);
      }
#pragma unroll 1
      for (; kb < o.tiles; ++kb) {
        float c[2][4];
        before(c, kb, std::true_type());
        block_product<T, HD>(c, c, qa, k_at + kb * kTile);
        if (shifted() && late) subtract(c);
        f(c, kb);
      }
    };
    // the rows' sums are those of the rounded values that are multiplied, by one more product (with ones): so a row's
    // weights add up to one as they are, and the sum costs an instruction where eight additions would
    float acc[CH][4], sum[4];
    const uint32_t ones = pack2<T>(1.f, 1.f);
    const auto weights = [&](float (&c)[2][4], int kb, float drop) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[j][e] = fast_exp2(drop == 0.f ? c[j][e] : c[j][e] - drop);
      const uint32_t p[4] = {pack2<T>(c[0][0], c[0][1]), pack2<T>(c[0][2], c[0][3]), pack2<T>(c[1][0], c[1][1]),
                             pack2<T>(c[1][2], c[1][3])};
      mma16816<T>(sum, p, ones, ones);
      block_add<T, HD>(acc, p, v_at + kb * kTile);
    };
    const auto clear = [&]() {
      sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll
      for (int d = 0; d < CH; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.f;
    };
    float m0 = 0.f, m1 = 0.f, drop = 0.f;  // besides `less`
    bool again = exact;
    if (!exact) {
      clear();
      each_tile(0.f, 0.f, false, std::false_type(), [&](float (&c)[2][4], int kb) { weights(c, kb, 0.f); });
      bool redo = sum[0] < Bound<T>::least || sum[2] < Bound<T>::least;
      if constexpr (Bound<T>::drop > 0.f) {  // zero times what is not finite is not zero
        float2 finite = {0.f, 0.f};
#pragma unroll
        for (int d = 0; d < CH; ++d) {
          finite = fma2(make_float2(acc[d][0], acc[d][1]), make_float2(0.f, 0.f), finite);
          finite = fma2(make_float2(acc[d][2], acc[d][3]), make_float2(0.f, 0.f), finite);
        }
        redo = redo || !(finite.x + finite.y == 0.f);
        if (__any_sync(0xffffffffu, sum[0] < 1.f || sum[2] < 1.f)) {
          float s0 = INFINITY, s1 = INFINITY;
#pragma unroll
          for (int d = 0; d < CH; ++d) {
            s0 = fminf(s0, fminf(fabsf(acc[d][0]), fabsf(acc[d][1])));
            s1 = fminf(s1, fminf(fabsf(acc[d][2]), fabsf(acc[d][3])));
          }
          redo = redo || (sum[0] < 1.f && s0 < 7.8886091e-31f) || (sum[2] < 1.f && s1 < 7.8886091e-31f);  // 2^-100
        }
      }
      again = __any_sync(0xffffffffu, redo);
    }
    if (again) {
      m0 = m1 = -INFINITY;
      each_tile(0.f, 0.f, false, std::false_type(), [&](float (&c)[2][4], int) {
        m0 = fmaxf(m0, fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1])));
        m1 = fmaxf(m1, fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3])));
      });
      m0 = quad_max(m0);
      m1 = quad_max(m1);
      if (m0 == -INFINITY) m0 = 0.f;  // a row that the bias masks throughout: P = 0
      if (m1 == -INFINITY) m1 = 0.f;
      // rows of entries beyond kAbsorbs throughout absorb the product before they are subtracted
      const bool late = __any_sync(0xffffffffu, fabsf(m0) > kAbsorbs || fabsf(m1) > kAbsorbs);
      clear();
      drop = Bound<T>::drop;  // (apart from m0 and m1, which may be too large to hold it)
      each_tile(m0, m1, late, std::true_type(), [&](float (&c)[2][4], int kb) { weights(c, kb, Bound<T>::drop); });
    }
    const float l0 = sum[0], l1 = sum[2];
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
#pragma unroll
    for (int d = 0; d < CH; ++d) {
      acc[d][0] *= i0;
      acc[d][1] *= i0;
      acc[d][2] *= i1;
      acc[d][3] *= i1;
    }
    if (tq == 0) {
      float2* at = lse + (int64_t)blockIdx.x * L;
      if (r0 < L) at[r0] = l0 == 0.f ? make_float2(0.f, 0.f) : make_float2(m0 + less, __log2f(l0) + drop);
      if (r1 < L) at[r1] = l1 == 0.f ? make_float2(0.f, 0.f) : make_float2(m1 + less, __log2f(l1) + drop);
    }
    T* st = S.stage + warp * 16 * RS;
    __syncwarp();
    stage_rows<T, HD, RS>(st, acc, lane);
    __syncwarp();
    store_rows<T, HD, RS>(st, out + (int64_t)head * HD, g.out_stride, S.tok, qt * 16, L, lane);
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// Blocks walk the (head, window) list in contiguous pieces, a warp for each 16 tokens of a window.  For an item:
//   norms   the raw rows of q and k, copied to shared memory while the item before was worked on, become what the
//           forward took; D_i = <dO_i, O_i>
//   A       a warp's 16 keys against all queries: S^T begins with the entries less the row's logarithm of the sum, dP^T
//           with -D, so that P^T is an exponential and dS^T a product away; dV and dK stay in registers; dS goes to shared
//           memory in T (as the products take it; the bias's sums take it too, each term off by at most half a step of no
//           sign: an fp32 copy, 103 KB at 162 tokens, does not fit), queries down
//   B       a warp's 16 queries: dQ = dS K.  The next item's rows are on their way.
// The bias's gradient sums dS over the windows of a head, without atomics and in a fixed order: of the two extents of the
// window, one, a, is summed at once and the other, b, kept as a pair, acc[dt][da][b_i][b_j], whose entries belong to
// threads; the diagonals b_i - b_j are summed when the head is done, into the block's row for it.
// The norms' backward takes the raw rows from global memory (L2) again, in the fragments' layout.
struct BiasSums {
  bool a_is_s;         // a: the slow extent
  int na, nb, sa, sb;  // extents and strides in tokens
  int entries;         // in all
  int places;          // (b_i, b_j) of one (dt, da)
};
__host__ __device__ __forceinline__ BiasSums sums_of(const Order& o) {
  BiasSums b;
  b.a_is_s = (2 * o.ns - 1) * o.nf * o.nf <= (2 * o.nf - 1) * o.ns * o.ns;
  b.na = b.a_is_s ? o.ns : o.nf;
  b.nb = b.a_is_s ? o.nf : o.ns;
  b.sa = b.a_is_s ? o.nf : 1;
  b.sb = b.a_is_s ? 1 : o.nf;
  b.entries = (2 * o.nt - 1) * (2 * b.na - 1) * b.nb * b.nb;
  b.places = b.nb * b.nb;
  return b;
}

template <typename T, int HD>
struct BwdSmem {
  float *tab, *acc, *sub, *late, *ll, *negD, *rq, *rk, *qw, *qn, *kw, *kn;
  T *q, *v, *g, *k, *s;
  int *tok, *off4, *offs;
  float* side;
  // entries: of the bias's sums; k_bufs: buffers for k (two, where there is room: the next item's keys arrive while this
  // one's are read)
  __host__ __device__ size_t carve(unsigned char* base, const Order& o, int entries, int k_bufs) {
    const int rows = o.tiles * 16, RS = HD + 8;
    Carve c{base, 0};
    acc = c.take<float>(entries);
    q = c.take<T>(rows * RS * (3 + k_bufs));
    v = q + rows * RS;
    g = v + rows * RS;  // dO
    k = g + rows * RS;
    s = c.take<T>(rows * (rows + 8));  // dS, [query][key]
    tok = c.take<int>(2 * rows);
    off4 = c.take<int>(rows);
    offs = c.take<int>(rows);
    sub = c.take<float>(rows);   // what the exponents are less: of each query
    late = c.take<float>(rows);  // wide rows: and after the product, first this, then this
    ll = c.take<float>(rows);
    negD = c.take<float>(rows);
    rq = c.take<float>(rows);
    rk = c.take<float>(rows);
    qw = c.take<float>(HD);  // with scale and log2 e
    qn = c.take<float>(HD);  // with scale
    kw = c.take<float>(HD);
    kn = c.take<float>(HD);  // with ln 2
    side = c.take<float>(2 * rows);
    tab = c.take<float>(o.entries);
    return c.at;
  }
};

// rows past the window become zeros (their places in shared memory hold zeros for good)
template <typename T, int HD, int RS>
__device__ __forceinline__ void stage_live(T* rows, float (&o)[HD / 8][4], int row, int length, int lane) {
  if (row + 16 > length) {
    const bool live0 = row + (lane >> 2) < length, live1 = row + (lane >> 2) + 8 < length;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      if (!live0) o[d][0] = o[d][1] = 0.f;
      if (!live1) o[d][2] = o[d][3] = 0.f;
    }
  }
  stage_rows<T, HD, RS>(rows, o, lane);
}
// A tile's gradient g (times `scale`, which w holds too) of y = x rs w becomes that of x, dx = rs w g - x rs^3 mean(w g x);
// sums gets the tile's columns of g x rs: two of them a lane, after a butterfly over the rows that halves what a lane holds.
template <typename T, int HD>
__device__ __forceinline__ void norm_backward(float (&g)[HD / 8][4], const uint32_t (&raw)[HD / 16][4], const float* w,
                                              float scale, float rs0, float rs1, float (&sums)[2], int lane) {
  constexpr int CH = HD / 8;
  const int tq = lane & 3;
  float dot0 = 0.f, dot1 = 0.f, c[2 * CH];
#pragma unroll
  for (int d = 0; d < CH; ++d) {
    float x0[2], x1[2];
    unpack2(raw[d >> 1][(d & 1) * 2], x0, T());
    unpack2(raw[d >> 1][(d & 1) * 2 + 1], x1, T());
    const float2 wd = *reinterpret_cast<const float2*>(w + 8 * d + 2 * tq);
    const float we[2] = {wd.x, wd.y};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      c[2 * d + e] = fmaf(g[d][e] * x0[e], rs0, g[d][2 + e] * x1[e] * rs1);
      g[d][e] *= we[e];
      g[d][2 + e] *= we[e];
      dot0 = fmaf(g[d][e], x0[e], dot0);
      dot1 = fmaf(g[d][2 + e], x1[e], dot1);
    }
  }
  const float k0 = rs0 * rs0 * rs0 * quad_sum(dot0) * (1.f / HD), k1 = rs1 * rs1 * rs1 * quad_sum(dot1) * (1.f / HD);
#pragma unroll
  for (int d = 0; d < CH; ++d) {
    float x0[2], x1[2];
    unpack2(raw[d >> 1][(d & 1) * 2], x0, T());
    unpack2(raw[d >> 1][(d & 1) * 2 + 1], x1, T());
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      g[d][e] = fmaf(g[d][e], rs0, -x0[e] * k0);
      g[d][2 + e] = fmaf(g[d][2 + e], rs1, -x1[e] * k1);
    }
  }
#pragma unroll
  for (int o = 16, n = 2 * CH; o >= 4; o >>= 1) {
    const bool up = lane & o;
    if (n > 2) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (i < n) {
          const float send = up ? c[i] : c[i + n];
          c[i] = (up ? c[i + n] : c[i]) + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      c[0] += __shfl_xor_sync(0xffffffffu, c[0], o);
      c[1] += __shfl_xor_sync(0xffffffffu, c[1], o);
    }
  }
  sums[0] = fmaf(c[0], scale, sums[0]);
  sums[1] = fmaf(c[1], scale, sums[1]);
}
// the columns that norm_backward left with this lane (where lanes hold the same ones, they are equal)
template <int HD>
__device__ __forceinline__ void put_cols(float* dst, const float (&sums)[2], int lane) {
  const int d = HD == 64 ? (lane >> 4) * 4 + ((lane >> 3) & 1) * 2 + ((lane >> 2) & 1)
                : HD == 32 ? (lane >> 4) * 2 + ((lane >> 3) & 1) : lane >> 4;
  dst[8 * d + 2 * (lane & 3)] = sums[0];
  dst[8 * d + 2 * (lane & 3) + 1] = sums[1];
}

constexpr int kBwdWarps = 12;  // 192 tokens
template <typename T, int HD>
__global__ void __launch_bounds__(32 * kBwdWarps, 1)
    bwd_kernel(const T* __restrict__ qkv, const AttnBias bias, const float* __restrict__ norms, const T* __restrict__ out,
               const T* __restrict__ dout, const float2* __restrict__ lse, T* __restrict__ dqkv,
               float* __restrict__ dqw_part, float* __restrict__ dkw_part, float* __restrict__ dbias_part, int k_bufs,
               const __grid_constant__ AttnGeom g, const __grid_constant__ Order o) {
  constexpr int RS = HD + 8, KS = HD / 16, CH = HD / 8;
  constexpr uint32_t kTile = 16 * RS * sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  const BiasSums bs = sums_of(o);
  const int L = o.length, rows = o.tiles * 16, DS = rows + 8, nthreads = blockDim.x;
  const int buckets = (2 * g.T - 1) * (2 * g.wh - 1) * (2 * g.ww - 1);
  BwdSmem<T, HD> S;
  S.carve(smem, o, dbias_part ? bs.entries : 0, k_bufs);
  float *tab = S.tab, *acc = S.acc, *sub = S.sub, *late = S.late, *ll = S.ll, *negD = S.negD, *rq = S.rq, *rk = S.rk, *qw = S.qw,
        *qn = S.qn, *kw = S.kw, *kn = S.kn;
  T *sQ = S.q, *sV = S.v, *sG = S.g, *sK0 = S.k, *sS = S.s;
  int *tok2 = S.tok, *off4 = S.off4;
  float* side2 = S.side;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int64_t C = (int64_t)g.nh * HD;
  const int64_t n_win = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww), n_items = n_win * g.nh;
  const int64_t i_begin = n_items * blockIdx.x / gridDim.x, i_end = n_items * (blockIdx.x + 1) / gridDim.x;

  const int3 place = place_of(o, min((int)threadIdx.x, L - 1));  // of this thread's token
  if (threadIdx.x < rows) {
    off4[threadIdx.x] = threadIdx.x < L ? 4 * off_of(o, place) : 0;
    put_off(S.offs, threadIdx.x, threadIdx.x < L ? 4 * off_of(o, place) : 0);
  }
  for (int i = threadIdx.x; i < HD; i += nthreads) {
    qw[i] = norms[i] * (g.scale * kLog2e);
    qn[i] = norms[i] * g.scale;
    kw[i] = norms[HD + i];
    kn[i] = norms[HD + i] * 0.69314718055994530942f;
  }
  // padding rows stay zero: copies and staged rows write the window's rows alone
  for (int i = threadIdx.x; i < (rows - L) * CH * (3 + k_bufs); i += nthreads) {
    const int b = i / ((rows - L) * CH), r = i % ((rows - L) * CH);
    *reinterpret_cast<uint4*>(sQ + (b * rows + L + r / CH) * RS + 8 * (r % CH)) = make_uint4(0, 0, 0, 0);
  }
  if (dbias_part)
    for (int i = threadIdx.x; i < bs.entries; i += nthreads) acc[i] = 0.f;
  // this thread's part of the bias's sums (groups of threads, if there are several for all places)
  const int groups = max(1, nthreads / bs.places);
  const int my_group = groups > 1 ? threadIdx.x / bs.places : 0;
  const int my_place = my_group >= groups ? bs.places : threadIdx.x - my_group * bs.places;

  // a window's tokens and sides into table `buf`
  const auto build = [&](const Window& w, int buf) {
    if (threadIdx.x >= rows) return;
    const int at = buf * rows + threadIdx.x;
    const bool live = threadIdx.x < L;
    tok2[at] = live ? token_of(g, o, w, place) : 0;
    side2[at] = w.y + place.y >= o.far ? 1.f : 0.f;
  };
  // an item's rows into shared memory: k's (where given a place), and the others'
  const auto copy = [&](int head, const int* tok, T* k, bool others) {
    const T* src = qkv + (int64_t)head * HD;
    const T* src_g = dout + (int64_t)head * HD;
    for (int i = threadIdx.x; i < L * CH; i += nthreads) {
      const int r = i / CH, c = i % CH, at = r * RS + 8 * c;
      const int64_t t = tok[r];
      const T* p = src + t * g.qkv_stride + 8 * c;
      if (k) cp_async16(k + at, p + C);
      if (others) {
        cp_async16(sQ + at, p);
        cp_async16(sV + at, p + 2 * C);
        cp_async16(sG + at, src_g + t * g.out_stride + 8 * c);
      }
    }
  };
  const auto flush = [&](int head) {  // the head's sums into the block's row for it; between barriers
    float* dst = dbias_part + ((int64_t)blockIdx.x + head) * buckets;
    const int ny = 2 * g.wh - 1, nx = 2 * g.ww - 1;
    for (int c = threadIdx.x; c < buckets; c += nthreads) {
      const int dt = c / (ny * nx), dy = c / nx - dt * ny, dx = c % nx;
      const int da = bs.a_is_s ? dy : dx, db = (bs.a_is_s ? dx : dy) - (bs.nb - 1);
      const float* a = acc + (dt * (2 * bs.na - 1) + da) * bs.nb * bs.nb + max(db, 0) * bs.nb + max(-db, 0);
      float s = 0.f;
      for (int i = 0; i < bs.nb - abs(db); ++i) s += a[i * (bs.nb + 1)];
      dst[c] = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bs.entries; i += nthreads) acc[i] = 0.f;
  };

  int cur = 0, tab_head = -1;
  int head = (int)(i_begin / n_win);
  int64_t win = i_begin - head * n_win;  // of its head's
  Window window = window_of(g, o, (int)win);
  if (i_begin < i_end) {
    build(window, 0);
    __syncthreads();
    copy(head, tok2, sK0, true);
  }
  float wq[2] = {0.f, 0.f}, wk[2] = {0.f, 0.f};  // this lane's columns of the norms' weights' gradients

  for (int64_t item = i_begin; item < i_end; ++item) {
    const int* tok = tok2 + cur * rows;
    const float* side = side2 + cur * rows;
    T* sK = sK0 + (k_bufs > 1 ? cur * rows * RS : 0);
    const T* base = qkv + (int64_t)head * HD;
    const bool next = item + 1 < i_end;
    // O's rows (for D) and the rows' statistics are on their way while the copies land
    constexpr int kOut = CH / 2;  // of a thread: the block has two for each token
    uint4 o_raw[kOut];
#pragma unroll
    for (int u = 0; u < kOut; ++u) {
      const int i = u * nthreads + threadIdx.x;
      o_raw[u] = i < L * CH ? __ldg(reinterpret_cast<const uint4*>(out + (int64_t)tok[i / CH] * g.out_stride +
                                                                  (int64_t)head * HD + 8 * (i % CH)))
                            : make_uint4(0, 0, 0, 0);
    }
    float2 st = make_float2(INFINITY, 0.f);
    if (threadIdx.x < L) st = lse[(win * g.nh + head) * L + threadIdx.x];
    const bool mixed = window.y < o.far && window.y + g.wh > o.far;
    // the item after
    int head_n = head;
    Window window_n = window;
    int64_t win_n = win + 1;
    next_window(g, window_n);
    if (win_n == n_win) {
      win_n = 0;
      ++head_n;
    }
    __syncthreads();  // the item before has been worked through
    if (head != tab_head) {
      if (tab_head >= 0 && dbias_part) flush(tab_head);
      load_table<false>(tab, bias, o.entries, head, 0.f);
      tab_head = head;
    }
    cp_async_wait_all();
    __syncthreads();
    // ---- norms in place, and D
    constexpr int kChunks = CH < 4 ? CH : 4;  // of a thread at once; it has CH (rows of q, then of k, two threads a token)
#pragma unroll 1
    for (int u0 = 0; u0 < CH; u0 += kChunks) {
      uint4 x[kChunks];
      T* at[kChunks];
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        const int i = (u0 + u) * nthreads + threadIdx.x;
        const bool isk = i >= rows * CH;
        const int j = isk ? i - rows * CH : i;
        at[u] = (isk ? sK : sQ) + (j / CH) * RS + 8 * (j % CH);
        x[u] = *reinterpret_cast<const uint4*>(at[u]);
      }
#pragma unroll
      for (int u = 0; u < kChunks; ++u) {
        const int i = (u0 + u) * nthreads + threadIdx.x;
        const bool isk = i >= rows * CH;
        const int j = isk ? i - rows * CH : i;
        uint4 y;
        const float rs = norm_chunk<T, HD>(x[u], (isk ? kw : qw) + 8 * (j % CH), y);
        *reinterpret_cast<uint4*>(at[u]) = y;
        if (j % CH == 0) (isk ? rk : rq)[j / CH] = rs;
      }
    }
#pragma unroll
    for (int u = 0; u < kOut; ++u) {
      const int i = u * nthreads + threadIdx.x;
      float a[8], b[8], d = 0.f;
      if (i < L * CH) {
        unpack8<T>(o_raw[u], a);
        unpack8<T>(*reinterpret_cast<const uint4*>(sG + (i / CH) * RS + 8 * (i % CH)), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(a[e], b[e], d);
      }
#pragma unroll
      for (int s = 1; s < CH; s <<= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
      if (i < L * CH && i % CH == 0) negD[i / CH] = -d;
    }
    // (largest logit, log2 of the sum): one number, unless the first is so large that the second would be lost beside it
    const int wide = __syncthreads_or(threadIdx.x < L && fabsf(st.x) > 4096.f);
    if (threadIdx.x < rows) {
      const bool absorbs = threadIdx.x < L && fabsf(st.x) > kAbsorbs;  // as the forward
      sub[threadIdx.x] = !wide ? st.x + st.y : absorbs ? 0.f : st.x;
      late[threadIdx.x] = absorbs ? st.x : 0.f;
      ll[threadIdx.x] = st.y;
      if (threadIdx.x >= L) negD[threadIdx.x] = 0.f;
    }
    if (next) build(window_n, 1 - cur);
    __syncthreads();

    // ---- A
    {
      const int k0 = warp * 16 + gq;
      uint32_t kf[KS][4], vf[KS][4];
      load_frags<T, HD, RS>(kf, sK + warp * 16 * RS, lane);
      load_frags<T, HD, RS>(vf, sV + warp * 16 * RS, lane);
      float dv[CH][4], dk[CH][4];
#pragma unroll
      for (int d = 0; d < CH; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) dv[d][e] = dk[d][e] = 0.f;
      const uint32_t row0 = smem_u32(tab + o.center - (off4[k0] >> 2));
      const uint32_t row1 = smem_u32(tab + o.center - (off4[k0 + 8] >> 2));
      const uint32_t off_at = smem_u32(S.offs) + tq * kOffBytes;
      const uint32_t q_nt = rows_nt<T, RS>(sQ, lane), q_nn = rows_nn<T, RS>(sQ, lane);
      const uint32_t g_nt = rows_nt<T, RS>(sG, lane), g_nn = rows_nn<T, RS>(sG, lane);
      const uint32_t sub_at = smem_u32(sub + 2 * tq), d_at = smem_u32(negD + 2 * tq);
      const uint32_t ds_at = smem_u32(sS + ((lane & 7) + (lane >> 4) * 8) * DS + warp * 16 + ((lane >> 3) & 1) * 8);
      const uint32_t ds_tile = 16 * DS * sizeof(T);
      const auto tile = [&](int qb, auto masked) {
        float s[2][4], dp[2][4], nd[2][4];
        load_block(s, row0, row1, off_at + qb * kOffTile);
        if (masked() && mixed) mask_block(s, side, side[k0], side[k0 + 8], qb * 16, tq);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx, my;
          lds_f2(sub_at + qb * 64 + j * 32, mx, my);
          lds_f2(d_at + qb * 64 + j * 32, nd[j][0], nd[j][1]);
          nd[j][2] = nd[j][0];
          nd[j][3] = nd[j][1];
          s[j][0] -= mx;
          s[j][1] -= my;
          s[j][2] -= mx;
          s[j][3] -= my;
        }
        block_products<T, HD>(s, s, kf, q_nt + qb * kTile, dp, nd, vf, g_nt + qb * kTile);
        if (masked() && wide) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 m = *reinterpret_cast<const float2*>(late + qb * 16 + 8 * j + 2 * tq);
            const float2 l = *reinterpret_cast<const float2*>(ll + qb * 16 + 8 * j + 2 * tq);
            s[j][0] = (s[j][0] - m.x) - l.x;
            s[j][1] = (s[j][1] - m.y) - l.y;
            s[j][2] = (s[j][2] - m.x) - l.x;
            s[j][3] = (s[j][3] - m.y) - l.y;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[j][e] = fast_exp2(s[j][e]);
            if (masked() && k0 + 8 * (e >> 1) >= L) s[j][e] = 0.f;  // padding keys
          }
        const uint32_t p[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                               pack2<T>(s[1][2], s[1][3])};
        uint32_t ds[4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 v = mul2(make_float2(s[j][2 * e], s[j][2 * e + 1]), make_float2(dp[j][2 * e], dp[j][2 * e + 1]));
            ds[2 * j + e] = pack2<T>(v.x, v.y);
          }
        // ds: (keys, queries) = (0, 0), (8, 0), (0, 8), (8, 8) -> rows of queries
        stsm_x4_t(ds_at + qb * ds_tile, ds[0], ds[1], ds[2], ds[3]);
        block_add<T, HD>(dv, p, g_nn + qb * kTile);
        block_add<T, HD>(dk, ds, q_nn + qb * kTile);
      };
      if (mixed || warp * 16 + 16 > L || wide) {
#pragma unroll 1
        for (int qb = 0; qb < o.tiles; ++qb) tile(qb, std::true_type());
      } else {
#pragma unroll 1
        for (int qb = 0; qb < o.tiles; ++qb) tile(qb, std::false_type());
      }
      // dV, then dK through the norm, by way of this warp's rows of sV
      T* st_rows = sV + warp * 16 * RS;
      T* dst = dqkv + (int64_t)head * HD;
      uint32_t raw[KS][4];
      raw_rows<T, HD>(raw, base + C, g.qkv_stride, tok, warp * 16, L, lane);
      __syncwarp();
      stage_live<T, HD, RS>(st_rows, dv, warp * 16, L, lane);
      __syncwarp();
      store_rows<T, HD, RS>(st_rows, dst + 2 * C, g.qkv_stride, tok, warp * 16, L, lane);
      // dL/dk' = ln 2 dS^T q', q' with log2 e
      norm_backward<T, HD>(dk, raw, kn, 0.69314718055994530942f, rk[k0], rk[k0 + 8], wk, lane);
      __syncwarp();
      stage_live<T, HD, RS>(st_rows, dk, warp * 16, L, lane);
      __syncwarp();
      store_rows<T, HD, RS>(st_rows, dst + C, g.qkv_stride, tok, warp * 16, L, lane);
    }
    __syncthreads();
    // ---- the next item's rows
    const int* tok_n = tok2 + (1 - cur) * rows;
    if (next) copy(head_n, tok_n, k_bufs > 1 ? sK0 + (1 - cur) * rows * RS : nullptr, true);
    const auto add_sums = [&]() {
      // A thread has a place (or several) and every groups-th displacement (dt, da) there
      const int step = bs.sa * (DS + 1), displacements = (2 * o.nt - 1) * (2 * bs.na - 1);
      for (int place = my_place; place < bs.places; place += nthreads) {
        const int bi = place / bs.nb, bj = place - bi * bs.nb;
        const T* at = sS + bi * bs.sb * DS + bj * bs.sb;
        float* sum = acc + bi * bs.nb + bj + my_group * bs.nb * bs.nb;
        int dt = 1 - o.nt, da = 1 - bs.na + my_group;
        for (int d = my_group; d < displacements; d += groups) {
          while (da >= bs.na) {
            da -= 2 * bs.na - 1;
            ++dt;
          }
          const int n = bs.na - abs(da);
          float s = 0.f;
          for (int t = max(dt, 0); t < o.nt + min(dt, 0); ++t) {
            const T* p = at + (t * o.ns * o.nf + max(da, 0) * bs.sa) * DS + (t - dt) * o.ns * o.nf + max(-da, 0) * bs.sa;
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
              s += to_f(*p);
              p += step;
            }
          }
          *sum += s;
          sum += groups * bs.nb * bs.nb;
          da += groups;
        }
      }
    };
    // ---- B.  The sums wait for shared memory, the products for one another: half of the warps begin with either.
    float dq[CH][4];
#pragma unroll
    for (int d = 0; d < CH; ++d) dq[d][0] = dq[d][1] = dq[d][2] = dq[d][3] = 0.f;
    uint32_t raw[KS][4];
    raw_rows<T, HD>(raw, base, g.qkv_stride, tok, warp * 16, L, lane);
    const uint32_t k_nn = rows_nn<T, RS>(sK, lane);
    const uint32_t a_at = smem_u32(sS + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * DS + (lane >> 4) * 8);
    if (dbias_part && (warp & 1)) add_sums();
#pragma unroll 2
    for (int kb = 0; kb < o.tiles; ++kb) {
      uint32_t a[4];
      ldsm_x4(a_at + kb * 32, a[0], a[1], a[2], a[3]);
      block_add<T, HD>(dq, a, k_nn + kb * kTile);
    }
    if (dbias_part && !(warp & 1)) add_sums();
    __syncthreads();  // k's rows have been read: dQ leaves by way of this warp's
    {
      const int q0 = warp * 16 + gq;
      T* st_rows = sK + warp * 16 * RS;
      // dL/dq' = ln 2 dS k', and q' is scale log2 e times the norm's result
      norm_backward<T, HD>(dq, raw, qn, g.scale, rq[q0], rq[q0 + 8], wq, lane);
      stage_live<T, HD, RS>(st_rows, dq, warp * 16, L, lane);
      __syncwarp();
      store_rows<T, HD, RS>(st_rows, dqkv + (int64_t)head * HD, g.qkv_stride, tok, warp * 16, L, lane);
    }
    if (next && k_bufs == 1) {
      __syncthreads();
      copy(head_n, tok_n, sK0, false);
    }
    cur = 1 - cur;
    head = head_n;
    win = win_n;
    window = window_n;
  }
  __syncthreads();
  if (dbias_part && tab_head >= 0) {
    flush(tab_head);
    __syncthreads();
  }
  // the warps' sums of the norms' weights' gradients, in order
  float* red = reinterpret_cast<float*>(sQ);  // [2][warps][HD]
  const int nw = nthreads / 32;
  put_cols<HD>(red + warp * HD, wq, lane);
  put_cols<HD>(red + (nw + warp) * HD, wk, lane);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * HD; i += nthreads) {
    const float* p = red + (i / HD) * nw * HD + i % HD;
    float s = 0.f;
    for (int w = 0; w < nw; ++w) s += p[w * HD];
    (i < HD ? dqw_part : dkw_part)[(int64_t)blockIdx.x * HD + i % HD] = s;
  }
}

// ------------------------------------------------------------------------------------------------------- launches
constexpr size_t kBlockSmem = 232448, kSmSmem = 233472;

template <typename T, int HD>
cudaError_t launch_fwd(const void* qkv, const AttnBias& bias, const float* norms, void* out, float* lse, const AttnGeom& g,
                       int sms, cudaStream_t s) {
  const Order o = order_of(g);
  FwdSmem<T, HD> S;
  const size_t smem = S.carve(nullptr, o);
  auto k = fwd_kernel<T, HD>;
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
  if (items > INT32_MAX) return cudaErrorInvalidValue;
  const int warps = std::min(o.tiles, kFwdWarps);
  // Few items: two blocks share one's queries, so that a warp has at most one tile (16 heads of one window of 162 tokens:
  // with the preparation 16.4 us in a graph, one block 20.5; 128 items 20.5 and 22.6, 224 items 30.5 and 26.6).
  const int parts = items <= sms && o.tiles > warps ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)items, (unsigned)parts);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, (const T*)qkv, bias, norms, (T*)out, reinterpret_cast<float2*>(lse), g, o);
}

// How many blocks the device holds at once, and whether keys have two buffers: where that costs no block of an SM
template <typename T, int HD>
AttnBiasPlan plan_bwd(const AttnGeom& g, bool dbias, int sms) {
  const Order o = order_of(g);
  const int entries = dbias ? sums_of(o).entries : 0;
  int blocks[2];
  for (int k = 1; k <= 2; ++k) {
    BwdSmem<T, HD> S;
    const size_t smem = S.carve(nullptr, o, entries, k);
    // (the launch bounds leave a thread 168 registers)
    const int fit = (int)std::min<size_t>(kSmSmem / (smem + 1024), 65536 / (168 * 32 * (size_t)o.tiles));
    blocks[k - 1] = smem > kBlockSmem ? 0 : std::max(1, std::min(fit, 16));
  }
  AttnBiasPlan p;
  p.k_bufs = blocks[1] == blocks[0] ? 2 : 1;
  const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
  p.blocks = (int)std::min<int64_t>(items, (int64_t)sms * blocks[0]);
  p.norm_rows = p.blocks;
  p.bias_rows = p.blocks + g.nh - 1;
  return p;
}

template <typename T, int HD>
cudaError_t launch_bwd(const void* qkv, const AttnBias& bias, const float* norms, const void* out, const void* dout,
                       const float* lse, void* dqkv, float* dqw_part, float* dkw_part, float* dbias_part,
                       const AttnBiasPlan& plan, const AttnGeom& g, cudaStream_t s) {
  const Order o = order_of(g);
  BwdSmem<T, HD> S;
  const size_t smem = S.carve(nullptr, o, dbias_part ? sums_of(o).entries : 0, plan.k_bufs);
  auto k = bwd_kernel<T, HD>;
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  k<<<plan.blocks, 32 * o.tiles, smem, s>>>((const T*)qkv, bias, norms, (const T*)out, (const T*)dout,
                                            reinterpret_cast<const float2*>(lse), (T*)dqkv, dqw_part, dkw_part, dbias_part,
                                            plan.k_bufs, g, o);
  return cudaGetLastError();
}

// f(type, head_dim) of the call's; WIDE: head_dim 128 too
template <bool WIDE, typename F>
auto dispatch(const AttnGeom& g, int dtype, F f) {
  const auto hd = [&](auto t) {
    using I16 = std::integral_constant<int, 16>;
    using I32 = std::integral_constant<int, 32>;
    using I64 = std::integral_constant<int, 64>;
    if constexpr (WIDE)
      if (g.hd == 128) return f(t, std::integral_constant<int, 128>());
    return g.hd == 16 ? f(t, I16()) : g.hd == 32 ? f(t, I32()) : f(t, I64());
  };
  return dtype == kBF16 ? hd(__nv_bfloat16()) : hd(__half());
}

}  // namespace attn_bias

static bool attn_bias_ok(const AttnGeom& g, int dtype) {
  return (g.hd == 16 || g.hd == 32 || g.hd == 64 || g.hd == 128) && (dtype == kBF16 || dtype == kF16) && g.T > 0 &&
         g.wh > 0 && g.ww > 0 && (int64_t)g.T * g.wh * g.ww <= 192 && g.H % g.wh == 0 && g.W % g.ww == 0 &&
         (int64_t)g.B * g.T * g.H * g.W < INT32_MAX;
}

static int buckets_of(const AttnGeom& g) { return (2 * g.T - 1) * (2 * g.wh - 1) * (2 * g.ww - 1); }
AttnBias attn_bias_layout(const AttnGeom& g) { return {nullptr, (4 + buckets_of(g) + 3) / 4 * 4}; }

cudaError_t attn_bias_prepare(const AnyMatrix& table, const AnyMatrix& qw, const AnyMatrix& kw, const AttnGeom& g,
                              const AttnBias& b, float* tab, cudaStream_t s) {
  attn_bias::prepare_kernel<<<g.nh + 1, 256, 0, s>>>(table, qw, kw, b, g.nh, g.hd, buckets_of(g), g.scale, tab);
  return cudaGetLastError();
}

cudaError_t attn_bias_fwd(const void* qkv, const AttnBias& bias, const float* norms, void* out, float* lse,
                          const AttnGeom& g, int dtype, int sms, cudaStream_t s) {
  if (!attn_bias_ok(g, dtype)) return cudaErrorInvalidValue;
  return attn_bias::dispatch<true>(g, dtype, [&](auto t, auto hd) {
    return attn_bias::launch_fwd<decltype(t), hd()>(qkv, bias, norms, out, lse, g, sms, s);
  });
}

AttnBiasPlan attn_bias_plan(const AttnGeom& g, int dtype, bool dbias, int sms) {
  if (g.hd == 128) {
    const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
    return {0, 0, items, items};
  }
  return attn_bias::dispatch<false>(g, dtype, [&](auto t, auto hd) {
    return attn_bias::plan_bwd<decltype(t), hd()>(g, dbias, sms);
  });
}

cudaError_t attn_bias_bwd(const void* qkv, const AttnBias& bias, const float* norms, const void* out, const void* dout,
                          const float* lse, void* dqkv, float* dqw_part, float* dkw_part, float* dbias_part,
                          const AttnBiasPlan& plan, const AttnGeom& g, int dtype, cudaStream_t s) {
  if (!attn_bias_ok(g, dtype)) return cudaErrorInvalidValue;
  if (g.hd == 128)
    return window_attn_bwd(qkv, norms, norms + g.hd, out, dout, lse, dqkv, dqw_part, dkw_part, g, dtype, s, bias, dbias_part);
  return attn_bias::dispatch<false>(g, dtype, [&](auto t, auto hd) {
    return attn_bias::launch_bwd<decltype(t), hd()>(qkv, bias, norms, out, dout, lse, dqkv, dqw_part, dkw_part,
                                                            dbias_part, plan, g, s);
  });
}

cudaError_t attn_bias_grads(const AttnGrad& bias, const AttnGrad& q, const AttnGrad& k, const AttnBiasPlan& plan,
                            const AttnGeom& g, cudaStream_t s) {
  attn_bias::Grads p{};
  p.bias = bias;
  p.q = q;
  p.k = k;
  p.windows = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww);
  p.qk_rows = plan.norm_rows;
  p.heads = g.nh;
  p.grid = plan.blocks;
  p.buckets = buckets_of(g);
  p.hd = g.hd;
  attn_bias::grad_kernel<<<dim3((std::max(p.buckets, g.hd) + 31) / 32, g.nh + 2), 1024, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace nsw
