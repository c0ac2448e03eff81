// Window attention with a learned relative position bias, forward and backward, on mma.sync.
//
//   s_ij = scale <rms(q_i) qw, rms(k_j) kw> + table[head, bucket(i, j)] - 100 [i and j on different sides of the wrap]
//   p = softmax(s);  o = p v
//   dv = p^T do;  dp = do v^T;  ds = p (dp - <do, o>);  dq = scale ds k;  dk = scale ds^T q;  dtable[c] = sum of ds in c
//   bucket = ((t_i - t_j + T - 1) (2 wh - 1) + y_i - y_j + wh - 1) (2 ww - 1) + x_i - x_j + ww - 1
//
// A window is at most 192 tokens of one head, so its products are short: what counts is how few instructions stand around
// them, and that several windows are worked on at once on an SM.
#include <float.h>

#include <algorithm>

#include "attn_mma.cuh"
#include "kernels.h"

namespace nsw {
namespace attn_bias {

using attn::cp_async16;
using attn::cp_async_wait_all;
using attn::fast_exp2;
using attn::kLog2e;
using attn::ldsm_x4;
using attn::ldsm_x4_t;
using attn::mma16816;
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

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == kBF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return to_f(reinterpret_cast<const __half*>(p)[i]);
}

constexpr float kAbsorbs = 1099511627776.f;  // 2^40

// One block a head, and one for the norms' weights.  Entries are less the head's largest, so that an offset of all of them
// costs no precision, unless that is beyond 2^40: a head of the lowest value throughout, say, absorbs the logits, as it
// does in 64 bits, and its rows are even.  A finite entry stays finite.
__global__ void __launch_bounds__(256) prepare_kernel(const AnyMatrix table, const AnyMatrix qw, const AnyMatrix kw, const AttnBias b,
                                                      int heads, int hd, int nt, int ny, int nx,
                                                      float* __restrict__ tab) {
  __shared__ float hi_w[8], lo_w[8];
  const int h = blockIdx.x, n = nt * ny * nx;
  float* out = tab + (int64_t)h * b.stride;
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
  const bool shifted = fabsf(hi) <= kAbsorbs;
  const float shift = shifted ? hi : 0.f;
  const auto entry = [&](float v) {
    const float e = (v - shift) * kLog2e;
    return isinf(e) && !isinf(v) ? copysignf(FLT_MAX, e) : e;
  };
  const int nf = b.y_fast ? ny : nx, ns = b.y_fast ? nx : ny;
  for (int i = threadIdx.x; i < b.stride; i += 256) {
    const int at = i - 4, row = at / b.pitch, f = at - row * b.pitch, t = row / ns, s = row - t * ns;
    float v = 0.f;
    if (i == 0) {
      v = shifted ? -entry(lo) : INFINITY;  // (the forward's bound on the logits needs the largest to be 0)
    } else if (at >= 0 && t < nt && f < nf) {
      const int y = b.y_fast ? f : s, x = b.y_fast ? s : f;
      v = entry(load_any(table.p, table.dtype, h * table.s0 + ((t * ny + y) * nx + x) * table.s1));
    }
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
  if (t.dtype == kF32)
    reinterpret_cast<float*>(t.out)[at] = a;
  else if (t.dtype == kBF16)
    reinterpret_cast<__nv_bfloat16*>(t.out)[at] = from_f<__nv_bfloat16>(a);
  else
    reinterpret_cast<__half*>(t.out)[at] = from_f<__half>(a);
}

// ------------------------------------------------------------------------------------------------------ layout
// Tokens of a window in the order in which the kernels take them: one of latitude and longitude fastest (extent nf), the
// other (ns) next, time slowest.
struct Order {
  int nf, ns, nt, length, tiles;  // tiles of 16 tokens
  bool y_fast;
  int pitch, entries;             // entry of query i and key j: center + off(i) - off(j)
  int center;
};
__host__ __device__ __forceinline__ Order order_of(const AttnGeom& g, const AttnBias& b) {
  Order o;
  o.y_fast = b.y_fast != 0;
  o.nf = o.y_fast ? g.wh : g.ww;
  o.ns = o.y_fast ? g.ww : g.wh;
  o.nt = g.T;
  o.length = g.T * g.wh * g.ww;
  o.tiles = (o.length + 15) / 16;
  o.pitch = b.pitch;
  o.entries = (2 * g.T - 1) * (2 * o.ns - 1) * b.pitch;
  o.center = ((g.T - 1) * (2 * o.ns - 1) + o.ns - 1) * b.pitch + o.nf - 1;
  return o;
}
__device__ __forceinline__ int off_of(const Order& o, int i) {
  const int s = i / o.nf, t = s / o.ns;
  return (t * (2 * o.ns - 1) + s - t * o.ns) * o.pitch + i - s * o.nf;
}
// Grid token of window token i, and its side of the latitude wrap
__device__ __forceinline__ int token_of(const AttnGeom& g, const Order& o, int64_t win, int i, int& side) {
  const int nww = g.W / g.ww, nwh = g.H / g.wh;
  const int wx = (int)(win % nww), wy = (int)((win / nww) % nwh), b = (int)(win / ((int64_t)nww * nwh));
  const int r = i / o.nf, f = i - r * o.nf, t = r / o.ns, s = r - t * o.ns;
  const int y = wy * g.wh + (o.y_fast ? f : s), x = wx * g.ww + (o.y_fast ? s : f);
  int gy = (y + g.sh) % g.H, gx = (x + g.sw) % g.W;
  if (gy < 0) gy += g.H;
  if (gx < 0) gx += g.W;
  side = g.mask && g.mask_shift > 0 && g.row_offset + y >= g.h_global - g.mask_shift;
  return (int)((((int64_t)b * g.T + t) * g.H + gy) * g.W + gx);
}

// The entries of a head in shared memory, twice: a lane of the products has pairs of neighbouring tokens across and one
// token down, whose entries are two neighbours in either order; if the fast extent and the pitch are even, the pair's
// place has the parity of the token down, and one of the copies (the second begins one entry later) has it 8-byte
// aligned, one load for two entries.  Their distance modulo the banks keeps the copies' reads apart.
__host__ __device__ __forceinline__ int second_copy(int entries) { return (entries + 31) / 32 * 32 + 16; }
__host__ __device__ __forceinline__ int table_floats(int entries) { return second_copy(entries) + (entries + 1) / 2 * 2; }
__device__ __forceinline__ void load_table(float* tab, const AttnBias& b, int entries, int head) {
  const float* src = b.tab + (int64_t)head * b.stride + 4;
  for (int i = threadIdx.x; i < entries; i += blockDim.x) {
    const float v = src[i];
    tab[i] = v;
    if (i > 0) tab[second_copy(entries) + i - 1] = v;
  }
}
// where the entry `base` and the next one are a pair
__device__ __forceinline__ const float* pair_at(const float* tab, int entries, int base) {
  return tab + (base & 1 ? second_copy(entries) - 1 : 0) + base;
}

// Eight entries of a 16 x 16 block of logits less `sub` of their row (DOWN: of their column), in the layout of mma's
// results: c[j][e] for row r0 (e < 2) or r0 + 8 and column 8 j + 2 tq + (e & 1).
//   rows are queries: entry = center + off(row) - off(column)      (ACROSS = -1)
//   rows are keys:    entry = center + off(column) - off(row)      (ACROSS = +1)
// row0 / row1: with pairs, pair_at(center +- off(row) (- 1 for rows of queries)), else tab + center +- off(row).
// off4: the offsets in bytes.
template <bool PAIR, int ACROSS>
__device__ __forceinline__ void load_block(float (&v)[2][4], const float* row0, const float* row1, const int* off4,
                                           int col, int tq) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (PAIR) {
      const int o = ACROSS * off4[col + 8 * j + 2 * tq];
      const float2 a = *reinterpret_cast<const float2*>(reinterpret_cast<const char*>(row0) + o);
      const float2 b = *reinterpret_cast<const float2*>(reinterpret_cast<const char*>(row1) + o);
      v[j][0] = ACROSS < 0 ? a.y : a.x;
      v[j][1] = ACROSS < 0 ? a.x : a.y;
      v[j][2] = ACROSS < 0 ? b.y : b.x;
      v[j][3] = ACROSS < 0 ? b.x : b.y;
    } else {
      const int2 o = *reinterpret_cast<const int2*>(off4 + col + 8 * j + 2 * tq);
      v[j][0] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(row0) + ACROSS * o.x);
      v[j][1] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(row0) + ACROSS * o.y);
      v[j][2] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(row1) + ACROSS * o.x);
      v[j][3] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(row1) + ACROSS * o.y);
    }
  }
}
// The latitude-wrap mask, and -inf for padding keys: side is 0 / 1, -1 for padding.  Rows are queries or (KEYS) keys.
template <bool KEYS>
__device__ __forceinline__ void mask_block(float (&v)[2][4], const signed char* side, int row, int col, int tq) {
  const int s0 = side[row], s1 = side[row + 8];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int sr = e < 2 ? s0 : s1, sc = side[col + 8 * j + 2 * tq + (e & 1)];
      const int key = KEYS ? sr : sc, query = KEYS ? sc : sr;
      if (key < 0)
        v[j][e] = -INFINITY;
      else if (query >= 0 && key != query)
        v[j][e] += -100.f * kLog2e;
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

// a 16 x 16 block of A B^T: A in fragments, B's 16 rows at `rows` in shared memory (row stride RS)
template <typename T, int HD, int RS>
__device__ __forceinline__ void block_product(float (&c)[2][4], const uint32_t (&a)[HD / 16][4], const T* rows, int lane) {
  const uint32_t at = smem_u32(rows + ((lane & 7) + (lane >> 4) * 8) * RS + ((lane >> 3) & 1) * 8);
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    uint32_t b0, b1, b2, b3;
    ldsm_x4(at + ks * 32, b0, b1, b2, b3);
    mma16816<T>(c[0], a[ks], b0, b1);
    mma16816<T>(c[1], a[ks], b2, b3);
  }
}
// o += P V for 16 rows of P (one fragment) and the 16 rows of V at `rows`
template <typename T, int HD, int RS>
__device__ __forceinline__ void block_add(float (&o)[HD / 8][4], const uint32_t (&p)[4], const T* rows, int lane) {
  const uint32_t at = smem_u32(rows + ((lane & 7) + ((lane >> 3) & 1) * 8) * RS + (lane >> 4) * 8);
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

// RMSNorm of one row by HD / 8 lanes, eight elements each: x * rs * w (w in shared memory); rs of the row
template <typename T, int HD>
__device__ __forceinline__ float norm_chunk(const uint4& raw, const float* w, uint4& out, float* norm2) {
  float f[8], v[8];
  unpack8<T>(raw, f);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
#pragma unroll
  for (int o = 1; o < HD / 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float rs = rsqrtf(ss * (1.f / HD) + FLT_EPSILON);
  float n2 = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = f[i] * (rs * w[i]);
    n2 = fmaf(v[i], v[i], n2);
  }
  out = pack8<T>(v);
  if (norm2) {
#pragma unroll
    for (int o = 1; o < HD / 8; o <<= 1) n2 += __shfl_xor_sync(0xffffffffu, n2, o);
    *norm2 = n2;
  }
  return rs;
}

// A row's exponentials are taken less a bound on its logits where that keeps them normal in T: with the largest entry 0,
// a logit is at most |q| max |k| and at least its negative less the entries' range.  bf16: results in [2^-96, 1]; fp16: in
// [2^-14, 2^14].  Otherwise less the row's largest logit, for one more product of q and k.
template <typename T>
struct Bound;
template <>
struct Bound<__nv_bfloat16> {
  static constexpr float most = 48.f, top = 0.f;
};
template <>
struct Bound<__half> {
  static constexpr float most = 14.f, top = 14.f;
};

// ----------------------------------------------------------------------------------------------------- forward
// A block takes a window and head, a warp 16 queries at a time.  K is normalised into shared memory, V copied there; the
// queries' fragments come straight from global memory and are normalised in registers, with scale and log2 e, so that
// the first product, which begins with the entries less the row's bound, ends in the exponents themselves.  P goes from
// registers into the second product.  Nothing waits for a row's maximum, and several blocks share an SM, so that one's
// loads and norms run beside the others' products.
constexpr int kFwdWarps = 6;
template <typename T, int HD>
struct FwdSmem {
  float *tab, *qw, *kw, *red;
  T *k, *v, *stage;
  int *tok, *off4;
  signed char* side;
  __host__ __device__ size_t carve(unsigned char* base, const Order& o) {
    const int rows = o.tiles * 16, RS = HD + 8;
    Carve c{base, 0};
    tab = c.take<float>(table_floats(o.entries));
    k = c.take<T>(rows * RS);
    v = c.take<T>(rows * RS);
    stage = c.take<T>(16 * kFwdWarps * RS);
    tok = c.take<int>(rows);
    off4 = c.take<int>(rows);
    qw = c.take<float>(HD);  // with scale and log2 e
    kw = c.take<float>(HD);
    red = c.take<float>(kFwdWarps);
    side = c.take<signed char>(rows);
    return c.at;
  }
};
template <typename T, int HD, bool PAIR>
__global__ void __launch_bounds__(32 * kFwdWarps, HD <= 64 ? 3 : 2)
    fwd_kernel(const T* __restrict__ qkv, const AttnBias bias, const float* __restrict__ norms, T* __restrict__ out,
               float2* __restrict__ lse, const AttnGeom g) {
  constexpr int RS = HD + 8, KS = HD / 16, CH = HD / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  const Order o = order_of(g, bias);
  const int L = o.length, rows = o.tiles * 16, nthreads = blockDim.x, nw = nthreads / 32;
  FwdSmem<T, HD> S;
  S.carve(smem, o);
  float *tab = S.tab, *qw = S.qw, *kw = S.kw, *red = S.red;
  T *sK = S.k, *sV = S.v, *stage = S.stage;
  int *tok = S.tok, *off4 = S.off4;
  signed char* side = S.side;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int head = blockIdx.x % g.nh;
  const int64_t win = blockIdx.x / g.nh;
  const int64_t C = (int64_t)g.nh * HD;
  const T* base = qkv + (int64_t)head * HD;

  int mixed = 0;
  {
    int first;
    token_of(g, o, win, 0, first);
    for (int i = threadIdx.x; i < rows; i += nthreads) {
      int s = -1;
      tok[i] = i < L ? token_of(g, o, win, i, s) : 0;
      off4[i] = i < L ? 4 * off_of(o, i) : 0;
      side[i] = (signed char)s;
      mixed |= i < L && s != first;
    }
  }
  for (int i = threadIdx.x; i < HD; i += nthreads) {
    qw[i] = norms[i] * (g.scale * kLog2e);
    kw[i] = norms[HD + i];
  }
  mixed = __syncthreads_or(mixed);
  // the first tile's raw queries, on their way under what follows
  uint32_t raw[KS][4];
  const auto load_queries = [&](int qt) {
    const int r0 = qt * 16 + gq, r1 = r0 + 8;
    const T* p0 = base + (int64_t)tok[r0] * g.qkv_stride + 2 * tq;
    const T* p1 = base + (int64_t)tok[r1] * g.qkv_stride + 2 * tq;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      raw[ks][0] = r0 < L ? ld32(p0 + ks * 16) : 0u;
      raw[ks][1] = r1 < L ? ld32(p1 + ks * 16) : 0u;
      raw[ks][2] = r0 < L ? ld32(p0 + ks * 16 + 8) : 0u;
      raw[ks][3] = r1 < L ? ld32(p1 + ks * 16 + 8) : 0u;
    }
  };
  if (warp < o.tiles) load_queries(warp);
  for (int i = threadIdx.x; i < rows * CH; i += nthreads) {
    const int r = i / CH, c = i % CH;
    T* dst = sV + r * RS + 8 * c;
    if (r < L)
      cp_async16(dst, base + (int64_t)tok[r] * g.qkv_stride + 2 * C + 8 * c);
    else
      *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
  }
  load_table(tab, bias, o.entries, head);
  // keys: the lanes of a row are neighbours, and a warp's rows are whole (32 is a multiple of CH)
  float kmax = 0.f;
  for (int i0 = 0; i0 < rows * CH; i0 += 4 * nthreads) {
    uint4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * nthreads + threadIdx.x, r = i / CH;
      x[u] = i < rows * CH && r < L
                 ? __ldg(reinterpret_cast<const uint4*>(base + (int64_t)tok[r] * g.qkv_stride + C + 8 * (i % CH)))
                 : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * nthreads + threadIdx.x;
      float n2;
      uint4 y;
      norm_chunk<T, HD>(x[u], kw + 8 * (i % CH), y, &n2);
      kmax = fmaxf(kmax, n2);
      if (i < rows * CH) *reinterpret_cast<uint4*>(sK + (i / CH) * RS + 8 * (i % CH)) = y;
    }
  }
  kmax = warp_max(kmax);
  if (lane == 0) red[warp] = kmax;
  cp_async_wait_all();
  __syncthreads();
  for (int w = 0; w < nw; ++w) kmax = fmaxf(kmax, red[w]);
  kmax = sqrtf(kmax) * 1.01f;  // (a margin for the roundings of q and k)
  const float spread = 0.5f * bias.tab[(int64_t)head * bias.stride];

  for (int qt = warp; qt < o.tiles; qt += nw) {
    if (qt != warp) load_queries(qt);
    const int r0 = qt * 16 + gq, r1 = r0 + 8;
    uint32_t qa[KS][4];
    float n0, n1;
    {
      float s0 = 0.f, s1 = 0.f;
      float f[2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unpack2(raw[ks][e], f, T());
          float& s = e & 1 ? s1 : s0;
          s = fmaf(f[0], f[0], fmaf(f[1], f[1], s));
        }
      const float rs0 = rsqrtf(quad_sum(s0) * (1.f / HD) + FLT_EPSILON);
      const float rs1 = rsqrtf(quad_sum(s1) * (1.f / HD) + FLT_EPSILON);
      s0 = s1 = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unpack2(raw[ks][e], f, T());
          const float2 w = *reinterpret_cast<const float2*>(qw + ks * 16 + (e >> 1) * 8 + 2 * tq);
          const float rs = e & 1 ? rs1 : rs0;
          f[0] *= rs * w.x;
          f[1] *= rs * w.y;
          float& s = e & 1 ? s1 : s0;
          s = fmaf(f[0], f[0], fmaf(f[1], f[1], s));
          qa[ks][e] = pack2<T>(f[0], f[1]);
        }
      n0 = sqrtf(quad_sum(s0));
      n1 = sqrtf(quad_sum(s1));
    }
    const int at0 = o.center + (off4[r0] >> 2), at1 = o.center + (off4[r1] >> 2);
    const float* row0 = PAIR ? pair_at(tab, o.entries, at0 - 1) : tab + at0;
    const float* row1 = PAIR ? pair_at(tab, o.entries, at1 - 1) : tab + at1;
    const auto logits = [&](float (&c)[2][4], int kb, float m0, float m1) {
      load_block<PAIR, -1>(c, row0, row1, off4, kb * 16, tq);
      if (mixed || kb * 16 + 16 > L) mask_block<false>(c, side, r0, kb * 16, tq);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c[j][0] -= m0;
        c[j][1] -= m0;
        c[j][2] -= m1;
        c[j][3] -= m1;
      }
      block_product<T, HD, RS>(c, qa, sK + kb * 16 * RS, lane);
    };
    float m0 = n0 * kmax, m1 = n1 * kmax;
    bool late = false;  // a row of entries beyond kAbsorbs throughout: they absorb the product before they are subtracted
    if (__all_sync(0xffffffffu, m0 + spread <= Bound<T>::most && m1 + spread <= Bound<T>::most)) {
      m0 -= Bound<T>::top;
      m1 -= Bound<T>::top;
    } else {
      m0 = m1 = -INFINITY;
      for (int kb = 0; kb < o.tiles; ++kb) {
        float c[2][4];
        logits(c, kb, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          m0 = fmaxf(m0, fmaxf(c[j][0], c[j][1]));
          m1 = fmaxf(m1, fmaxf(c[j][2], c[j][3]));
        }
      }
      m0 = quad_max(m0);
      m1 = quad_max(m1);
      if (m0 == -INFINITY) m0 = 0.f;  // a row that the bias masks throughout: P = 0
      if (m1 == -INFINITY) m1 = 0.f;
      late = __any_sync(0xffffffffu, fabsf(m0) > kAbsorbs || fabsf(m1) > kAbsorbs);
    }
    // the rows' sums are those of the rounded values that are multiplied, by one more product (with ones): so a row's
    // weights add up to one as they are, and the sum costs an instruction where eight additions would
    float acc[CH][4], sum[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t ones = pack2<T>(1.f, 1.f);
#pragma unroll
    for (int d = 0; d < CH; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.f;
#pragma unroll 1
    for (int kb = 0; kb < o.tiles; ++kb) {
      float c[2][4];
      logits(c, kb, late ? 0.f : m0, late ? 0.f : m1);
      if (late) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          c[j][0] -= m0;
          c[j][1] -= m0;
          c[j][2] -= m1;
          c[j][3] -= m1;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[j][e] = fast_exp2(c[j][e]);
      const uint32_t p[4] = {pack2<T>(c[0][0], c[0][1]), pack2<T>(c[0][2], c[0][3]), pack2<T>(c[1][0], c[1][1]),
                             pack2<T>(c[1][2], c[1][3])};
      mma16816<T>(sum, p, ones, ones);
      block_add<T, HD, RS>(acc, p, sV + kb * 16 * RS, lane);
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
      float2* at = lse + ((int64_t)win * g.nh + head) * L;
      if (r0 < L) at[r0] = l0 == 0.f ? make_float2(0.f, 0.f) : make_float2(m0, log2f(l0));
      if (r1 < L) at[r1] = l1 == 0.f ? make_float2(0.f, 0.f) : make_float2(m1, log2f(l1));
    }
    T* st = stage + warp * 16 * RS;
    __syncwarp();
    stage_rows<T, HD, RS>(st, acc, lane);
    __syncwarp();
    store_rows<T, HD, RS>(st, out + (int64_t)head * HD, g.out_stride, tok, qt * 16, L, lane);
  }
}

// ---------------------------------------------------------------------------------------------------- backward
// Blocks walk the (head, window) list in contiguous pieces, a warp for each 16 tokens of a window.  For an item:
//   norms   the raw rows of q and k, copied to shared memory while the item before was worked on, become what the
//           forward took; D_i = <dO_i, O_i>
//   A       a warp's 16 keys against all queries: S^T begins with the entries less the row's logarithm of the sum, dP^T
//           with -D, so that P^T is an exponential and dS^T a product away; dV and dK stay in registers; dS goes to shared
//           memory in T (as the products take it), queries down
//   B       a warp's 16 queries: dQ = dS K.  The next item's rows are on their way.
// The bias's gradient sums dS over the windows of a head, without atomics and in a fixed order: of the two extents of the
// window, one, a, is summed at once and the other, b, kept as a pair, acc[dt][da][b_i][b_j], whose entries belong to
// threads; the diagonals b_i - b_j are summed when the head is done, into the block's row for it.
// The norms' backward takes the raw rows from global memory (L2) again, in the fragments' layout.
struct BiasSums {
  bool a_is_s;           // a: the slow extent
  int na, nb, sa, sb;    // extents and strides in tokens
  int entries, width;    // width: entries a thread's task has, neighbours in b_j
  uint32_t div_b, div_b2, div_a;
};
__host__ __device__ __forceinline__ uint32_t magic_of(int d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); }
__device__ __forceinline__ int quick_div(int v, uint32_t magic) {  // v / d for v < 2^16
  return magic ? (int)__umulhi((uint32_t)v, magic) : v;
}
template <bool PAIR>
__host__ __device__ __forceinline__ BiasSums sums_of(const Order& o) {
  BiasSums b;
  b.a_is_s = PAIR || (2 * o.ns - 1) * o.nf * o.nf <= (2 * o.nf - 1) * o.ns * o.ns;
  b.na = b.a_is_s ? o.ns : o.nf;
  b.nb = b.a_is_s ? o.nf : o.ns;
  b.sa = b.a_is_s ? o.nf : 1;
  b.sb = b.a_is_s ? 1 : o.nf;
  b.width = PAIR ? 2 : 1;
  b.entries = (2 * o.nt - 1) * (2 * b.na - 1) * b.nb * b.nb;
  b.div_b = magic_of(b.nb / b.width);
  b.div_b2 = magic_of(b.nb);
  b.div_a = magic_of(2 * b.na - 1);
  return b;
}

template <typename T, int HD>
struct BwdSmem {
  float *tab, *acc, *sub, *late, *ll, *negD, *rq, *rk, *qw, *qn, *kw;
  T *q, *v, *g, *k, *s;
  int *tok, *off4;
  signed char* side;
  // entries: of the bias's sums; k_bufs: buffers for k (two, where there is room: the next item's keys arrive while this
  // one's are read)
  __host__ __device__ size_t carve(unsigned char* base, const Order& o, int entries, int k_bufs) {
    const int rows = o.tiles * 16, RS = HD + 8;
    Carve c{base, 0};
    tab = c.take<float>(table_floats(o.entries));
    acc = c.take<float>(entries);
    q = c.take<T>(rows * RS * (3 + k_bufs));
    v = q + rows * RS;
    g = v + rows * RS;  // dO
    k = g + rows * RS;
    s = c.take<T>(rows * (rows + 8));  // dS, [query][key]
    tok = c.take<int>(2 * rows);
    off4 = c.take<int>(rows);
    sub = c.take<float>(rows);   // what the exponents are less: of each query
    late = c.take<float>(rows);  // wide rows: and after the product, first this, then this
    ll = c.take<float>(rows);
    negD = c.take<float>(rows);
    rq = c.take<float>(rows);
    rk = c.take<float>(rows);
    qw = c.take<float>(HD);  // with scale and log2 e
    qn = c.take<float>(HD);
    kw = c.take<float>(HD);
    side = c.take<signed char>(2 * rows);
    return c.at;
  }
};

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
// rows past the window become zeros (their places in shared memory hold zeros for good)
template <typename T, int HD, int RS>
__device__ __forceinline__ void stage_live(T* rows, float (&o)[HD / 8][4], int row, int length, int lane) {
  const bool live0 = row + (lane >> 2) < length, live1 = row + (lane >> 2) + 8 < length;
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) {
    if (!live0) o[d][0] = o[d][1] = 0.f;
    if (!live1) o[d][2] = o[d][3] = 0.f;
  }
  stage_rows<T, HD, RS>(rows, o, lane);
}
// A tile's gradient g (times `scale`) of y = x rs w becomes that of x, dx = rs w g - x rs^3 mean(w g x); sums gets the
// tile's columns of g x rs: two of them a lane, after a butterfly over the rows that halves what a lane holds.
template <typename T, int HD>
__device__ __forceinline__ void norm_backward(float (&g)[HD / 8][4], const uint32_t (&raw)[HD / 16][4], const float* w,
                                              float scale, float rs0, float rs1, bool live0, bool live1, float (&sums)[2],
                                              int lane) {
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
      const float g0 = live0 ? g[d][e] * scale : 0.f, g1 = live1 ? g[d][2 + e] * scale : 0.f;
      c[2 * d + e] = fmaf(g0 * x0[e], rs0, g1 * x1[e] * rs1);
      g[d][e] = g0 * we[e];
      g[d][2 + e] = g1 * we[e];
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
  sums[0] += c[0];
  sums[1] += c[1];
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
template <typename T, int HD, bool PAIR>
__global__ void __launch_bounds__(32 * kBwdWarps, 1)
    bwd_kernel(const T* __restrict__ qkv, const AttnBias bias, const float* __restrict__ norms, const T* __restrict__ out,
               const T* __restrict__ dout, const float2* __restrict__ lse, T* __restrict__ dqkv,
               float* __restrict__ dqw_part, float* __restrict__ dkw_part, float* __restrict__ dbias_part, int k_bufs,
               const AttnGeom g) {
  constexpr int RS = HD + 8, KS = HD / 16, CH = HD / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  const Order o = order_of(g, bias);
  const BiasSums bs = sums_of<PAIR>(o);
  const int L = o.length, rows = o.tiles * 16, DS = rows + 8, nthreads = blockDim.x;
  const int buckets = (2 * g.T - 1) * (2 * g.wh - 1) * (2 * g.ww - 1);
  BwdSmem<T, HD> S;
  S.carve(smem, o, dbias_part ? bs.entries : 0, k_bufs);
  float *tab = S.tab, *acc = S.acc, *sub = S.sub, *late = S.late, *ll = S.ll, *negD = S.negD, *rq = S.rq, *rk = S.rk, *qw = S.qw,
        *qn = S.qn, *kw = S.kw;
  T *sQ = S.q, *sV = S.v, *sG = S.g, *sK0 = S.k, *sS = S.s;
  int *tok2 = S.tok, *off4 = S.off4;
  signed char* side2 = S.side;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, tq = lane & 3;
  const int64_t C = (int64_t)g.nh * HD;
  const int64_t n_win = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww), n_items = n_win * g.nh;
  const int64_t i_begin = n_items * blockIdx.x / gridDim.x, i_end = n_items * (blockIdx.x + 1) / gridDim.x;

  for (int i = threadIdx.x; i < rows; i += nthreads) off4[i] = i < L ? 4 * off_of(o, i) : 0;
  for (int i = threadIdx.x; i < HD; i += nthreads) {
    qw[i] = norms[i] * (g.scale * kLog2e);
    qn[i] = norms[i];
    kw[i] = norms[HD + i];
  }
  // padding rows stay zero: copies and staged rows write the window's rows alone
  for (int i = threadIdx.x; i < (rows - L) * CH * (3 + k_bufs); i += nthreads) {
    const int b = i / ((rows - L) * CH), r = i % ((rows - L) * CH);
    *reinterpret_cast<uint4*>(sQ + (b * rows + L + r / CH) * RS + 8 * (r % CH)) = make_uint4(0, 0, 0, 0);
  }
  if (dbias_part)
    for (int i = threadIdx.x; i < bs.entries; i += nthreads) acc[i] = 0.f;

  // the window's tokens and sides into table `buf`; its mix of sides by the caller's barrier
  const auto build = [&](int64_t win, int buf) {
    int first, mix = 0;
    token_of(g, o, win, 0, first);
    for (int i = threadIdx.x; i < rows; i += nthreads) {
      int s = -1;
      tok2[buf * rows + i] = i < L ? token_of(g, o, win, i, s) : 0;
      side2[buf * rows + i] = (signed char)s;
      mix |= i < L && s != first;
    }
    return mix;
  };
  // one operand's rows of an item
  const auto copy = [&](T* dst, const T* src, int64_t stride, const int* tok) {
    for (int i = threadIdx.x; i < L * CH; i += nthreads) {
      const int r = i / CH, c = i % CH;
      cp_async16(dst + r * RS + 8 * c, src + (int64_t)tok[r] * stride + 8 * c);
    }
  };
  const auto head_of = [&](int64_t item) { return (int)(item / n_win); };
  const auto flush = [&](int head) {  // the head's sums into the block's row for it; between barriers
    float* dst = dbias_part + ((int64_t)blockIdx.x + head) * buckets;
    const int ny = 2 * g.wh - 1, nx = 2 * g.ww - 1;
    for (int c = threadIdx.x; c < buckets; c += nthreads) {
      const int dt = c / (ny * nx), dy = c / nx - dt * ny, dx = c % nx;
      const int df = o.y_fast ? dy : dx, ds = o.y_fast ? dx : dy;
      const int da = bs.a_is_s ? ds : df, db = (bs.a_is_s ? df : ds) - (bs.nb - 1);
      const float* a = acc + (dt * (2 * bs.na - 1) + da) * bs.nb * bs.nb + max(db, 0) * bs.nb + max(-db, 0);
      float s = 0.f;
      for (int i = 0; i < bs.nb - abs(db); ++i) s += a[i * (bs.nb + 1)];
      dst[c] = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bs.entries; i += nthreads) acc[i] = 0.f;
  };

  int mix_next = 0, cur = 0, tab_head = -1;
  if (i_begin < i_end) {
    const int64_t win = i_begin % n_win;
    mix_next = build(win, 0);
    __syncthreads();
    const T* base = qkv + (int64_t)head_of(i_begin) * HD;
    copy(sQ, base, g.qkv_stride, tok2);
    copy(sK0, base + C, g.qkv_stride, tok2);
    copy(sV, base + 2 * C, g.qkv_stride, tok2);
    copy(sG, dout + (int64_t)head_of(i_begin) * HD, g.out_stride, tok2);
  }
  float wq[2] = {0.f, 0.f}, wk[2] = {0.f, 0.f};  // this lane's columns of the norms' weights' gradients

  for (int64_t item = i_begin; item < i_end; ++item) {
    const int64_t win = item % n_win;
    const int head = head_of(item);
    const int* tok = tok2 + cur * rows;
    const signed char* side = side2 + cur * rows;
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
    if (threadIdx.x < L) st = lse[((int64_t)win * g.nh + head) * L + threadIdx.x];
    const int mixed = __syncthreads_or(mix_next);  // (and the item before has been worked through)
    if (head != tab_head) {
      if (tab_head >= 0 && dbias_part) flush(tab_head);
      load_table(tab, bias, o.entries, head);
      tab_head = head;
    }
    cp_async_wait_all();
    __syncthreads();
    // ---- norms in place, and D
    for (int i0 = 0; i0 < 2 * rows * CH; i0 += nthreads) {
      const int i = i0 + threadIdx.x;
      const bool isk = i >= rows * CH;
      const int j = isk ? i - rows * CH : i, r = j / CH, c = j % CH;
      T* at = (isk ? sK : sQ) + r * RS + 8 * c;
      const bool live = i < 2 * rows * CH;
      uint4 y;
      const uint4 x = live ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
      const float rs = norm_chunk<T, HD>(x, (isk ? kw : qw) + 8 * c, y, nullptr);
      if (live) {
        *reinterpret_cast<uint4*>(at) = y;
        if (c == 0) (isk ? rk : rq)[r] = rs;
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
    if (next) mix_next = build((item + 1) % n_win, 1 - cur);
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
      const int at0 = o.center - (off4[k0] >> 2), at1 = o.center - (off4[k0 + 8] >> 2);
      const float* row0 = PAIR ? pair_at(tab, o.entries, at0) : tab + at0;
      const float* row1 = PAIR ? pair_at(tab, o.entries, at1) : tab + at1;
      const bool edge = mixed || warp * 16 + 16 > L;
      const uint32_t ds_at = smem_u32(sS + ((lane & 7) + (lane >> 4) * 8) * DS + warp * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll 1
      for (int qb = 0; qb < o.tiles; ++qb) {
        float s[2][4], dp[2][4];
        load_block<PAIR, 1>(s, row0, row1, off4, qb * 16, tq);
        if (edge) mask_block<true>(s, side, k0, qb * 16, tq);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 m = *reinterpret_cast<const float2*>(sub + qb * 16 + 8 * j + 2 * tq);
          const float2 d = *reinterpret_cast<const float2*>(negD + qb * 16 + 8 * j + 2 * tq);
          s[j][0] -= m.x;
          s[j][1] -= m.y;
          s[j][2] -= m.x;
          s[j][3] -= m.y;
          dp[j][0] = dp[j][2] = d.x;
          dp[j][1] = dp[j][3] = d.y;
        }
        block_product<T, HD, RS>(s, kf, sQ + qb * 16 * RS, lane);
        block_product<T, HD, RS>(dp, vf, sG + qb * 16 * RS, lane);
        if (wide) {
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
            dp[j][e] *= s[j][e];
          }
        const uint32_t p[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]),
                               pack2<T>(s[1][2], s[1][3])};
        const uint32_t ds[4] = {pack2<T>(dp[0][0], dp[0][1]), pack2<T>(dp[0][2], dp[0][3]), pack2<T>(dp[1][0], dp[1][1]),
                                pack2<T>(dp[1][2], dp[1][3])};
        // ds: (keys, queries) = (0, 0), (8, 0), (0, 8), (8, 8) -> rows of queries
        stsm_x4_t(ds_at + qb * 16 * DS * (uint32_t)sizeof(T), ds[0], ds[1], ds[2], ds[3]);
        block_add<T, HD, RS>(dv, p, sG + qb * 16 * RS, lane);
        block_add<T, HD, RS>(dk, ds, sQ + qb * 16 * RS, lane);
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
      norm_backward<T, HD>(dk, raw, kw, 0.69314718055994530942f, rk[k0], rk[k0 + 8], k0 < L, k0 + 8 < L, wk, lane);
      __syncwarp();
      stage_live<T, HD, RS>(st_rows, dk, warp * 16, L, lane);
      __syncwarp();
      store_rows<T, HD, RS>(st_rows, dst + C, g.qkv_stride, tok, warp * 16, L, lane);
    }
    __syncthreads();
    // ---- the next item's rows
    const int64_t after = item + 1;
    const T* base_n = qkv + (int64_t)head_of(after) * HD;
    const int* tok_n = tok2 + (1 - cur) * rows;
    if (next) {
      copy(sQ, base_n, g.qkv_stride, tok_n);
      if (k_bufs > 1) copy(sK0 + (1 - cur) * rows * RS, base_n + C, g.qkv_stride, tok_n);
      copy(sV, base_n + 2 * C, g.qkv_stride, tok_n);
      copy(sG, dout + (int64_t)head_of(after) * HD, g.out_stride, tok_n);
    }
    // ---- B
    float dq[CH][4];
#pragma unroll
    for (int d = 0; d < CH; ++d) dq[d][0] = dq[d][1] = dq[d][2] = dq[d][3] = 0.f;
    uint32_t raw[KS][4];
    raw_rows<T, HD>(raw, base, g.qkv_stride, tok, warp * 16, L, lane);
    const uint32_t a_at = smem_u32(sS + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * DS + (lane >> 4) * 8);
#pragma unroll 1
    for (int kb = 0; kb < o.tiles; ++kb) {
      uint32_t a[4];
      ldsm_x4(a_at + kb * 32, a[0], a[1], a[2], a[3]);
      block_add<T, HD, RS>(dq, a, sK + kb * 16 * RS, lane);
    }
    if (dbias_part) {
      // tasks of `width` entries: acc[dt][da][bi][bj ..]
      const int tasks = bs.entries / bs.width, step = bs.sa * (DS + 1);
      for (int e = threadIdx.x; e < tasks; e += nthreads) {
        const int e1 = quick_div(e, bs.div_b), bj = (e - e1 * (bs.nb / bs.width)) * bs.width;
        const int e2 = quick_div(e1, bs.div_b2), bi = e1 - e2 * bs.nb;
        const int e3 = quick_div(e2, bs.div_a), da = e2 - e3 * (2 * bs.na - 1) - (bs.na - 1), dt = e3 - (o.nt - 1);
        const int n = bs.na - abs(da);
        float s0 = 0.f, s1 = 0.f;
        for (int t = max(dt, 0); t < o.nt + min(dt, 0); ++t) {
          const int q = t * o.ns * o.nf + max(da, 0) * bs.sa + bi * bs.sb;
          const int k = (t - dt) * o.ns * o.nf + max(-da, 0) * bs.sa + bj * bs.sb;
          const T* p = sS + q * DS + k;
#pragma unroll 4
          for (int i = 0; i < n; ++i) {
            if (PAIR) {
              float f[2];
              unpack2(*reinterpret_cast<const uint32_t*>(p + i * step), f, T());
              s0 += f[0];
              s1 += f[1];
            } else {
              s0 += to_f(p[i * step]);
            }
          }
        }
        if (PAIR) {
          float2* at = reinterpret_cast<float2*>(acc + 2 * e);
          const float2 old = *at;
          *at = make_float2(old.x + s0, old.y + s1);
        } else {
          acc[e] += s0;
        }
      }
    }
    __syncthreads();  // k's rows have been read: dQ leaves by way of this warp's
    {
      const int q0 = warp * 16 + gq;
      T* st_rows = sK + warp * 16 * RS;
      // dL/dq' = ln 2 dS k', and q' is scale log2 e times the norm's result
      norm_backward<T, HD>(dq, raw, qn, g.scale, rq[q0], rq[q0 + 8], q0 < L, q0 + 8 < L, wq, lane);
      stage_live<T, HD, RS>(st_rows, dq, warp * 16, L, lane);
      __syncwarp();
      store_rows<T, HD, RS>(st_rows, dqkv + (int64_t)head * HD, g.qkv_stride, tok, warp * 16, L, lane);
    }
    if (next && k_bufs == 1) {
      __syncthreads();
      copy(sK0, base_n + C, g.qkv_stride, tok_n);
    }
    cur = 1 - cur;
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

template <typename T, int HD, bool PAIR>
cudaError_t launch_fwd(const void* qkv, const AttnBias& bias, const float* norms, void* out, float* lse, const AttnGeom& g,
                       cudaStream_t s) {
  const Order o = order_of(g, bias);
  FwdSmem<T, HD> S;
  const size_t smem = S.carve(nullptr, o);
  auto k = fwd_kernel<T, HD, PAIR>;
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
  if (items > INT32_MAX) return cudaErrorInvalidValue;
  k<<<(unsigned)items, 32 * std::min(o.tiles, kFwdWarps), smem, s>>>((const T*)qkv, bias, norms, (T*)out,
                                                                    reinterpret_cast<float2*>(lse), g);
  return cudaGetLastError();
}

// How many blocks the device holds at once, and whether keys have two buffers: where that costs no block of an SM
template <typename T, int HD, bool PAIR>
AttnBiasPlan plan_bwd(const AttnGeom& g, const AttnBias& bias, bool dbias, int sms) {
  const Order o = order_of(g, bias);
  const int entries = dbias ? sums_of<PAIR>(o).entries : 0;
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

template <typename T, int HD, bool PAIR>
cudaError_t launch_bwd(const void* qkv, const AttnBias& bias, const float* norms, const void* out, const void* dout,
                       const float* lse, void* dqkv, float* dqw_part, float* dkw_part, float* dbias_part,
                       const AttnBiasPlan& plan, const AttnGeom& g, cudaStream_t s) {
  const Order o = order_of(g, bias);
  BwdSmem<T, HD> S;
  const size_t smem = S.carve(nullptr, o, dbias_part ? sums_of<PAIR>(o).entries : 0, plan.k_bufs);
  auto k = bwd_kernel<T, HD, PAIR>;
  NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  k<<<plan.blocks, 32 * o.tiles, smem, s>>>((const T*)qkv, bias, norms, (const T*)out, (const T*)dout,
                                            reinterpret_cast<const float2*>(lse), (T*)dqkv, dqw_part, dkw_part, dbias_part,
                                            plan.k_bufs, g);
  return cudaGetLastError();
}

// f(type, head_dim, pairs) of the call's; WIDE: head_dim 128 too
template <bool WIDE, typename F>
auto dispatch(const AttnGeom& g, const AttnBias& b, int dtype, F f) {
  const auto hd = [&](auto t, auto pair) {
    using I16 = std::integral_constant<int, 16>;
    using I32 = std::integral_constant<int, 32>;
    using I64 = std::integral_constant<int, 64>;
    if constexpr (WIDE)
      if (g.hd == 128) return f(t, std::integral_constant<int, 128>(), pair);
    return g.hd == 16 ? f(t, I16(), pair) : g.hd == 32 ? f(t, I32(), pair) : f(t, I64(), pair);
  };
  const auto type = [&](auto pair) { return dtype == kBF16 ? hd(__nv_bfloat16(), pair) : hd(__half(), pair); };
  return b.pair ? type(std::true_type()) : type(std::false_type());
}

}  // namespace attn_bias

static bool attn_bias_ok(const AttnGeom& g, int dtype) {
  return (g.hd == 16 || g.hd == 32 || g.hd == 64 || g.hd == 128) && (dtype == kBF16 || dtype == kF16) && g.T > 0 &&
         g.wh > 0 && g.ww > 0 && (int64_t)g.T * g.wh * g.ww <= 192 && g.H % g.wh == 0 && g.W % g.ww == 0 &&
         (int64_t)g.B * g.T * g.H * g.W < INT32_MAX;
}

// The fast extent of the tokens' order: one that is even, so that the kernels read entries by pairs (64800 tokens x 16
// heads: see DESIGN), if the sums of its pairs leave room (at most 6144); of two, the one with fewer of them.  Otherwise
// longitude, entries one by one, and a pitch that puts a warp's consecutive tokens on consecutive banks where there is room.
AttnBias attn_bias_layout(const AttnGeom& g) {
  AttnBias b{};
  int64_t best = 6145;
  if (g.hd != 128)
    for (int y = 0; y < 2; ++y) {
      const int nf = y ? g.wh : g.ww, ns = y ? g.ww : g.wh;
      const int64_t sums = (int64_t)(2 * g.T - 1) * (2 * ns - 1) * nf * nf;
      if (nf % 2 == 0 && sums < best) {
        best = sums;
        b.pair = 1;
        b.y_fast = y;
      }
    }
  const int nf = b.y_fast ? g.wh : g.ww, ns = b.y_fast ? g.ww : g.wh, rows = (2 * g.T - 1) * (2 * ns - 1);
  b.pitch = 2 * nf - 1;
  if (b.pair) {
    b.pitch = 2 * nf;
  } else {
    while (b.pitch % 32 != nf % 32) ++b.pitch;
    if (rows * b.pitch > 1600) b.pitch = 2 * nf - 1;
  }
  b.stride = (4 + rows * b.pitch + 3) / 4 * 4;
  return b;
}

cudaError_t attn_bias_prepare(const AnyMatrix& table, const AnyMatrix& qw, const AnyMatrix& kw, const AttnGeom& g,
                              const AttnBias& b, float* tab, cudaStream_t s) {
  attn_bias::prepare_kernel<<<g.nh + 1, 256, 0, s>>>(table, qw, kw, b, g.nh, g.hd, 2 * g.T - 1, 2 * g.wh - 1, 2 * g.ww - 1,
                                                     tab);
  return cudaGetLastError();
}

cudaError_t attn_bias_fwd(const void* qkv, const AttnBias& bias, const float* norms, void* out, float* lse,
                          const AttnGeom& g, int dtype, cudaStream_t s) {
  if (!attn_bias_ok(g, dtype)) return cudaErrorInvalidValue;
  return attn_bias::dispatch<true>(g, bias, dtype, [&](auto t, auto hd, auto pair) {
    return attn_bias::launch_fwd<decltype(t), hd(), pair()>(qkv, bias, norms, out, lse, g, s);
  });
}

AttnBiasPlan attn_bias_plan(const AttnGeom& g, const AttnBias& bias, int dtype, bool dbias, int sms) {
  if (g.hd == 128) {
    const int64_t items = (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww) * g.nh;
    return {0, 0, items, items};
  }
  return attn_bias::dispatch<false>(g, bias, dtype, [&](auto t, auto hd, auto pair) {
    return attn_bias::plan_bwd<decltype(t), hd(), pair()>(g, bias, dbias, sms);
  });
}

cudaError_t attn_bias_bwd(const void* qkv, const AttnBias& bias, const float* norms, const void* out, const void* dout,
                          const float* lse, void* dqkv, float* dqw_part, float* dkw_part, float* dbias_part,
                          const AttnBiasPlan& plan, const AttnGeom& g, int dtype, cudaStream_t s) {
  if (!attn_bias_ok(g, dtype)) return cudaErrorInvalidValue;
  if (g.hd == 128)
    return window_attn_bwd(qkv, norms, norms + g.hd, out, dout, lse, dqkv, dqw_part, dkw_part, g, dtype, s, bias, dbias_part);
  return attn_bias::dispatch<false>(g, bias, dtype, [&](auto t, auto hd, auto pair) {
    return attn_bias::launch_bwd<decltype(t), hd(), pair()>(qkv, bias, norms, out, dout, lse, dqkv, dqw_part, dkw_part,
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
  p.buckets = (2 * g.T - 1) * (2 * g.wh - 1) * (2 * g.ww - 1);
  p.hd = g.hd;
  attn_bias::grad_kernel<<<dim3((std::max(p.buckets, g.hd) + 31) / 32, g.nh + 2), 1024, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace nsw
