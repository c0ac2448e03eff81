// The norms before and after a residual connection, fused with its gate and scale:
//
//   s = c skip + gate * (y / rms(y)) * wp,    n = (s / rms(s)) * wn,    rms(v) = sqrt(mean(v^2) + eps)
//
// and its gradient, in one pass over the rows: with yh = y / rms(y), sh = s / rms(s), a = dn * wn,
//   d     = ds + (a - sh mean(a sh)) / rms(s)                    (gradient of s)
//   dskip = c d,   b = d gate wp,   dy = (b - yh mean(b yh)) / rms(y)
//   dwn = sum dn sh,   Q = sum over a sample's rows of d yh,   dgate = wp Q,   dwp = sum over samples gate Q
//
// Bound by memory: the forward reads two rows and writes two, the backward reads four (it recomputes s from
// y and skip in fp32 instead of reading the rounded stream) and writes two; everything in between stays in
// registers.  A row belongs to WPR warps, a lane holds NV groups of eight elements of it.  Rows that do not begin on
// 16 bytes (a width that is no multiple of eight) are still accessed in aligned groups: a lane's group then starts
// up to seven elements before the row, what is not the row's is masked, and the two groups at a row's ends are stored
// in pieces.  A row group's rows are eight rows apart, so its shift stays the same and the parameters
// and sums can stay in its lanes' registers.  The row sums go
// through shuffles and, for WPR > 1, one shared-memory exchange behind a barrier of the row's warps.  The
// sums over rows (Q, dwn) stay in the lanes' registers over all rows of a block, then are added over the
// block's rows in a fixed order and written as one partial per block; a second kernel adds the partials in
// block order, so results repeat bit for bit.  All arithmetic is fp32; only the outputs are rounded.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace nsw {
namespace ng {

struct Params {
  const void *y, *skip, *ds, *dn;
  void *stream, *normed, *dy, *dskip;
  const float *wp, *gate, *wn;  // gate, wn: null for none
  int64_t gate_stride;          // elements from one sample's gate to the next
  float* part;                  // backward: [samples][blocks][2][n] partials (Q, dwn)
  int64_t rows, total;          // rows of one sample, elements of all
  int n;
  float c, eps, inv_n;
};

// how rows are accessed: 2-byte accesses, 16-byte ones, or 16-byte ones of rows that begin anywhere
enum Access { kScalar = 0, kVec = 1, kShift = 2 };

// the elements a lane holds: contiguous groups of eight (16-byte accesses), or strided single elements
// where the rows are not 16-byte aligned (coalesced 2-byte accesses)
template <bool VEC, int GL>
__device__ __forceinline__ int elem(int v, int j, int gl) {
  return VEC ? (v * GL + gl) * 8 + j : (v * 8 + j) * GL + gl;
}

template <typename T, bool VEC, int GL>
__device__ __forceinline__ uint4 load_row(const T* row, int v, int gl, int n) {
  uint4 r = make_uint4(0, 0, 0, 0);
  if (VEC) {
    const int e = elem<VEC, GL>(v, 0, gl);
    if (e < n) r = __ldcs(reinterpret_cast<const uint4*>(row + e));
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = elem<VEC, GL>(v, j, gl);
      if (e < n) w[j >> 1] |= (uint32_t)p[e] << (16 * (j & 1));
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}
template <typename T, bool VEC, int GL>
__device__ __forceinline__ void store_row(T* row, int v, int gl, int n, const float* f) {
  if (VEC) {
    const int e = elem<VEC, GL>(v, 0, gl);
    if (e < n) __stcs(reinterpret_cast<uint4*>(row + e), pack8<T>(f));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = elem<VEC, GL>(v, j, gl);
      if (e < n) row[e] = from_f<T>(f[j]);
    }
  }
}
// a parameter vector's elements of this lane (`none` past the end and for a null pointer)
template <bool VEC, int GL>
__device__ __forceinline__ void load_vec(const float* p, int v, int gl, int n, float none, float* f) {
  if constexpr (VEC) {
    const int e = elem<VEC, GL>(v, 0, gl);
    float4 a = make_float4(none, none, none, none), b = a;
    if (p && e < n) {
      a = __ldg(reinterpret_cast<const float4*>(p + e));
      b = __ldg(reinterpret_cast<const float4*>(p + e) + 1);
    }
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = elem<VEC, GL>(v, j, gl);
      f[j] = p && e < n ? __ldg(p + e) : none;
    }
  }
}

// Two fp32 values in one register pair: the packed forms of add, multiply and fma halve the instructions of the
// backward, which they bound (64800 x 1024: 164 us with scalar ones, 142 us packed)
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split2(F2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  float x, y;
  split2(a, x, y);
  return x + y;
}
template <typename T>
__device__ __forceinline__ void widen(const uint4 u, F2* f) {
  float x[8];
  unpack8<T>(u, x);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack2(x[2 * j], x[2 * j + 1]);
}
__device__ __forceinline__ void narrow(const F2* f, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) split2(f[j], x[2 * j], x[2 * j + 1]);
}

// sums of K values over the row's warps (every lane gets them); `slot` names the exchange buffer: two
// consecutive exchanges use different slots, so one barrier each is enough
template <int WPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[WPR][2], int slot, int bar) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if (WPR > 1) {
    const int w = (threadIdx.x >> 5) % WPR;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[slot][w][k] = v[k];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(32 * WPR) : "memory");
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = red[slot][0][k];
#pragma unroll
      for (int i = 1; i < WPR; ++i) v[k] += red[slot][i][k];
    }
  }
}

template <typename T, bool VEC, int WPR, int NV>
__global__ void __launch_bounds__(WPR > 8 ? 32 * WPR : 256) fwd_kernel(const Params p) {
  constexpr int GL = 32 * WPR;
  constexpr int RPB = WPR > 8 ? 1 : 8 / WPR;  // rows a block works on at a time
  __shared__ float red[RPB][2][WPR][2];
  const int rg = threadIdx.x / GL, gl = threadIdx.x % GL;
  const int64_t sample = blockIdx.y;
  const float* gate = p.gate ? p.gate + sample * p.gate_stride : nullptr;
  for (int64_t r = (int64_t)blockIdx.x * RPB + rg; r < p.rows; r += (int64_t)gridDim.x * RPB) {
    const int64_t at = (sample * p.rows + r) * p.n;
    const T* y = reinterpret_cast<const T*>(p.y) + at;
    const T* k = reinterpret_cast<const T*>(p.skip) + at;
    uint4 yr[NV], kr[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) yr[v] = load_row<T, VEC, GL>(y, v, gl, p.n);
#pragma unroll
    for (int v = 0; v < NV; ++v) kr[v] = load_row<T, VEC, GL>(k, v, gl, p.n);
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[8];
      unpack8<T>(yr[v], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) q[0] = fmaf(f[j], f[j], q[0]);
    }
    row_sum<WPR>(q, red[rg], 0, 1 + rg);
    const float ry = rsqrtf(q[0] * p.inv_n + p.eps);
    float s[NV][8];
    q[0] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[8], w[8], g[8];
      unpack8<T>(yr[v], f);
      unpack8<T>(kr[v], s[v]);
      load_vec<VEC, GL>(p.wp, v, gl, p.n, 0.f, w);
      load_vec<VEC, GL>(gate, v, gl, p.n, 1.f, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[v][j] = fmaf(p.c, s[v][j], f[j] * ry * (w[j] * g[j]));
        q[0] = fmaf(s[v][j], s[v][j], q[0]);
      }
      store_row<T, VEC, GL>(reinterpret_cast<T*>(p.stream) + at, v, gl, p.n, s[v]);
    }
    row_sum<WPR>(q, red[rg], 1, 1 + rg);  // also without a second norm: it separates two uses of slot 0
    if (p.normed) {
      const float rs = rsqrtf(q[0] * p.inv_n + p.eps);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float w[8];
        load_vec<VEC, GL>(p.wn, v, gl, p.n, 0.f, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[v][j] *= rs * w[j];
        store_row<T, VEC, GL>(reinterpret_cast<T*>(p.normed) + at, v, gl, p.n, s[v]);
      }
    }
  }
}

// `bytes` (0 to 16) into 16 bytes of shared memory behind the thread's back, the rest zeros
__device__ __forceinline__ void copy_async(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// Rows ahead that operands are copied (kRing - 1) where a lane holds one group; each thread reads back only what it
// copied itself, so there is no barrier.
constexpr int kRing = 4;
// as many rows as eight warps hold
constexpr int block_threads(int warps) { return 32 * warps * (warps > 8 ? 1 : 8 / warps); }
// Blocks an SM of the backward: with three or six warps a row a third one fits (64800 x 1536: 209 us, 230 with two),
// but the shifted rows' masks and places do not fit its 96 registers (30000 x 1301: 142 us, 126 with two).
constexpr int bwd_blocks(int mode, int warps) {
  return warps > 8 ? 1 : mode == kVec && (warps == 3 || warps == 6) ? 3 : 2;
}
template <int MODE, int WPR, int NV>
constexpr bool use_ring() {
  return MODE != kScalar && WPR <= 8 && NV == 1;
}

// A lane's group of eight elements in rows that begin `o` elements after a 16-byte boundary
template <int MODE>
struct Group {
  int e0, n;
  uint4 mask;
  int i2, i4, i8;  // a row's end in this group leaves as at most one store of 2, 4 and 8 bytes: their places, or -1
  __device__ __forceinline__ Group(int gl, int o, int n) : e0(8 * gl - o), n(n) {
    const int a = -e0, b = n - e0;  // elements before the row, or up to its end (n >= 8: never both in one group)
    i2 = i4 = i8 = -1;
    if (a > 0 && a < 8) {
      const int w = (a + 1) >> 1;
      if (a & 1) i2 = a;
      if (w & 1) i4 = w;
      if (w <= 2) i8 = 1;
    } else if (b > 0 && b < 8) {
      if (b & 1) i2 = b - 1;
      if (b & 2) i4 = (b & 4) >> 1;
      if (b & 4) i8 = 0;
    }
    uint32_t m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = (has(2 * j) ? 0xffffu : 0u) | (has(2 * j + 1) ? 0xffff0000u : 0u);
    mask = make_uint4(m[0], m[1], m[2], m[3]);
  }
  __device__ __forceinline__ bool has(int j) const { return e0 + j >= 0 && e0 + j < n; }
  __device__ __forceinline__ uint4 own(uint4 u) const {
    if (MODE == kShift) u = make_uint4(u.x & mask.x, u.y & mask.y, u.z & mask.z, u.w & mask.w);
    return u;
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float* f) const {
    const uint4 u = pack8<T>(f);
    T* d = row + e0;
    if (e0 >= 0 && e0 + 8 <= n) {
      __stcs(reinterpret_cast<uint4*>(d), u);
    } else if (MODE == kShift) {
      const auto word = [&](int i) { return i < 2 ? (i ? u.y : u.x) : (i == 2 ? u.z : u.w); };
      if (i2 >= 0) reinterpret_cast<uint16_t*>(d)[i2] = (uint16_t)(word(i2 >> 1) >> (16 * (i2 & 1)));
      if (i4 >= 0) reinterpret_cast<uint32_t*>(d)[i4] = word(i4);
      if (i8 >= 0) reinterpret_cast<uint2*>(d)[i8] = i8 ? make_uint2(u.z, u.w) : make_uint2(u.x, u.y);
    }
  }
  __device__ __forceinline__ void load_vec(const float* p, float none, float* f) const {
    if (MODE == kVec) {
      float4 a = make_float4(none, none, none, none), b = a;
      if (p && e0 < n) {
        a = __ldg(reinterpret_cast<const float4*>(p + e0));
        b = __ldg(reinterpret_cast<const float4*>(p + e0) + 1);
      }
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = p && has(j) ? __ldg(p + e0 + j) : none;
    }
  }
  // the group at element `at` of a tensor of `total` (a multiple of eight; nothing past its end is read)
  static __device__ __forceinline__ int bytes(int64_t at, int64_t total) {
    return MODE == kShift && total - at < 8 ? 2 * (int)(total - at) : 16;
  }
};

// The forward with the operands of three rows ahead in shared memory.  64800 x 1024: 83 us, the measured copy rate;
// 92 with a row's operands loaded when it begins and 16 elements a lane.  20001 x 1001 twice: 62 us; 92 with 2-byte
// accesses.
constexpr int kFwdBlocks = 4;  // at most, an SM
template <typename T, int MODE, int WPR>
__global__ void __launch_bounds__(block_threads(WPR), kFwdBlocks) fwd_ring_kernel(const Params p) {
  constexpr int GL = 32 * WPR, NT = block_threads(WPR);
  constexpr int RPB = 8 / WPR;
  __shared__ __align__(16) uint4 ring_all[kRing * 2 * NT];
  __shared__ float red[RPB][2][WPR][2];
  const int rg = threadIdx.x / GL, gl = threadIdx.x % GL;
  const int64_t sample = blockIdx.y, step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + rg;
  const int o = MODE == kShift ? (int)(((sample * p.rows + r) * p.n) & 7) : 0;
  const Group<MODE> g(gl, o, p.n);
  uint4* ring = ring_all + threadIdx.x;
  auto copy = [&](int64_t row, int slot) {
    const bool ok = row < p.rows && g.e0 < p.n;
    const int64_t at = ok ? (sample * p.rows + row) * p.n + g.e0 : 0;
    const int bytes = ok ? Group<MODE>::bytes(at, p.total) : 0;
    copy_async(ring + (slot * 2 + 0) * NT, reinterpret_cast<const T*>(p.y) + at, bytes);
    copy_async(ring + (slot * 2 + 1) * NT, reinterpret_cast<const T*>(p.skip) + at, bytes);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < kRing - 1; ++k) copy(r + k * step, k);
  F2 gw[4], wn[4];  // gate * wp, wn
  {
    float a[8], b[8];
    g.load_vec(p.wp, 0.f, a);
    g.load_vec(p.gate ? p.gate + sample * p.gate_stride : nullptr, 1.f, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) gw[j] = pack2(a[2 * j] * b[2 * j], a[2 * j + 1] * b[2 * j + 1]);
    g.load_vec(p.wn, 0.f, a);
#pragma unroll
    for (int j = 0; j < 4; ++j) wn[j] = pack2(a[2 * j], a[2 * j + 1]);
  }
  const F2 zero = pack2(0.f, 0.f), c2 = pack2(p.c, p.c);
  int slot = 0;
  for (; r < p.rows; r += step) {
    const int64_t at = (sample * p.rows + r) * p.n;
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    const uint4 yr = g.own(ring[(slot * 2 + 0) * NT]), kr = g.own(ring[(slot * 2 + 1) * NT]);
    copy(r + (kRing - 1) * step, (slot + kRing - 1) % kRing);
    slot = (slot + 1) % kRing;
    F2 y[4], s[4], t = zero;
    widen<T>(yr, y);
    widen<T>(kr, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) t = fma2(y[j], y[j], t);
    float q[1] = {sum2(t)};
    row_sum<WPR>(q, red[rg], 0, 1 + rg);
    const float ry = rsqrtf(q[0] * p.inv_n + p.eps);
    const F2 ry2 = pack2(ry, ry);
    t = zero;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = fma2(c2, s[j], mul2(mul2(y[j], ry2), gw[j]));
      t = fma2(s[j], s[j], t);
    }
    float f[8];
    narrow(s, f);
    g.store(reinterpret_cast<T*>(p.stream) + at, f);
    q[0] = sum2(t);
    row_sum<WPR>(q, red[rg], 1, 1 + rg);  // also without a second norm: it separates two uses of slot 0
    if (p.normed) {
      const float rs = rsqrtf(q[0] * p.inv_n + p.eps);
      const F2 rs2 = pack2(rs, rs);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = mul2(s[j], mul2(rs2, wn[j]));
      narrow(s, f);
      g.store(reinterpret_cast<T*>(p.normed) + at, f);
    }
  }
}

// What bounds it is the bytes in flight and the latency of three row sums a row.  64800 x 1024: 245 us with 16 elements a
// lane and no prefetch, 167 with 8 and the next row's operands in registers, 142 with packed arithmetic, 132 with
// the operands of three rows ahead in shared memory; x 768 with four warps a row 123, with three 114.  20001 x 1001
// twice: 105 us; 201 with 2-byte accesses, 120 with a row's ends stored element by element.
template <typename T, int MODE, int WPR, int NV>
__global__ void __launch_bounds__(block_threads(WPR), bwd_blocks(MODE, WPR)) bwd_kernel(const Params p) {
  constexpr bool VEC = MODE != kScalar;
  constexpr bool kUseRing = use_ring<MODE, WPR, NV>();
  constexpr int GL = 32 * WPR, NT = block_threads(WPR);
  constexpr int RPB = WPR > 8 ? 1 : 8 / WPR;
  extern __shared__ __align__(16) float sums[];  // [2][n], then the ring [kRing][4][threads] of 16 bytes
  __shared__ float red[RPB][3][WPR][2];
  const int rg = threadIdx.x / GL, gl = threadIdx.x % GL;
  const int64_t sample = blockIdx.y;
  const float* gate = p.gate ? p.gate + sample * p.gate_stride : nullptr;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r = (int64_t)blockIdx.x * RPB + rg;
  const int o = MODE == kShift ? (int)(((sample * p.rows + r) * p.n) & 7) : 0;
  const Group<MODE> grp(gl, o, p.n);  // (of the ring's variants)
  const auto vec = [&](const float* q, int v, float none, float* f) {
    if constexpr (kUseRing)
      grp.load_vec(q, none, f);
    else
      load_vec<VEC, GL>(q, v, gl, p.n, none, f);
  };
  // q null: not wanted.  The predicated form has no branch (20000 x 3000: 215 us; 233 with one); 32 warps a row have no
  // registers left for a test (3000 x 16384: 519 us; 587 with either).
  const auto store = [&](void* q, int64_t at, int v, const float* f) {
    if constexpr (kUseRing) {
      if (q) grp.store(reinterpret_cast<T*>(q) + at, f);
    } else if constexpr (VEC) {
      store_row<T, VEC, GL>(reinterpret_cast<T*>(q) + at, v, gl, WPR == 32 || q ? p.n : 0, f);
    } else {
      if (WPR == 32 || q) store_row<T, VEC, GL>(reinterpret_cast<T*>(q) + at, v, gl, p.n, f);
    }
  };
  F2 gw[NV][4], wn[NV][4], aq[NV][4], aw[NV][4];  // gate * wp, wn, and the sums of d yh and dn sh
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float g[8], w[8];
    vec(p.wp, v, 0.f, w);
    vec(gate, v, 1.f, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) gw[v][j] = pack2(w[2 * j] * g[2 * j], w[2 * j + 1] * g[2 * j + 1]);
    vec(p.wn, v, 0.f, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      wn[v][j] = pack2(w[2 * j], w[2 * j + 1]);
      aq[v][j] = aw[v][j] = pack2(0.f, 0.f);
    }
  }
  uint4 nxt[4][NV];  // the next row's y, skip, ds, dn
  auto fetch = [&](int64_t r) {
    const int64_t at = (sample * p.rows + r) * p.n;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      nxt[0][v] = load_row<T, VEC, GL>(reinterpret_cast<const T*>(p.y) + at, v, gl, p.n);
      nxt[1][v] = load_row<T, VEC, GL>(reinterpret_cast<const T*>(p.skip) + at, v, gl, p.n);
      nxt[2][v] = nxt[3][v] = make_uint4(0, 0, 0, 0);
      if (p.ds) nxt[2][v] = load_row<T, VEC, GL>(reinterpret_cast<const T*>(p.ds) + at, v, gl, p.n);
      if (p.dn) nxt[3][v] = load_row<T, VEC, GL>(reinterpret_cast<const T*>(p.dn) + at, v, gl, p.n);
    }
  };
  uint4* ring = reinterpret_cast<uint4*>(sums + ((2 * p.n + 3) & ~3)) + threadIdx.x;
  auto copy = [&](int64_t row, int slot) {
    const bool ok = row < p.rows && grp.e0 < p.n;
    const int64_t at = ok ? (sample * p.rows + row) * p.n + grp.e0 : 0;
    const int bytes = ok ? Group<MODE>::bytes(at, p.total) : 0;
    const void* src[4] = {p.y, p.skip, p.ds, p.dn};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      copy_async(ring + (slot * 4 + k) * NT, reinterpret_cast<const T*>(src[k] ? src[k] : p.y) + at, src[k] ? bytes : 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int slot = 0;
  if (kUseRing) {
#pragma unroll
    for (int k = 0; k < kRing - 1; ++k) copy(r + k * step, k);
  } else if (r < p.rows) {
    fetch(r);
  }
  for (; r < p.rows; r += step) {
    const int64_t at = (sample * p.rows + r) * p.n;
    uint4 yr[NV], kr[NV], dsr[NV], dnr[NV];
    if (kUseRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      yr[0] = grp.own(ring[(slot * 4 + 0) * NT]);
      kr[0] = grp.own(ring[(slot * 4 + 1) * NT]);
      dsr[0] = grp.own(ring[(slot * 4 + 2) * NT]);
      dnr[0] = grp.own(ring[(slot * 4 + 3) * NT]);
      copy(r + (kRing - 1) * step, (slot + kRing - 1) % kRing);
      slot = (slot + 1) % kRing;
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        yr[v] = nxt[0][v];
        kr[v] = nxt[1][v];
        dsr[v] = nxt[2][v];
        dnr[v] = nxt[3][v];
      }
      if (r + step < p.rows) fetch(r + step);
    }
    const F2 zero = pack2(0.f, 0.f), c2 = pack2(p.c, p.c);
    F2 y[NV][4], t = zero;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      widen<T>(yr[v], y[v]);
#pragma unroll
      for (int j = 0; j < 4; ++j) t = fma2(y[v][j], y[v][j], t);
    }
    float q1[1] = {sum2(t)};
    row_sum<WPR>(q1, red[rg], 0, 1 + rg);
    const float ry = rsqrtf(q1[0] * p.inv_n + p.eps);
    const F2 ry2 = pack2(ry, ry);
    F2 s[NV][4], an[NV][4], ss = zero, as = zero;  // s, dn, and the sums of s^2 and dn wn s
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      widen<T>(kr[v], s[v]);
      widen<T>(dnr[v], an[v]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[v][j] = mul2(y[v][j], ry2);  // from here: yh
        s[v][j] = fma2(c2, s[v][j], mul2(y[v][j], gw[v][j]));
        ss = fma2(s[v][j], s[v][j], ss);
        as = fma2(mul2(an[v][j], wn[v][j]), s[v][j], as);
      }
    }
    float q2[2] = {sum2(ss), sum2(as)};
    row_sum<WPR>(q2, red[rg], 1, 1 + rg);
    const float rs = rsqrtf(q2[0] * p.inv_n + p.eps);
    const float m = q2[1] * rs * p.inv_n;  // mean(a sh)
    const F2 rs2 = pack2(rs, rs), m2 = pack2(-m, -m);
    F2 by = zero;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      F2 d[4], o[4];
      widen<T>(dsr[v], d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 sh = mul2(s[v][j], rs2);
        aw[v][j] = fma2(an[v][j], sh, aw[v][j]);
        d[j] = fma2(rs2, fma2(sh, m2, mul2(an[v][j], wn[v][j])), d[j]);
        const F2 dq = mul2(d[j], y[v][j]);
        aq[v][j] = add2(aq[v][j], dq);
        by = fma2(gw[v][j], dq, by);
        s[v][j] = mul2(d[j], gw[v][j]);  // from here: b
        o[j] = mul2(c2, d[j]);
      }
      float f[8];
      narrow(o, f);
      store(p.dskip, at, v, f);
    }
    float q3[1] = {sum2(by)};
    row_sum<WPR>(q3, red[rg], 2, 1 + rg);
    const float my = q3[0] * p.inv_n;  // mean(b yh)
    const F2 my2 = pack2(-my, -my);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      F2 o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = mul2(ry2, fma2(y[v][j], my2, s[v][j]));
      float f[8];
      narrow(o, f);
      store(p.dy, at, v, f);
    }
  }
  // the block's sums: its row groups in order
  for (int g = 0; g < RPB; ++g) {
    if (rg == g) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float q[8], w[8];
        narrow(aq[v], q);
        narrow(aw[v], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = kUseRing ? grp.e0 + j : elem<VEC, GL>(v, j, gl);
          if (e >= 0 && e < p.n) {
            sums[e] = g ? sums[e] + q[j] : q[j];
            sums[p.n + e] = g ? sums[p.n + e] + w[j] : w[j];
          }
        }
      }
    }
    __syncthreads();
  }
  float* part = p.part + (sample * gridDim.x + blockIdx.x) * 2 * p.n;
  for (int e = threadIdx.x; e < 2 * p.n; e += blockDim.x) part[e] = sums[e];
}

// dwn[e] = sum of all partials; per sample Q[e]; dgate = wp Q (gate_stride > 0: of each sample, else summed
// over the one "sample"), dwp = sum gate Q.  32 columns by 32 rows of threads a block; rows in a fixed order.
__global__ void __launch_bounds__(1024) finish_kernel(const float* __restrict__ part, int64_t samples, int64_t blocks, int n,
                              const float* __restrict__ wp, const float* __restrict__ gate, int64_t gate_stride,
                              float* dwp, float* dgate, float* dwn) {
  __shared__ float acc[2][32][33];
  const int c = threadIdx.x & 31, t = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + c;
  float wn_sum = 0.f, wp_sum = 0.f;
  for (int64_t s = 0; s < samples; ++s) {
    float q = 0.f, w = 0.f;
    if (e < n)
      for (int64_t b = t; b < blocks; b += 32) {
        const float* p = part + (s * blocks + b) * 2 * n;
        q += p[e];
        w += p[n + e];
      }
    acc[0][t][c] = q;
    acc[1][t][c] = w;
    __syncthreads();
    if (t == 0 && e < n) {
      q = acc[0][0][c];
      w = acc[1][0][c];
      for (int i = 1; i < 32; ++i) {
        q += acc[0][i][c];
        w += acc[1][i][c];
      }
      wn_sum += w;
      wp_sum += q * (gate ? gate[s * gate_stride + e] : 1.f);
      if (dgate) dgate[s * gate_stride + e] = q * wp[e];
    }
    __syncthreads();
  }
  if (t == 0 && e < n) {
    dwp[e] = wp_sum;
    if (dwn) dwn[e] = wn_sum;
  }
}

template <typename T, bool VEC, int WPR, int NV>
static cudaError_t launch_fwd(const Params& p, dim3 grid, cudaStream_t s) {
  fwd_kernel<T, VEC, WPR, NV><<<grid, WPR > 8 ? 32 * WPR : 256, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int MODE, int WPR>
static cudaError_t launch_ring(const Params& p, dim3 grid, cudaStream_t s) {
  fwd_ring_kernel<T, MODE, WPR><<<grid, block_threads(WPR), 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int MODE, int WPR, int NV>
static cudaError_t launch_bwd(const Params& p, dim3 grid, cudaStream_t s) {
  auto k = bwd_kernel<T, MODE, WPR, NV>;
  const size_t smem = sizeof(float) * ((2 * p.n + 3) & ~3) + (use_ring<MODE, WPR, NV>() ? kRing * 4 * block_threads(WPR) * 16 : 0);
  if (smem + 1024 > 48 * 1024)  // (with the kernel's own at most 768 bytes)
    NSW_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  k<<<grid, block_threads(WPR), smem, s>>>(p);
  return cudaGetLastError();
}

// A row's elements with those that its first group may hold before it
constexpr int span(int n) { return n + (n % 8 == 0 ? 0 : n % 4 == 0 ? 4 : n % 2 == 0 ? 6 : 7); }
constexpr int kRingWidth = 2048;  // the longest span of eight warps with eight elements a lane
// Warps a row.  A lane holds 8 elements: in the backward it keeps two sums, two parameters and eight operand values of
// each in registers.  16 only for rows longer than a block of 512 threads covers with 8, and in the forward without
// copies ahead (two rows of registers).
constexpr int ring_warps(int n) {
  return n <= 256 ? 1 : n <= 512 ? 2 : n <= 768 ? 3 : n <= 1024 ? 4 : n <= 1536 ? 6 : 8;
}
constexpr int fwd_warps(int n) { return n <= 512 ? 1 : n <= 1024 ? 2 : n <= 2048 ? 4 : n <= 4096 ? 8 : n <= 8192 ? 16 : 32; }
constexpr int bwd_warps(int n) { return n <= kRingWidth ? ring_warps(n) : n <= 8192 ? 16 : 32; }
constexpr int rows_per_block(int warps) { return warps > 8 ? 1 : 8 / warps; }

// Blocks a sample of at most `most`; where they take more than one step over the rows and the rows are shifted, the
// step is a multiple of eight rows.
static int row_blocks(int64_t rows, int n, int warps, int64_t most) {
  const int64_t rpb = rows_per_block(warps), need = (rows + rpb - 1) / rpb;
  if (need <= most) return (int)need;
  const int64_t unit = n % 8 ? 8 / rpb : 1;
  return (int)std::max<int64_t>(unit, most / unit * unit);
}

template <typename T>
static cudaError_t launch_forward(const Params& p, Access mode, int64_t samples, int sms, cudaStream_t s) {
  if (mode != kScalar && span(p.n) <= kRingWidth) {
    // as many blocks an SM as have 48 KB on their way; more of them only spread the accesses over more of memory
    // (64800 x 1024: 83 us with two, 89 with four; x 520, with idle lanes: 53 with three, 48 with four)
    const int warps = ring_warps(span(p.n)), ahead = (kRing - 1) * rows_per_block(warps) * p.n * 2 * 2;
    const int64_t most = std::min(kFwdBlocks, (48 * 1024 + ahead - 1) / ahead) * (int64_t)sms / samples;
    const dim3 grid((unsigned)row_blocks(p.rows, p.n, warps, std::max<int64_t>(1, most)), (unsigned)samples);
    switch (warps) {
      case 1: return mode == kVec ? launch_ring<T, kVec, 1>(p, grid, s) : launch_ring<T, kShift, 1>(p, grid, s);
      case 2: return mode == kVec ? launch_ring<T, kVec, 2>(p, grid, s) : launch_ring<T, kShift, 2>(p, grid, s);
      case 3: return mode == kVec ? launch_ring<T, kVec, 3>(p, grid, s) : launch_ring<T, kShift, 3>(p, grid, s);
      case 6: return mode == kVec ? launch_ring<T, kVec, 6>(p, grid, s) : launch_ring<T, kShift, 6>(p, grid, s);
      case 4: return mode == kVec ? launch_ring<T, kVec, 4>(p, grid, s) : launch_ring<T, kShift, 4>(p, grid, s);
      default: return mode == kVec ? launch_ring<T, kVec, 8>(p, grid, s) : launch_ring<T, kShift, 8>(p, grid, s);
    }
  }
  const bool vec = mode == kVec;
  const int warps = fwd_warps(p.n);
  const dim3 grid((unsigned)row_blocks(p.rows, 8, warps, std::max<int64_t>(1, 16 * (int64_t)sms / samples)),
                  (unsigned)samples);
  switch (warps) {  // 16-byte accesses reach only rows that are too long for the ring
    case 1: return launch_fwd<T, false, 1, 2>(p, grid, s);
    case 2: return launch_fwd<T, false, 2, 2>(p, grid, s);
    case 4: return launch_fwd<T, false, 4, 2>(p, grid, s);
    case 8: return vec ? launch_fwd<T, true, 8, 2>(p, grid, s) : launch_fwd<T, false, 8, 2>(p, grid, s);
    case 16: return vec ? launch_fwd<T, true, 16, 2>(p, grid, s) : launch_fwd<T, false, 16, 2>(p, grid, s);
    default: return vec ? launch_fwd<T, true, 32, 2>(p, grid, s) : launch_fwd<T, false, 32, 2>(p, grid, s);
  }
}

template <typename T, int MODE>
static cudaError_t launch_backward(const Params& p, dim3 grid, cudaStream_t s) {
  switch (bwd_warps(span(p.n))) {
    case 1: return launch_bwd<T, MODE, 1, 1>(p, grid, s);
    case 2: return launch_bwd<T, MODE, 2, 1>(p, grid, s);
    case 3: return launch_bwd<T, MODE, 3, 1>(p, grid, s);
    case 4: return launch_bwd<T, MODE, 4, 1>(p, grid, s);
    case 6: return launch_bwd<T, MODE, 6, 1>(p, grid, s);
    case 8: return launch_bwd<T, MODE, 8, 1>(p, grid, s);
    default: break;
  }
  if constexpr (MODE == kShift) {
    return cudaErrorInvalidValue;  // shifted rows are of the ring's widths
  } else {
    if (bwd_warps(span(p.n)) == 32) return launch_bwd<T, MODE, 32, 2>(p, grid, s);
    return span(p.n) <= 4096 ? launch_bwd<T, MODE, 16, 1>(p, grid, s) : launch_bwd<T, MODE, 16, 2>(p, grid, s);
  }
}

}  // namespace ng

int norm_gate_blocks(int64_t samples, int64_t rows, int n, int sms) {
  // as many as are resident over all samples, at least one a sample
  const int warps = ng::bwd_warps(ng::span(n));
  const int64_t most = ng::bwd_blocks(n % 8 ? ng::kShift : ng::kVec, warps) * (int64_t)sms / samples;
  return ng::row_blocks(rows, n, warps, std::max<int64_t>(1, most));
}

static cudaError_t norm_gate_launch(const NormGateArgs& a, bool backward, int blocks, int sms, cudaStream_t s) {
  if (a.n < 1 || a.n > kNormGateMaxWidth || a.samples < 1 || a.samples > 65535 || a.rows < 1 ||
      (a.dtype != kBF16 && a.dtype != kF16))
    return cudaErrorInvalidValue;
  ng::Params p;
  p.y = a.y;
  p.skip = a.skip;
  p.ds = a.ds;
  p.dn = a.dn;
  p.stream = a.stream;
  p.normed = a.normed;
  p.dy = a.dy;
  p.dskip = a.dskip;
  p.wp = a.wp;
  p.gate = a.gate;
  p.wn = a.wn;
  p.gate_stride = a.gate_stride;
  p.part = a.part;
  p.rows = a.rows;
  p.total = a.samples * a.rows * a.n;
  p.n = a.n;
  p.c = a.skip_scale;
  p.eps = a.eps;
  p.inv_n = 1.f / (float)a.n;
  uintptr_t tensors = 0, vectors = 0;
  for (const void* q : {a.y, a.skip, a.ds, a.dn, (const void*)a.stream, (const void*)a.normed, (const void*)a.dy,
                        (const void*)a.dskip})
    tensors |= reinterpret_cast<uintptr_t>(q);
  for (const float* q : {a.wp, a.gate, a.wn}) vectors |= reinterpret_cast<uintptr_t>(q);
  const ng::Access mode = (tensors & 15) != 0                          ? ng::kScalar
                          : a.n % 8 == 0 && (vectors & 15) == 0        ? ng::kVec
                          : a.n >= 8 && ng::span(a.n) <= ng::kRingWidth ? ng::kShift
                                                                       : ng::kScalar;
  if (backward && a.n > kNormGateSkipWidth && (!a.dy || !a.dskip)) return cudaErrorInvalidValue;
  const bool bf = a.dtype == kBF16;
  if (!backward)
    return bf ? ng::launch_forward<__nv_bfloat16>(p, mode, a.samples, sms, s)
              : ng::launch_forward<__half>(p, mode, a.samples, sms, s);
  const dim3 grid((unsigned)blocks, (unsigned)a.samples, 1);
  switch (mode) {
    case ng::kVec:
      return bf ? ng::launch_backward<__nv_bfloat16, ng::kVec>(p, grid, s)
                : ng::launch_backward<__half, ng::kVec>(p, grid, s);
    case ng::kShift:
      return bf ? ng::launch_backward<__nv_bfloat16, ng::kShift>(p, grid, s)
                : ng::launch_backward<__half, ng::kShift>(p, grid, s);
    default:
      return bf ? ng::launch_backward<__nv_bfloat16, ng::kScalar>(p, grid, s)
                : ng::launch_backward<__half, ng::kScalar>(p, grid, s);
  }
}

cudaError_t norm_gate_fwd(const NormGateArgs& a, int sms, cudaStream_t s) {
  return norm_gate_launch(a, false, 0, sms, s);
}

cudaError_t norm_gate_bwd(const NormGateArgs& a, int blocks, cudaStream_t s) {
  NSW_CUDA_CHECK(norm_gate_launch(a, true, blocks, 0, s));
  ng::finish_kernel<<<(a.n + 31) / 32, 1024, 0, s>>>(a.part, a.samples, blocks, a.n, a.wp, a.gate, a.gate_stride,
                                                     a.dwp, a.dgate, a.dwn);
  return cudaGetLastError();
}

}  // namespace nsw
