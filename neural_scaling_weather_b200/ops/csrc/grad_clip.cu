// The global norm of many tensors and the tensors scaled to it:
//
//   norm = sqrt(sum over all tensors of g^2),   out = g * (norm > max ? max / (norm + 1e-6) : 1)
//
// Bound by memory: the norm has to be known before the first element can be scaled, so every element is read
// twice and written once.  The tensors come as a table in the kernel's parameters (no device table to build,
// no copy): work is cut into chunks of kChunk elements of one tensor, block b takes chunks b, b + grid, ...
// The second kernel walks the chunks from the last to the first, so that the part of them that the L2 cache
// still holds from the first kernel is not read from memory again.  Sums are fp32 per thread over at most a few
// thousand elements, then added in fixed orders (bit-identical reruns).
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace nsw {
namespace gc {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // elements

// N tensors: the few of a small model travel in a small table (a launch copies its parameters)
template <int N>
struct Table {
  const void* in[N];
  void* out[N];
  int64_t n[N];
  int first[N + 1];  // a tensor's first chunk
  uint8_t dtype[N];
  int count;
};

template <int N>
__device__ __forceinline__ int find(const Table<N>& t, int chunk) {
  int lo = 0, hi = t.count;  // the last tensor whose first chunk is <= chunk
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float w[kThreads / 32];
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = v;
  __syncthreads();
  v = w[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v += w[i];
  return v;
}

template <typename T>
__device__ __forceinline__ float chunk_sumsq(const T* p, int len) {
  constexpr int V = 16 / sizeof(T);
  float a = 0.f;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const int nv = len / V;
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += kThreads) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      float f[8];
      if (sizeof(T) == 4) {
        f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
      } else {
        if constexpr (sizeof(T) == 2) unpack8<T>(u, f);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) a = fmaf(f[j], f[j], a);
    }
    for (int i = nv * V + threadIdx.x; i < len; i += kThreads) {
      const float f = to_f(p[i]);
      a = fmaf(f, f, a);
    }
  } else {
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const float f = to_f(p[i]);
      a = fmaf(f, f, a);
    }
  }
  return a;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* p, T* o, int len, float c) {
  constexpr int V = 16 / sizeof(T);
  int i0 = 0;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
    const int nv = len / V;
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += kThreads) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + i);
      uint4 r;
      if constexpr (sizeof(T) == 2) {
        float f[8];
        unpack8<T>(u, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= c;
        r = pack8<T>(f);
      } else {
        r = make_uint4(__float_as_uint(__uint_as_float(u.x) * c), __float_as_uint(__uint_as_float(u.y) * c),
                       __float_as_uint(__uint_as_float(u.z) * c), __float_as_uint(__uint_as_float(u.w) * c));
      }
      __stcs(reinterpret_cast<uint4*>(o) + i, r);
    }
    i0 = nv * V;
  }
  for (int i = i0 + threadIdx.x; i < len; i += kThreads) o[i] = from_f<T>(to_f(p[i]) * c);
}

template <int N>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ Table<N> t, float* partial) {
  float a = 0.f;
  const int chunks = t.first[t.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find(t, c);
    const int64_t off = (int64_t)(c - t.first[i]) * kChunk;
    const int len = (int)(t.n[i] - off < kChunk ? t.n[i] - off : kChunk);
    if (t.dtype[i] == kF32)
      a += chunk_sumsq(reinterpret_cast<const float*>(t.in[i]) + off, len);
    else if (t.dtype[i] == kBF16)
      a += chunk_sumsq(reinterpret_cast<const __nv_bfloat16*>(t.in[i]) + off, len);
    else
      a += chunk_sumsq(reinterpret_cast<const __half*>(t.in[i]) + off, len);
  }
  a = block_sum(a);
  if (threadIdx.x == 0) partial[blockIdx.x] = a;
}

template <int N>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table<N> t, const float* partial,
                                                         int partials, float max_norm, float* norm_out) {
  float a = 0.f;
  for (int i = threadIdx.x; i < partials; i += kThreads) a += partial[i];
  const float norm = sqrtf(block_sum(a));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float coef = norm > max_norm ? max_norm / (norm + 1e-6f) : 1.f;
  const int chunks = t.first[t.count];
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const int i = find(t, c);
    if (coef == 1.f && t.in[i] == t.out[i]) continue;  // in place and within the limit: nothing changes
    const int64_t off = (int64_t)(c - t.first[i]) * kChunk;
    const int len = (int)(t.n[i] - off < kChunk ? t.n[i] - off : kChunk);
    if (t.dtype[i] == kF32)
      chunk_scale(reinterpret_cast<const float*>(t.in[i]) + off, reinterpret_cast<float*>(t.out[i]) + off, len, coef);
    else if (t.dtype[i] == kBF16)
      chunk_scale(reinterpret_cast<const __nv_bfloat16*>(t.in[i]) + off,
                  reinterpret_cast<__nv_bfloat16*>(t.out[i]) + off, len, coef);
    else
      chunk_scale(reinterpret_cast<const __half*>(t.in[i]) + off, reinterpret_cast<__half*>(t.out[i]) + off, len,
                  coef);
  }
}

}  // namespace gc

// false: more than 2^31 - 1 chunks
template <int N>
static bool fill(gc::Table<N>& t, const ClipTensor* v, int count) {
  t.count = count;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    t.in[i] = v[i].in;
    t.out[i] = v[i].out;
    t.n[i] = v[i].n;
    t.dtype[i] = (uint8_t)v[i].dtype;
    t.first[i] = (int)chunks;
    chunks += (v[i].n + gc::kChunk - 1) / gc::kChunk;
    if (chunks > INT32_MAX) return false;
  }
  t.first[count] = (int)chunks;
  return true;
}

template <int N>
static cudaError_t clip_tables(const ClipTensor* v, int count, float max_norm, float* partial, int blocks, float* norm,
                               cudaStream_t s) {
  // every table's blocks write their own partials; every scaling launch adds all of them
  const int tables = (count + N - 1) / N;
  gc::Table<N> t;
  for (int pass = 0; pass < 2; ++pass)
    for (int k = 0; k < tables; ++k) {
      const int i = pass ? tables - 1 - k : k;
      if ((pass == 0 || tables > 1) && !fill(t, v + i * N, std::min(N, count - i * N))) return cudaErrorInvalidValue;
      if (pass == 0)
        gc::sumsq_kernel<N><<<blocks, gc::kThreads, 0, s>>>(t, partial + i * blocks);
      else
        gc::scale_kernel<N>
            <<<blocks, gc::kThreads, 0, s>>>(t, partial, tables * blocks, max_norm, k == 0 ? norm : nullptr);
      NSW_CUDA_CHECK(cudaGetLastError());
    }
  return cudaSuccess;
}

cudaError_t clip_tensors(const ClipTensor* v, int count, float max_norm, float* partial, int blocks, float* norm,
                         cudaStream_t s) {
  if (count <= 32) return clip_tables<32>(v, count, max_norm, partial, blocks, norm, s);
  return clip_tables<kClipTensors>(v, count, max_norm, partial, blocks, norm, s);
}

}  // namespace nsw
