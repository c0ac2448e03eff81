// What the bindings of several operators share: argument checks, operands in rows that TMA can read, and where
// parameters' gradients go.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/extension.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "kernels.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e));
}

int dt_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return nsw::kBF16;
    case at::kHalf: return nsw::kF16;
    case at::kFloat: return nsw::kF32;
    default: TORCH_CHECK(false, what, ": unsupported dtype ", t.scalar_type());
  }
  return -1;
}

// in a node's backward: gradients of gradients would silently be missing
void once_differentiable(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": second derivatives are not implemented (create_graph=True)");
}

// The kernels read the values alone, and a missing tangent counts as zero.  (Without a level there are no tangents;
// the test of each tensor costs 50 ns where it is a view.)
bool tangents() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what,
              ": forward-mode derivatives are not implemented");
}
void no_tangent(const OptTensor& t, const char* what) {
  if (t) no_tangent(*t, what);
}

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// A [rows, cols] operand the TMA kernels can read: unit column stride, 16-byte aligned rows.
struct Rows {
  Tensor t;
  int64_t ld;
  void* ptr() const { return t.data_ptr(); }
};
bool rows_aligned(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) == 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&
         (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}
// contiguous and at a 16-byte boundary, which a view into a packed buffer may miss: t itself or a copy
Tensor packed(const Tensor& t) {
  const Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 ? c : c.clone();
}
// Operands as the kernels read them: each itself, or a copy with padded rows where its strides or address do not
// allow 16-byte accesses.  One launch makes all copies of a call.
struct Aligner {
  nsw::PadCopy v[nsw::kPadCopies];
  int count = 0;
  Rows add(const Tensor& t) {
    if (rows_aligned(t)) return {t, t.size(0) == 1 ? round8(t.size(1)) : t.stride(0)};
    TORCH_CHECK(count < nsw::kPadCopies, "too many operands to copy");
    const int64_t ld = round8(t.size(1));
    auto c = torch::empty({t.size(0), ld}, t.options());
    v[count++] = {t.data_ptr(), c.data_ptr(), t.stride(0), t.stride(1), ld, t.size(0), t.size(1)};
    return {c.narrow(1, 0, t.size(1)), ld};
  }
  void run() {
    if (count) check(nsw::pad_copy(v, count, stream()), "pad_copy");
  }
};

OptTensor packed_vec(const OptTensor& t) { return !t || t->is_contiguous() ? t : OptTensor(t->contiguous()); }
const void* opt_ptr(const OptTensor& t) { return t && t->defined() ? t->data_ptr() : nullptr; }

// (..., n) as a matrix; a matrix y with x's leading dimensions
Tensor flat(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }
OptTensor flat(const OptTensor& t) { return t ? OptTensor(flat(*t)) : OptTensor(); }
Tensor unflat(const Tensor& y, const Tensor& x) {
  if (x.dim() == 2) return y;
  auto sizes = x.sizes().vec();
  sizes.back() = y.size(1);
  return y.view(sizes);
}

// Where a parameter's gradient goes: added into the given fp32 buffer, or a fresh tensor (16-bit where that is
// the parameter's type, else fp32 and cast at the end)
struct GradOut {
  Tensor t;
  bool f32 = false, into = false;
  GradOut() = default;
  GradOut(const OptTensor& dst, at::IntArrayRef sizes, const Tensor& like, at::ScalarType dtype)
      : f32(dst.has_value() || dtype != like.scalar_type()), into(dst.has_value()) {
    t = into ? *dst : torch::empty(sizes, f32 ? like.options().dtype(at::kFloat) : like.options());
  }
  Tensor result(at::ScalarType dtype) const {
    if (into) return Tensor();
    return t.scalar_type() == dtype ? t : t.to(dtype);
  }
};

// The kernels read, add and write their targets without regard to one another
void check_apart(const std::vector<OptTensor>& into, const char* what) {
  std::vector<std::pair<const char*, const char*>> at;
  for (const OptTensor& t : into)
    if (t && t->numel() > 0) {
      const char* p = static_cast<const char*>(t->data_ptr());
      at.emplace_back(p, p + t->nbytes());
    }
  std::sort(at.begin(), at.end());
  for (size_t i = 1; i < at.size(); ++i)
    TORCH_CHECK(at[i].first >= at[i - 1].second, what, ": gradient buffers overlap");
}

int sm_count(const Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

}  // namespace
