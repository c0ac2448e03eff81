// PyTorch bindings of window attention with a learned relative position bias: argument checks, outputs and workspaces
// (from PyTorch's allocator, on the current stream) and the launches.
#include "bindings_util.h"

namespace {

// the 14 integers of a geometry: B, T, H, W, heads, head_dim, wh, ww, shifts, mask, mask_shift, row_offset, h_global
nsw::AttnGeom geom_of(const std::vector<int64_t>& gi, double scale, const Tensor& qkv) {
  TORCH_CHECK(gi.size() == 14, "geometry: 14 ints expected");
  nsw::AttnGeom g{};
  int* at[14] = {&g.B, &g.T, &g.H, &g.W, &g.nh, &g.hd, &g.wh, &g.ww, &g.sh, &g.sw, &g.mask, &g.mask_shift, &g.row_offset,
                 &g.h_global};
  for (int i = 0; i < 14; ++i) *at[i] = (int)gi[i];
  g.scale = (float)scale;
  g.qkv_stride = 3LL * g.nh * g.hd;
  g.out_stride = (int64_t)g.nh * g.hd;
  const int64_t length = (int64_t)g.T * g.wh * g.ww;
  TORCH_CHECK_VALUE(g.T > 0 && g.wh > 0 && g.ww > 0 && g.nh > 0 && g.H % g.wh == 0 && g.W % g.ww == 0,
                    "window_attention: a ", g.H, " x ", g.W, " grid is not whole windows of ", g.wh, " x ", g.ww);
  TORCH_CHECK_VALUE(length <= 192, "window_attention: windows of ", length, " tokens (at most 192)");
  TORCH_CHECK_VALUE(g.hd == 16 || g.hd == 32 || g.hd == 64 || g.hd == 128, "window_attention: head_dim ", g.hd,
                    " is not 16, 32, 64 or 128");
  TORCH_CHECK(qkv.is_cuda() && qkv.is_contiguous() && qkv.numel() == (int64_t)g.B * g.T * g.H * g.W * g.qkv_stride &&
                  (qkv.scalar_type() == at::kBFloat16 || qkv.scalar_type() == at::kHalf),
              "window_attention: qkv must be a contiguous 16-bit CUDA tensor of the grid's tokens");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(qkv.data_ptr()) & 15) == 0, "window_attention: qkv must be 16-byte aligned");
  return g;
}
int64_t buckets_of(const nsw::AttnGeom& g) { return (int64_t)(2 * g.T - 1) * (2 * g.wh - 1) * (2 * g.ww - 1); }
int64_t windows_of(const nsw::AttnGeom& g) { return (int64_t)g.B * (g.H / g.wh) * (g.W / g.ww); }
// {out [tokens, heads * head_dim], lse, tab}: lse has two values a row, tab what the kernels take of
// the parameters
std::vector<Tensor> attn_bias_fwd(const Tensor& qkv, const Tensor& qw, const Tensor& kw, const Tensor& rel_bias,
                                  const std::vector<int64_t>& gi, double scale) {
  const nsw::AttnGeom g = geom_of(gi, scale, qkv);
  const auto any = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.device() == qkv.device(), "window_attention: ", name, " must be on the input's device");
    return nsw::AnyMatrix{t.data_ptr(), dt_code(t, name), t.stride(0), t.dim() > 1 ? t.stride(1) : 0};
  };
  TORCH_CHECK_VALUE(rel_bias.dim() == 2 && rel_bias.size(0) == g.nh && rel_bias.size(1) == buckets_of(g),
                    "window_attention: rel_bias must be [", g.nh, ", ", buckets_of(g), "], got ", rel_bias.sizes());
  TORCH_CHECK_VALUE(qw.dim() == 1 && qw.size(0) == g.hd && kw.dim() == 1 && kw.size(0) == g.hd,
                    "window_attention: the norms' weights must be [", g.hd, "]");
  const nsw::AnyMatrix table = any(rel_bias, "rel_bias"), q = any(qw, "q_norm_w"), k = any(kw, "k_norm_w");
  const c10::cuda::CUDAGuard guard(qkv.device());
  const auto f32 = qkv.options().dtype(at::kFloat);
  auto out = torch::empty({qkv.numel() / g.qkv_stride, g.out_stride}, qkv.options());
  auto lse = torch::empty({2 * windows_of(g) * g.nh * g.T * g.wh * g.ww}, f32);
  nsw::AttnBias bias = nsw::attn_bias_layout(g);
  auto tab = torch::empty({(int64_t)g.nh * bias.stride + 2 * g.hd}, f32);
  if (qkv.numel() == 0) return {out, lse, tab};
  float* norms = tab.data_ptr<float>() + (int64_t)g.nh * bias.stride;
  check(nsw::attn_bias_prepare(table, q, k, g, bias, tab.data_ptr<float>(), stream()), "attn_bias_prepare");
  bias.tab = tab.data_ptr<float>();
  check(nsw::attn_bias_fwd(qkv.data_ptr(), bias, norms, out.data_ptr(), lse.data_ptr<float>(), g, dt_code(qkv, "qkv"),
                           sm_count(qkv), stream()),
        "window_attention");
  return {out, lse, tab};
}

// {dqkv, dqw, dkw, dbias}: the last three where need is set, of the given types, or undefined and added into their fp32
// buffers in `into`
std::vector<Tensor> attn_bias_bwd(const Tensor& qkv, const Tensor& tab, const Tensor& out, const Tensor& dout,
                                  const Tensor& lse, const std::vector<int64_t>& gi, double scale,
                                  const std::vector<bool>& need, const std::vector<OptTensor>& into,
                                  const std::vector<at::ScalarType>& types) {
  const nsw::AttnGeom g = geom_of(gi, scale, qkv);
  nsw::AttnBias bias = nsw::attn_bias_layout(g);
  TORCH_CHECK(need.size() == 3 && into.size() == 3 && types.size() == 3, "window_attention backward: three parameters");
  TORCH_CHECK(dout.is_contiguous() && dout.scalar_type() == qkv.scalar_type() && dout.numel() == out.numel() &&
                  dout.device() == qkv.device() && tab.numel() == (int64_t)g.nh * bias.stride + 2 * g.hd &&
                  lse.numel() == 2 * windows_of(g) * g.nh * g.T * g.wh * g.ww &&
                  (reinterpret_cast<uintptr_t>(dout.data_ptr()) & 15) == 0,
              "window_attention backward: arguments are not the forward's");
  check_apart(into, "window_attention backward");
  const c10::cuda::CUDAGuard guard(qkv.device());
  const auto f32 = qkv.options().dtype(at::kFloat);
  const std::vector<int64_t> sizes[3] = {{g.hd}, {g.hd}, {g.nh, buckets_of(g)}};
  auto dqkv = torch::empty(qkv.sizes(), qkv.options());
  std::vector<Tensor> res = {dqkv, {}, {}, {}};
  nsw::AttnGrad grad[3] = {};
  for (int i = 0; i < 3; ++i) {
    if (!need[i]) continue;
    if (into[i]) {
      TORCH_CHECK(into[i]->scalar_type() == at::kFloat && into[i]->is_contiguous() && into[i]->device() == qkv.device() &&
                      into[i]->numel() == (i < 2 ? g.hd : g.nh * buckets_of(g)),
                  "window_attention backward: gradient buffers must be contiguous fp32 CUDA tensors of their parameters' sizes");
      grad[i] = {nullptr, into[i]->data_ptr(), nsw::kF32, 1};
    } else {
      res[1 + i] = qkv.numel() == 0 ? torch::zeros(sizes[i], f32.dtype(types[i])) : torch::empty(sizes[i], f32.dtype(types[i]));
      grad[i] = {nullptr, res[1 + i].data_ptr(), dt_code(res[1 + i], "window_attention backward"), 0};
    }
  }
  if (qkv.numel() == 0) return res;
  bias.tab = tab.data_ptr<float>();
  const int dtype = dt_code(qkv, "qkv");
  const nsw::AttnBiasPlan plan = nsw::attn_bias_plan(g, dtype, need[2], sm_count(qkv));
  auto part = torch::empty({2 * plan.norm_rows * g.hd + (need[2] ? plan.bias_rows * buckets_of(g) : 0)}, f32);
  float* qp = part.data_ptr<float>();
  float* kp = qp + plan.norm_rows * g.hd;
  float* bp = need[2] ? kp + plan.norm_rows * g.hd : nullptr;
  check(nsw::attn_bias_bwd(qkv.data_ptr(), bias, tab.data_ptr<float>() + (int64_t)g.nh * bias.stride, out.data_ptr(),
                           dout.data_ptr(), lse.data_ptr<float>(), dqkv.data_ptr(), qp, kp, bp, plan, g, dtype, stream()),
        "window_attention backward");
  grad[0].part = qp;
  grad[1].part = kp;
  grad[2].part = bp;
  check(nsw::attn_bias_grads(grad[2], grad[0], grad[1], plan, g, stream()), "window_attention parameter gradients");
  return res;
}

struct AttnBiasNode : public torch::autograd::Function<AttnBiasNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& qkv, const Tensor& qw, const Tensor& kw,
                        const Tensor& rel_bias, const std::vector<int64_t>& gi, double scale) {
    auto r = attn_bias_fwd(qkv, qw, kw, rel_bias, gi, scale);
    ctx->save_for_backward({qkv, r[2], r[0], r[1]});
    ctx->saved_data["geom"] = gi;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)qw.scalar_type(), (int64_t)kw.scalar_type(),
                                                    (int64_t)rel_bias.scalar_type()};
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    once_differentiable("window_attention");
    const auto v = ctx->get_saved_variables();
    std::vector<at::ScalarType> types;
    for (int64_t t : ctx->saved_data["types"].toIntVector()) types.push_back((at::ScalarType)t);
    auto r = attn_bias_bwd(v[0], v[1], v[2], packed(grad[0]), v[3], ctx->saved_data["geom"].toIntVector(),
                           ctx->saved_data["scale"].toDouble(),
                           {ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(3)},
                           std::vector<OptTensor>(3), types);
    if (!ctx->needs_input_grad(0)) r[0] = Tensor();
    r.resize(6);
    return r;
  }
};

// qkv (B, T, H, W, 3 heads head_dim) in 16 bits -> (B, T, H, W, heads head_dim); parameters in any of the three types
Tensor window_attention_bias(const Tensor& qkv_in, const Tensor& qw, const Tensor& kw, const Tensor& rel_bias,
                             const std::vector<int64_t>& gi, double scale) {
  const Tensor qkv = packed(qkv_in);
  if (tangents())
    for (const Tensor* t : {&qkv, &qw, &kw, &rel_bias}) no_tangent(*t, "window_attention");
  bool grad = false;
  if (at::GradMode::is_enabled())
    for (const Tensor* t : {&qkv, &qw, &kw, &rel_bias}) grad = grad || t->requires_grad();
  const Tensor out = grad ? AttnBiasNode::apply(qkv, qw, kw, rel_bias, gi, scale)
                          : attn_bias_fwd(qkv, qw, kw, rel_bias, gi, scale)[0];
  return out.view({gi[0], gi[1], gi[2], gi[3], gi[4] * gi[5]});
}

}  // namespace

void bind_attention(py::module& m) {
  m.def("attn_bias_fwd", &attn_bias_fwd);
  m.def("attn_bias_bwd", &attn_bias_bwd);
  m.def("window_attention_bias", &window_attention_bias);
}
