// PyTorch bindings of the transformer-block operators: the gated feed-forward network, the norms with gate
// and skip connection, and gradient clipping.  Argument checks, outputs and workspaces (from PyTorch's
// allocator, on the current stream) and the launches.
#include "bindings_util.h"

namespace {

void check_matrix(const Tensor& t, int64_t rows, int64_t cols, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "gated_mlp: ", name, " must be on the input's device");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "gated_mlp: ", name, " must have the compute dtype ",
              like.scalar_type(), ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, "gated_mlp: ", name, " must be [", rows, ", ",
              cols, "], got ", t.sizes());
}
void check_bias(const OptTensor& b, int64_t n, const Tensor& like, int* dtype, const char* name) {
  if (!b || !b->defined()) return;
  TORCH_CHECK(b->is_cuda() && b->device() == like.device() && b->dim() == 1 && b->numel() == n, "gated_mlp: ", name,
              " must be a CUDA vector of ", n, " elements");
  const int d = dt_code(*b, name);
  TORCH_CHECK(*dtype < 0 || *dtype == d, "gated_mlp: the gate's and the up projection's biases must share a dtype");
  *dtype = d;
}

struct GatedShape {
  int64_t M, K, H, N, Hp;
};
GatedShape gated_shape(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "gated_mlp: x must be a CUDA matrix");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "gated_mlp: bf16 or fp16, got ",
              x.scalar_type());
  GatedShape d{x.size(0), x.size(1), wg.size(0), wd.size(0), 0};
  d.Hp = round8(d.H);
  check_matrix(wg, d.H, d.K, x, "w_gate");
  check_matrix(wu, d.H, d.K, x, "w_up");
  check_matrix(wd, d.N, d.H, x, "w_down");
  TORCH_CHECK(d.K > 0 && d.H > 0 && d.N > 0, "gated_mlp: empty weights");
  TORCH_CHECK(d.M < (int64_t(1) << 31) - 256 && d.K < (int64_t(1) << 30) && d.H < (int64_t(1) << 30) &&
                  d.N < (int64_t(1) << 30),
              "gated_mlp: too many rows or features");
  return d;
}

// y = (act(x wg^T + bg) * (x wu^T + bu)) wd^T + bd + residual.  With save, also what the backward reads:
// returns {y} or {y, x, g, u, h, wg, wu, wd} with x and the weights as read (copies with padded rows where theirs are
// not aligned) and the rows of g, u and h padded to a multiple of 8 elements.
std::vector<Tensor> gated_mlp_fwd(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                                  const OptTensor& b_gate, const OptTensor& b_up, const OptTensor& b_down,
                                  const OptTensor& residual, int64_t act, bool save) {
  const GatedShape d = gated_shape(x, wg, wu, wd);
  int bdt = -1, ddt = -1;
  check_bias(b_gate, d.H, x, &bdt, "b_gate");
  check_bias(b_up, d.H, x, &bdt, "b_up");
  check_bias(b_down, d.N, x, &ddt, "b_down");
  const bool has_res = residual && residual->defined();
  if (has_res) check_matrix(*residual, d.M, d.N, x, "residual");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto opt = x.options();
  if (d.M == 0) {
    auto y = torch::empty({0, d.N}, opt), e = torch::empty({0, d.Hp}, opt);
    if (!save) return {y};
    return {y, x, e, e, e, wg, wu, wd};
  }
  const OptTensor bg = packed_vec(b_gate), bu = packed_vec(b_up), bd = packed_vec(b_down);
  auto h = torch::empty({d.M, d.Hp}, opt);
  nsw::GatedArgs up{}, down{};
  up.mode = nsw::kGatedUp;
  down.mode = nsw::kGatedDown;
  up.dtype = down.dtype = dt_code(x, "x");
  up.act = (int)act;
  up.M = down.M = d.M;
  up.N = d.H;
  up.K = d.K;
  up.bias0 = opt_ptr(bg);
  up.bias1 = opt_ptr(bu);
  up.bias_dtype = bdt;
  up.out0 = h.data_ptr();
  up.ldout = d.Hp;
  down.N = d.N;
  down.K = d.H;
  down.a0 = h.data_ptr();
  down.lda = d.Hp;
  down.bias0 = opt_ptr(bd);
  down.bias_dtype = ddt;
  const auto unit = [](const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1; };
  if (!save && d.M <= nsw::kGatedSkinnyTokens && unit(x) && unit(wg) && unit(wu) && unit(wd) &&
      (!has_res || unit(*residual))) {
    auto y = torch::empty({d.M, d.N}, opt);
    up.a0 = x.data_ptr();
    up.lda = x.stride(0);
    up.b0 = wg.data_ptr();
    up.ldb0 = wg.stride(0);
    up.b1 = wu.data_ptr();
    up.ldb1 = wu.stride(0);
    check(nsw::gated_skinny(up, false, stream()), "gated_mlp up");
    down.b0 = wd.data_ptr();
    down.ldb0 = wd.stride(0);
    down.in0 = has_res ? residual->data_ptr() : nullptr;
    down.ldin = has_res ? residual->stride(0) : 0;
    down.out0 = y.data_ptr();
    down.ldout = d.N;
    check(nsw::gated_skinny(down, true, stream()), "gated_mlp down");
    return {y};
  }
  // all copies come before the first product: the second may start under it
  Aligner al;
  const Rows xa = al.add(x), ga = al.add(wg), ua = al.add(wu), da = al.add(wd);
  Rows ra;
  if (has_res) {  // rows of any alignment are read in place
    const bool rows = unit(*residual) && (d.M == 1 || residual->stride(0) >= d.N);
    ra = rows ? Rows{*residual, d.M == 1 ? d.N : residual->stride(0)} : al.add(*residual);
    down.in0 = ra.ptr();
    down.ldin = ra.ld;
  }
  al.run();
  Tensor g, u;
  if (save) {
    g = torch::empty({d.M, d.Hp}, opt);
    u = torch::empty({d.M, d.Hp}, opt);
    up.out1 = g.data_ptr();
    up.out2 = u.data_ptr();
    up.ldaux = d.Hp;
  }
  up.a0 = xa.ptr();
  up.lda = xa.ld;
  up.b0 = ga.ptr();
  up.ldb0 = ga.ld;
  up.b1 = ua.ptr();
  up.ldb1 = ua.ld;
  check(nsw::gated_product(up, false, stream()), "gated_mlp up");
  auto y = torch::empty({d.M, d.N}, opt);
  down.b0 = da.ptr();
  down.ldb0 = da.ld;
  down.out0 = y.data_ptr();
  down.ldout = d.N;
  check(nsw::gated_product(down, true, stream()), "gated_mlp down");
  if (!save) return {y};
  return {y, xa.t, g, u, h, ga.t, ua.t, da.t};
}

// Gradients from dy and what the forward saved: {dx, dwg, dwu, dwd, dbg, dbu, dbd}, of which only those with need
// set are computed.  An entry is undefined where it is not needed or was added into its fp32 buffer in `into` (three
// weights, three biases).  types: of the same six, their parameters'.
std::vector<Tensor> gated_mlp_bwd(const Tensor& dy, const Tensor& x, const Tensor& wg, const Tensor& wu,
                                  const Tensor& wd, const Tensor& g, const Tensor& u, const Tensor& h, int64_t act,
                                  const std::vector<bool>& need, const std::vector<OptTensor>& into,
                                  const std::vector<at::ScalarType>& types) {
  const GatedShape d = gated_shape(x, wg, wu, wd);
  check_matrix(dy, d.M, d.N, x, "dy");
  check_matrix(g, d.M, d.Hp, x, "g");
  check_matrix(u, d.M, d.Hp, x, "u");
  check_matrix(h, d.M, d.Hp, x, "h");
  TORCH_CHECK(g.is_contiguous() && u.is_contiguous() && h.is_contiguous() && (d.M == 0 || rows_aligned(x)),
              "gated_mlp backward: saved tensors must be as the forward returned them");
  TORCH_CHECK(need.size() == 7 && into.size() == 6 && types.size() == 6,
              "gated_mlp backward: x, three weights and three biases");
  check_apart(into, "gated_mlp backward");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto opt = x.options();
  std::vector<Tensor> out(7);
  const std::vector<int64_t> sizes[6] = {{d.H, d.K}, {d.H, d.K}, {d.N, d.H}, {d.H}, {d.H}, {d.N}};
  if (d.M == 0) {
    if (need[0]) out[0] = torch::empty({0, d.K}, opt);
    for (int i = 0; i < 6; ++i)
      if (need[1 + i] && !into[i]) out[1 + i] = torch::zeros(sizes[i], opt.dtype(types[i]));
    return out;
  }
  GradOut grad[6];
  for (int i = 0; i < 6; ++i)
    if (need[1 + i]) grad[i] = GradOut(into[i], sizes[i], x, types[i]);
  const bool need_hidden = need[0] || need[1] || need[2] || need[4] || need[5];  // what follows from dg and du
  Aligner al;  // (the weights are the forward's aligned ones already)
  const Rows dya = al.add(dy), ga = al.add(wg), ua = al.add(wu), da = al.add(wd);
  al.run();
  const Rows xa{x, d.M == 1 ? round8(d.K) : x.stride(0)};
  Tensor dgu, sums;
  char* du = nullptr;
  const int dtype = dt_code(x, "x");
  if (need_hidden) {
    dgu = torch::empty({d.M, 2 * d.Hp}, opt);
    du = reinterpret_cast<char*>(dgu.data_ptr()) + 2 * d.Hp;
    nsw::GatedArgs a{};
    a.mode = nsw::kGatedDh;
    a.dtype = dtype;
    a.act = (int)act;
    a.M = d.M;
    a.N = d.H;
    a.K = d.N;
    a.a0 = dya.ptr();
    a.lda = dya.ld;
    a.b0 = da.ptr();
    a.ldb0 = da.ld;
    a.in0 = g.data_ptr();
    a.in1 = u.data_ptr();
    a.ldin = d.Hp;
    a.out0 = dgu.data_ptr();
    a.out1 = du;
    a.ldout = a.ldaux = 2 * d.Hp;
    const int64_t rows = need[4] || need[5] ? nsw::gated_sum_rows(a) : 0;
    if (rows > 0) {
      sums = torch::empty({rows, 2 * d.Hp}, opt.dtype(at::kFloat));
      a.sums = sums.data_ptr<float>();
      a.sums_half = d.Hp;
    }
    check(nsw::gated_product(a, false, stream()), "gated_mlp dh");
  }
  if (need[0]) {
    auto dx = torch::empty({d.M, d.K}, opt);
    nsw::GatedArgs b{};
    b.mode = nsw::kGatedDx;
    b.dtype = dtype;
    b.M = d.M;
    b.N = d.K;
    b.K = d.H;
    b.a0 = dgu.data_ptr();
    b.a1 = du;
    b.lda = 2 * d.Hp;
    b.b0 = ga.ptr();
    b.ldb0 = ga.ld;
    b.b1 = ua.ptr();
    b.ldb1 = ua.ld;
    b.out0 = dx.data_ptr();
    b.ldout = d.K;
    check(nsw::gated_product(b, true, stream()), "gated_mlp dx");
    out[0] = dx;
  }
  if (need[1] || need[2] || need[3]) {
    nsw::GatedDwArgs w{};
    w.dtype = dtype;
    w.T = d.M;
    const auto dst = [&](int i) { return need[1 + i] ? grad[i].t.data_ptr() : nullptr; };
    w.w[0] = {need_hidden ? dgu.data_ptr() : nullptr, xa.ptr(), 2 * d.Hp, xa.ld, d.H, d.K, dst(0), grad[0].f32,
              grad[0].into};
    w.w[1] = {du, xa.ptr(), 2 * d.Hp, xa.ld, d.H, d.K, dst(1), grad[1].f32, grad[1].into};
    w.w[2] = {dya.ptr(), h.data_ptr(), dya.ld, d.Hp, d.N, d.H, dst(2), grad[2].f32, grad[2].into};
    Tensor ws;
    const int64_t wsn = nsw::gated_dw_workspace(w);
    if (wsn > 0) {
      ws = torch::empty({wsn}, opt.dtype(at::kFloat));
      w.ws = ws.data_ptr<float>();
    }
    check(nsw::gated_dw(w, stream()), "gated_mlp weight gradients");
  }
  if (need[4] || need[5] || need[6]) {
    // dy's columns, and those of dg and du where the product before has not summed them
    const int64_t n = 2 * d.Hp, pd = need[6] ? nsw::col_sum_parts(d.M, d.N) : 0,
                  pg = (need[4] || need[5]) && !sums.defined() ? nsw::col_sum_parts(d.M, n) : 0;
    Tensor partial;
    float* pp = nullptr;
    if (pd + pg > 0) {
      partial = torch::empty({pd * d.N + pg * n}, opt.dtype(at::kFloat));
      pp = partial.data_ptr<float>();
      nsw::ColSource src[2];
      int count = 0;
      if (pd > 0) src[count++] = {dya.ptr(), dya.ld, d.M, d.N, pd, pp};
      if (pg > 0) src[count++] = {dgu.data_ptr(), n, d.M, n, pg, pp + pd * d.N};
      check(nsw::col_partial(src, count, dtype, stream()), "gated_mlp bias gradients");
    }
    const float* ps = pg > 0 ? pp + pd * d.N : sums.defined() ? sums.data_ptr<float>() : nullptr;
    const int64_t rows = pg > 0 ? pg : sums.defined() ? sums.size(0) : 0;
    const auto dst = [&](int i) { return need[1 + i] ? grad[i].t.data_ptr() : nullptr; };
    const nsw::ColSum fin[3] = {{ps, rows, n, 0, d.H, dst(3), grad[3].f32, grad[3].into},
                                {ps, rows, n, d.Hp, d.H, dst(4), grad[4].f32, grad[4].into},
                                {pp, pd, d.N, 0, d.N, dst(5), grad[5].f32, grad[5].into}};
    check(nsw::col_finish(fin, dtype, stream()), "gated_mlp bias gradients");
  }
  for (int i = 0; i < 6; ++i)
    if (need[1 + i]) out[1 + i] = grad[i].result(types[i]);
  return out;
}

// The network of 16-bit parameters as one autograd node (fp32 master parameters, whose gradients may go
// straight into the optimizer's buffers, go through the Python node on the same two functions).
struct GatedNode : public torch::autograd::Function<GatedNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const Tensor& wd, const OptTensor& bg, const OptTensor& bu, const OptTensor& bd,
                        const OptTensor& residual, int64_t act) {
    auto out = gated_mlp_fwd(flat(x), wg, wu, wd, bg, bu, bd, flat(residual), act, true);
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->save_for_backward({out[1], out[5], out[6], out[7], out[2], out[3], out[4]});
    ctx->saved_data["act"] = act;
    int64_t given = 0;  // which optional inputs there are
    std::vector<int64_t> types(3, (int64_t)wg.scalar_type());
    int bit = 0;
    for (const OptTensor* t : {&bg, &bu, &bd, &residual}) {
      if (*t) given |= 1 << bit;
      if (bit < 3) types.push_back((int64_t)(*t ? (*t)->scalar_type() : at::kFloat));
      ++bit;
    }
    ctx->saved_data["given"] = given;
    ctx->saved_data["types"] = types;
    return unflat(out[0], x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    once_differentiable("gated_mlp");
    const auto v = ctx->get_saved_variables();
    const int64_t given = ctx->saved_data["given"].toInt();
    std::vector<at::ScalarType> types;
    for (int64_t t : ctx->saved_data["types"].toIntVector()) types.push_back((at::ScalarType)t);
    std::vector<bool> need(7);
    size_t edge = 4;  // graph edges exist for the inputs that were given, in order
    const auto opt_needed = [&](int i) { return ((given >> i) & 1) != 0 && ctx->needs_input_grad(edge++); };
    for (int i = 0; i < 7; ++i) need[i] = i < 4 ? ctx->needs_input_grad(i) : opt_needed(i - 4);
    const bool need_res = opt_needed(3);
    auto g = gated_mlp_bwd(flat(grad[0]), v[0], v[1], v[2], v[3], v[4], v[5], v[6], ctx->saved_data["act"].toInt(),
                           need, std::vector<OptTensor>(6), types);
    if (need[0]) g[0] = g[0].view(ctx->saved_data["shape"].toIntVector());
    g.push_back(need_res ? grad[0] : Tensor());  // residual
    g.push_back(Tensor());                      // act
    return g;
  }
};

// x (..., K) and residual (..., N) in the weights' 16-bit type (the public entry point on CUDA, which leaves the
// checks of the shapes to this function)
Tensor gated_mlp(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& bg,
                 const OptTensor& bu, const OptTensor& bd, const OptTensor& residual, int64_t act) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && wg.dim() == 2 && wd.dim() == 2 && wu.sizes() == wg.sizes() &&
                        x.size(-1) == wg.size(1) && wd.size(1) == wg.size(0),
                    "gated_mlp: x ", x.sizes(), ", w_gate ", wg.sizes(), ", w_up ", wu.sizes(), " and w_down ",
                    wd.sizes(), " do not fit together");
  TORCH_CHECK_VALUE(!residual || (residual->dim() == x.dim() && residual->size(-1) == wd.size(0) &&
                                  residual->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1)),
                    "gated_mlp: residual ", residual->sizes(), " is not the output's shape");
  if (tangents()) {
    for (const Tensor* t : {&x, &wg, &wu, &wd}) no_tangent(*t, "gated_mlp");
    for (const OptTensor* t : {&bg, &bu, &bd, &residual}) no_tangent(*t, "gated_mlp");
  }
  bool grad = false;
  if (at::GradMode::is_enabled()) {
    for (const Tensor* t : {&x, &wg, &wu, &wd}) grad = grad || t->requires_grad();
    for (const OptTensor* t : {&bg, &bu, &bd, &residual}) grad = grad || (*t && (*t)->requires_grad());
  }
  if (grad) return GatedNode::apply(x, wg, wu, wd, bg, bu, bd, residual, act);
  return unflat(gated_mlp_fwd(flat(x), wg, wu, wd, bg, bu, bd, flat(residual), act, false)[0], x);
}

// ------------------------------------------------------------------------------ norms, gate, skip
void check_vec(const OptTensor& v, int64_t rows, int64_t n, const Tensor& like, const char* name) {
  if (!v || !v->defined()) return;
  TORCH_CHECK(v->is_cuda() && v->device() == like.device() && v->scalar_type() == at::kFloat && v->is_contiguous() &&
                  v->numel() == rows * n,
              "norm_gate_residual: ", name, " must be a contiguous fp32 CUDA tensor of ", rows * n, " elements");
}
void check_like(const OptTensor& t, const Tensor& y, const char* name) {
  if (!t || !t->defined()) return;
  TORCH_CHECK(t->device() == y.device() && t->scalar_type() == y.scalar_type() && t->is_contiguous() &&
                  t->sizes() == y.sizes(),
              "norm_gate_residual: ", name, " must be a contiguous tensor like y");
}
// y (..., n); gate (n,), or (samples, n) with y's rows in as many equal groups
nsw::NormGateArgs norm_args(const Tensor& y, const Tensor& skip, const Tensor& wp, const OptTensor& gate,
                            const OptTensor& wn, double skip_scale, double eps) {
  TORCH_CHECK(y.is_cuda() && y.dim() >= 1 && y.is_contiguous(), "norm_gate_residual: y must be a contiguous CUDA tensor");
  TORCH_CHECK(y.scalar_type() == at::kBFloat16 || y.scalar_type() == at::kHalf, "norm_gate_residual: bf16 or fp16");
  const int64_t n = y.size(-1), samples = gate && gate->dim() == 2 ? gate->size(0) : 1;
  TORCH_CHECK(n >= 1 && n <= nsw::kNormGateMaxWidth, "norm_gate_residual: width ", n, " is not in 1 .. ",
              nsw::kNormGateMaxWidth);
  TORCH_CHECK(samples <= 65535, "norm_gate_residual: at most 65535 samples");
  TORCH_CHECK(y.numel() == 0 || (y.numel() / n) % samples == 0, "norm_gate_residual: ", y.numel() / n,
              " rows are not whole groups of ", samples, " samples");
  check_like(skip, y, "skip");
  check_vec(wp, 1, n, y, "w_post");
  check_vec(gate, samples, n, y, "gate");
  check_vec(wn, 1, n, y, "w_next");
  nsw::NormGateArgs a{};
  a.y = y.data_ptr();
  a.skip = skip.data_ptr();
  a.wp = wp.data_ptr<float>();
  a.gate = static_cast<const float*>(opt_ptr(gate));
  a.wn = static_cast<const float*>(opt_ptr(wn));
  a.gate_stride = n;
  a.samples = samples;
  a.rows = y.numel() == 0 ? 0 : y.numel() / n / samples;
  a.n = (int)n;
  a.dtype = dt_code(y, "y");
  a.skip_scale = (float)skip_scale;
  a.eps = (float)eps;
  return a;
}

// {stream, normed} (normed undefined without wn)
std::vector<Tensor> norm_gate_fwd(const Tensor& y, const Tensor& skip, const Tensor& wp, const OptTensor& gate,
                                  const OptTensor& wn, double skip_scale, double eps) {
  auto a = norm_args(y, skip, wp, gate, wn, skip_scale, eps);
  const c10::cuda::CUDAGuard guard(y.device());
  auto stream_out = torch::empty_like(y);
  Tensor normed;
  a.stream = stream_out.data_ptr();
  if (a.wn) {
    normed = torch::empty_like(y);
    a.normed = normed.data_ptr();
  }
  if (y.numel() > 0) check(nsw::norm_gate_fwd(a, sm_count(y), stream()), "norm_gate_fwd");
  return {stream_out, normed};
}

// {dy, dskip, dwp, dgate, dwn}: the first two where they are needed, gradients of the vectors in fp32
std::vector<Tensor> norm_gate_bwd(const OptTensor& ds, const OptTensor& dn, const Tensor& y, const Tensor& skip,
                                  const Tensor& wp, const OptTensor& gate, const OptTensor& wn, double skip_scale,
                                  double eps, bool need_dy, bool need_dskip) {
  auto a = norm_args(y, skip, wp, gate, wn, skip_scale, eps);
  check_like(ds, y, "ds");
  check_like(dn, y, "dn");
  const c10::cuda::CUDAGuard guard(y.device());
  const auto f32 = y.options().dtype(at::kFloat);
  if (a.n > nsw::kNormGateSkipWidth) need_dy = need_dskip = true;
  Tensor dy, dskip;
  if (need_dy) dy = torch::empty_like(y);
  if (need_dskip) dskip = torch::empty_like(y);
  const int64_t n = a.n;
  if (y.numel() == 0)
    return {dy, dskip, torch::zeros({n}, f32),  // (a gate of no samples has no address)
            gate && gate->defined() ? torch::zeros({a.samples, n}, f32) : Tensor(),
            a.wn ? torch::zeros({n}, f32) : Tensor()};
  const int blocks = nsw::norm_gate_blocks(a.samples, a.rows, a.n, sm_count(y));
  auto part = torch::empty({a.samples * blocks * 2 * n}, f32);
  auto dwp = torch::empty({n}, f32);
  Tensor dgate, dwn;
  if (a.gate) dgate = torch::empty({a.samples, n}, f32);
  if (a.wn) dwn = torch::empty({n}, f32);
  a.ds = opt_ptr(ds);
  a.dn = a.wn ? opt_ptr(dn) : nullptr;
  a.dy = need_dy ? dy.data_ptr() : nullptr;
  a.dskip = need_dskip ? dskip.data_ptr() : nullptr;
  a.part = part.data_ptr<float>();
  a.dwp = dwp.data_ptr<float>();
  a.dgate = a.gate ? dgate.data_ptr<float>() : nullptr;
  a.dwn = a.wn ? dwn.data_ptr<float>() : nullptr;
  check(nsw::norm_gate_bwd(a, blocks, stream()), "norm_gate_bwd");
  return {dy, dskip, dwp, dgate, dwn};
}

struct NormGateNode : public torch::autograd::Function<NormGateNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& y_in,
                                                const Tensor& skip_in, const Tensor& wp, const OptTensor& gate,
                                                const OptTensor& wn, double skip_scale, double eps) {
    const Tensor y = y_in.contiguous(), skip = skip_in.contiguous(), wpc = wp.contiguous();
    const OptTensor gc = packed_vec(gate), wnc = packed_vec(wn);
    auto out = norm_gate_fwd(y, skip, wpc, gc, wnc, skip_scale, eps);
    if (!out[1].defined()) out.pop_back();
    ctx->save_for_backward({y, skip, wpc, gc ? *gc : Tensor(), wnc ? *wnc : Tensor()});
    ctx->saved_data["c"] = skip_scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["gate"] = gate ? gate->dim() : (int64_t)0;
    ctx->saved_data["next"] = wn.has_value();
    ctx->set_materialize_grads(false);
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    once_differentiable("norm_gate_residual");
    const auto v = ctx->get_saved_variables();
    const auto o = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto c = [&](size_t i) {
      return i < grad.size() && grad[i].defined() ? OptTensor(grad[i].contiguous()) : OptTensor();
    };
    auto g = norm_gate_bwd(c(0), c(1), v[0], v[1], v[2], o(v[3]), o(v[4]), ctx->saved_data["c"].toDouble(),
                           ctx->saved_data["eps"].toDouble(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    const int64_t gate = ctx->saved_data["gate"].toInt();
    if (gate == 1) g[3] = g[3].view({-1});
    size_t edge = 0;  // graph edges exist for the inputs that were given, in order
    for (int i = 0; i < 5; ++i) {
      const bool given = i < 3 || (i == 3 ? gate > 0 : ctx->saved_data["next"].toBool());
      if (!given || !ctx->needs_input_grad(edge++)) g[i] = Tensor();
    }
    g.resize(7);
    return g;
  }
};

// y, skip (..., D) of one 16-bit type; fp32 vectors (as above: the shapes are checked here)
std::vector<Tensor> norm_gate(const Tensor& y, const Tensor& skip, const Tensor& wp, const OptTensor& gate,
                              const OptTensor& wn, double skip_scale, double eps) {
  const int64_t n = y.dim() ? y.size(-1) : 0;
  TORCH_CHECK_VALUE(y.dim() >= 2 && skip.sizes() == y.sizes(), "norm_gate_residual: y ", y.sizes(), " and skip ",
                    skip.sizes(), " must be of one shape (..., D)");
  TORCH_CHECK_VALUE(wp.dim() == 1 && wp.size(0) == n && (!wn || (wn->dim() == 1 && wn->size(0) == n)),
                    "norm_gate_residual: w_post and w_next must be (", n, ",)");
  TORCH_CHECK_VALUE(!gate || ((gate->dim() == 1 || (gate->dim() == 2 && gate->size(0) == y.size(0))) &&
                              gate->size(-1) == n),
                    "norm_gate_residual: gate ", gate->sizes(), " is neither (", n, ",) nor (", y.size(0), ", ", n, ")");
  if (tangents()) {
    for (const Tensor* t : {&y, &skip, &wp}) no_tangent(*t, "norm_gate_residual");
    for (const OptTensor* t : {&gate, &wn}) no_tangent(*t, "norm_gate_residual");
  }
  bool grad = false;
  if (at::GradMode::is_enabled()) {
    for (const Tensor* t : {&y, &skip, &wp}) grad = grad || t->requires_grad();
    for (const OptTensor* t : {&gate, &wn}) grad = grad || (*t && (*t)->requires_grad());
  }
  auto out = grad ? NormGateNode::apply(y, skip, wp, gate, wn, skip_scale, eps)
                  : norm_gate_fwd(y.contiguous(), skip.contiguous(), wp.contiguous(), packed_vec(gate),
                                  packed_vec(wn), skip_scale, eps);
  out.resize(2);
  return out;
}

// ------------------------------------------------------------------------------ clipping
// The blocks write all tensors at once, so none may be written that another one is read from or written to; a tensor
// may be its own result.
void check_separate(const std::vector<nsw::ClipTensor>& v) {
  if (v.empty()) return;
  struct Range {
    uintptr_t begin, end;
  };
  const auto range = [](const void* p, const nsw::ClipTensor& t) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Range{at, at + (uintptr_t)t.n * (t.dtype == nsw::kF32 ? 4 : 2)};
  };
  // the usual list is settled without sorting: results one after the other in memory, and no input among them
  const uintptr_t first = range(v.front().out, v.front()).begin, last = range(v.back().out, v.back()).end;
  uintptr_t at = 0;
  bool plain = true;
  for (const auto& t : v) {
    const Range in = range(t.in, t), out = range(t.out, t);
    plain = plain && out.begin >= at && (t.in == t.out || in.end <= first || in.begin >= last);
    at = out.end;
  }
  if (plain) return;
  std::vector<Range> read, written;  // (what is scaled in place: only written)
  read.reserve(v.size());
  written.reserve(v.size());
  for (const auto& t : v) {
    written.push_back(range(t.out, t));
    if (t.in != t.out) read.push_back(range(t.in, t));
  }
  for (auto* r : {&read, &written})
    std::sort(r->begin(), r->end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t end = 0, read_end = 0;
  size_t i = 0;
  bool apart = true;
  for (const Range& w : written) {
    apart = apart && w.begin >= end;
    for (; i < read.size() && read[i].begin < w.begin; ++i) {
      apart = apart && read[i].begin >= end;
      read_end = std::max(read_end, read[i].end);
    }
    apart = apart && w.begin >= read_end;
    end = std::max(end, w.end);
  }
  TORCH_CHECK(apart && (i == read.size() || read[i].begin >= end), "clip_grad_norm: tensors overlap");
}

// out[i] = grads[i] * min(1, max_norm / (norm + 1e-6)) (out empty: in place); returns the norm (fp32 scalar)
Tensor clip_grads(const std::vector<Tensor>& grads, double max_norm, const std::vector<Tensor>& out) {
  TORCH_CHECK(!grads.empty(), "clip_grad_norm: no tensors");
  TORCH_CHECK(out.empty() || out.size() == grads.size(), "clip_grad_norm: ", out.size(), " outputs for ",
              grads.size(), " tensors");
  const auto dev = grads[0].device();
  const bool dual = tangents();
  std::vector<nsw::ClipTensor> v;
  v.reserve(grads.size());
  int64_t total = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& g = grads[i];
    const Tensor& o = out.empty() ? g : out[i];
    if (dual) {
      no_tangent(g, "clip_grad_norm");
      no_tangent(o, "clip_grad_norm");
    }
    TORCH_CHECK(g.is_cuda() && g.device() == dev && o.device() == dev, "clip_grad_norm: tensor ", i,
                " is not on the first one's CUDA device");
    TORCH_CHECK(g.is_contiguous() && o.is_contiguous() && o.numel() == g.numel() &&
                    o.scalar_type() == g.scalar_type(),
                "clip_grad_norm: tensor ", i, " and its output must be contiguous, of one size and dtype");
    if (g.numel() == 0) continue;
    v.push_back({g.data_ptr(), o.data_ptr(), g.numel(), dt_code(g, "clip_grad_norm")});
    total += g.numel();
  }
  check_separate(v);
  const c10::cuda::CUDAGuard guard(dev);
  const auto f32 = grads[0].options().dtype(at::kFloat);
  if (v.empty()) return torch::zeros({}, f32);
  const int64_t tables = ((int64_t)v.size() + nsw::kClipTensors - 1) / nsw::kClipTensors;
  const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>(16 * sm_count(grads[0]), total / 2048 + (int64_t)v.size()));
  auto partial = torch::empty({tables * blocks + 1}, f32);
  auto norm = torch::empty({}, f32);
  check(nsw::clip_tensors(v.data(), (int)v.size(), (float)max_norm, partial.data_ptr<float>(), blocks,
                          norm.data_ptr<float>(), stream()),
        "clip_grad_norm");
  // written behind autograd's back: nodes that saved such a tensor and copies made from one have to notice
  for (const Tensor& t : out.empty() ? grads : out)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void bind_block(py::module& m) {
  m.def("gated_mlp_fwd", &gated_mlp_fwd);
  m.def("gated_mlp_bwd", &gated_mlp_bwd);
  m.def("gated_mlp", &gated_mlp);
  m.def("norm_gate", &norm_gate);
  m.def("clip_grads", &clip_grads);
}
