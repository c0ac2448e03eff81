// PyTorch bindings of the routed experts and their router: argument checks, outputs and workspaces (from PyTorch's
// allocator, on the current stream) and the launches.
#include "bindings_util.h"

namespace {

// ------------------------------------------------------------------------------ router
nsw::RouteArgs route_args(const Tensor& logits, int64_t k, bool normalize) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1),
              "route_tokens: logits must be a CUDA matrix with adjacent columns");
  const int64_t e = logits.size(1);
  TORCH_CHECK_VALUE(e >= 1 && e <= nsw::kMaxExperts, "route_tokens: ", e, " experts are not in 1 .. ", nsw::kMaxExperts);
  TORCH_CHECK_VALUE(k >= 1 && k <= e && k <= nsw::kMaxChosen, "route_tokens: top_k ", k, " is not in 1 .. ",
                    std::min<int64_t>(e, nsw::kMaxChosen));
  nsw::RouteArgs a{};
  a.logits = logits.data_ptr();
  a.tokens = logits.size(0);
  a.ld = logits.stride(0);
  a.experts = (int)e;
  a.k = (int)k;
  a.normalize = normalize;
  a.dtype = dt_code(logits, "route_tokens");
  return a;
}

// {weights, experts, balance, share}; share: experts' shares for the backward, in front of the blocks' partial sums
std::vector<Tensor> route_fwd(const Tensor& logits, int64_t k, bool normalize) {
  nsw::RouteArgs a = route_args(logits, k, normalize);
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto weights = torch::empty({a.tokens, k}, f32);
  auto chosen = torch::empty({a.tokens, k}, logits.options().dtype(at::kLong));
  auto balance = torch::empty({}, f32);
  const int blocks = nsw::route_blocks(a.tokens, a.experts, sm_count(logits));
  auto share = torch::empty({(2 * (int64_t)blocks + 1) * a.experts}, f32);
  a.weights = weights.data_ptr<float>();
  a.chosen = chosen.data_ptr<int64_t>();
  a.balance = balance.data_ptr<float>();
  a.share = share.data_ptr<float>();
  a.partial = a.share + a.experts;
  check(nsw::route_fwd(a, blocks, stream()), "route_tokens");
  return {weights, chosen, balance, share};
}

Tensor route_bwd(const Tensor& logits, const Tensor& weights, const Tensor& chosen, const Tensor& share,
                 const OptTensor& dweights, const OptTensor& dbalance, bool normalize) {
  nsw::RouteArgs a = route_args(logits, weights.size(1), normalize);
  const auto like = [&](const OptTensor& t, int64_t n) {
    TORCH_CHECK(!t || (t->device() == logits.device() && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                       t->numel() == n),
                "route_tokens backward: gradients must be contiguous fp32 tensors of the outputs' sizes");
  };
  like(dweights, weights.numel());
  like(dbalance, 1);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto d = torch::empty(logits.sizes(), logits.options());
  if (a.tokens == 0) return d;
  a.weights = weights.data_ptr<float>();
  a.chosen = chosen.data_ptr<int64_t>();
  a.share = share.data_ptr<float>();
  a.dweights = dweights ? dweights->data_ptr<float>() : nullptr;
  a.dbalance = dbalance ? dbalance->data_ptr<float>() : nullptr;
  a.dlogits = d.data_ptr();
  check(nsw::route_bwd(a, sm_count(logits), stream()), "route_tokens backward");
  return d;
}

struct RouteNode : public torch::autograd::Function<RouteNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, int64_t k,
                                                bool normalize) {
    const Tensor z = flat(logits), zu = z.stride(1) == 1 || z.size(1) == 1 ? z : z.contiguous();
    auto r = route_fwd(zu, k, normalize);
    ctx->save_for_backward({zu, r[0], r[1], r[3]});
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["shape"] = logits.sizes().vec();
    ctx->set_materialize_grads(false);
    const Tensor chosen = unflat(r[1], logits);
    ctx->mark_non_differentiable({chosen});
    return {unflat(r[0], logits), chosen, r[2]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    once_differentiable("route_tokens");
    const auto v = ctx->get_saved_variables();
    const auto f32 = [](const Tensor& t) {
      return t.defined() ? OptTensor(t.to(at::kFloat).contiguous()) : OptTensor();
    };
    const Tensor d = route_bwd(v[0], v[1], v[2], v[3], f32(grad[0]), f32(grad[2]), ctx->saved_data["normalize"].toBool());
    return {d.view(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor()};
  }
};

// logits (..., E) -> (weights (..., k), experts (..., k), balance)
std::tuple<Tensor, Tensor, Tensor> route_tokens(const Tensor& logits, int64_t k, bool normalize) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "route_tokens: logits ", logits.sizes());
  if (tangents()) no_tangent(logits, "route_tokens");
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto r = RouteNode::apply(logits, k, normalize);
    return {r[0], r[1], r[2]};
  }
  const Tensor z = flat(logits);
  auto r = route_fwd(z.stride(1) == 1 || z.size(1) == 1 ? z : z.contiguous(), k, normalize);
  return {unflat(r[0], logits), unflat(r[1], logits), r[2]};
}

// ------------------------------------------------------------------------------ experts
struct ExpertShape {
  int64_t M, k, A, E, K, H, N, Kp, Hp, Np, rows;
  int tile;
};

void check_stack(const Tensor& t, at::IntArrayRef sizes, const Tensor& x, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), "expert_mlp: ", name, " must be on the input's device");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), "expert_mlp: ", name, " must have the compute dtype ", x.scalar_type(),
              ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == sizes, "expert_mlp: ", name, " must be ", sizes, ", got ", t.sizes());
}

// weights as [E, rows, cols] or, in the backward, as the forward's matrices [E rows, cols]
ExpertShape expert_shape(const Tensor& x, const Tensor& weights, int64_t E, int64_t H, int64_t N) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "expert_mlp: x must be a CUDA matrix");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "expert_mlp: bf16 or fp16, got ",
              x.scalar_type());
  ExpertShape d{};
  d.M = x.size(0);
  d.K = x.size(1);
  d.k = weights.size(1);
  d.A = d.M * d.k;
  d.E = E;
  d.H = H;
  d.N = N;
  TORCH_CHECK_VALUE(E >= 1 && E <= nsw::kMaxExperts, "expert_mlp: ", E, " experts are not in 1 .. ", nsw::kMaxExperts);
  TORCH_CHECK_VALUE(d.k >= 1 && d.k <= nsw::kMaxChosen, "expert_mlp: ", d.k, " experts a token are not in 1 .. ",
                    nsw::kMaxChosen);
  TORCH_CHECK_VALUE(d.K > 0 && H > 0 && N > 0, "expert_mlp: empty weights");
  const int64_t most = int64_t(1) << 30;
  TORCH_CHECK_VALUE(d.M < most && d.A < most && d.K < most && H < most && N < most, "expert_mlp: too many rows or features");
  d.Kp = round8(d.K);
  d.Hp = round8(H);
  d.Np = round8(N);
  d.tile = nsw::kExpertTile;
  d.rows = d.tile * nsw::expert_tiles(d.A, E, d.tile);
  return d;
}

// the plan's arrays, one behind the other
int64_t plan_size(const ExpertShape& d) {
  return 1 + d.rows / d.tile + d.E + 1 + d.A + d.rows + nsw::expert_plan_hist(d.A, d.E);
}
nsw::ExpertPlan plan_of(const ExpertShape& d, const Tensor& t, const int64_t* experts) {
  nsw::ExpertPlan p{};
  p.experts = experts;
  p.count = d.A;
  p.num_experts = (int)d.E;
  p.tile = d.tile;
  p.tiles = t.data_ptr<int>();
  p.rows = p.tiles + 1 + d.rows / d.tile;
  p.row_of = p.rows + d.E + 1;
  p.src_of = p.row_of + d.A;
  p.hist = p.src_of + d.rows;
  return p;
}

// y[t] = residual[t] + sum_j weights[t, j] MLP_experts[t, j](x[t]); experts int64, outside [0, E): left out.  With save,
// also what the backward reads: {y, xs, g, u, h, ys, plan, wg, wu, wd} (rows sorted by expert; matrices [E rows, cols]).
std::vector<Tensor> expert_mlp_fwd(const Tensor& x, const Tensor& weights, const Tensor& experts, const Tensor& wg,
                                   const Tensor& wu, const Tensor& wd, const OptTensor& residual, int64_t act,
                                   bool save) {
  TORCH_CHECK_VALUE(wg.dim() == 3 && wd.dim() == 3 && weights.dim() == 2 && x.dim() == 2,
                    "expert_mlp: x and weights are matrices, the experts' weights of three dimensions");
  ExpertShape d = expert_shape(x, weights, wg.size(0), wg.size(1), wd.size(1));
  check_stack(wg, {d.E, d.H, d.K}, x, "w_gate");
  check_stack(wu, {d.E, d.H, d.K}, x, "w_up");
  check_stack(wd, {d.E, d.N, d.H}, x, "w_down");
  TORCH_CHECK_VALUE(weights.size(0) == d.M && experts.sizes() == weights.sizes(), "expert_mlp: weights ", weights.sizes(),
                    " and experts ", experts.sizes(), " must be [", d.M, ", k]");
  TORCH_CHECK(weights.device() == x.device() && experts.device() == x.device(),
              "expert_mlp: weights and experts must be on the input's device");
  TORCH_CHECK(experts.scalar_type() == at::kLong && experts.is_contiguous() && weights.is_contiguous(),
              "expert_mlp: experts are contiguous int64, weights contiguous");
  TORCH_CHECK(!residual || (residual->device() == x.device() && residual->scalar_type() == x.scalar_type() &&
                            residual->dim() == 2 && residual->size(0) == d.M && residual->size(1) == d.N),
              "expert_mlp: residual must be [", d.M, ", ", d.N, "] in the compute dtype on the input's device");
  const int wdt = dt_code(weights, "expert_mlp: weights"), dtype = dt_code(x, "x");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto opt = x.options();
  auto y = torch::empty({d.M, d.N}, opt);
  if (d.M == 0) {
    if (!save) return {y};
    auto e = torch::empty({0, 1}, opt);
    return {y, e, e, e, e, e, torch::empty({0}, opt.dtype(at::kInt)), wg.flatten(0, 1), wu.flatten(0, 1),
            wd.flatten(0, 1)};
  }
  const auto unit = [](const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1; };
  const Tensor xu = unit(x) ? x : x.contiguous();
  const OptTensor res = !residual || unit(*residual) ? residual : OptTensor(residual->contiguous());
  const Tensor g2 = wg.flatten(0, 1), u2 = wu.flatten(0, 1), d2 = wd.flatten(0, 1);
  if (!save && nsw::expert_few_pays(d.A, d.H, d.K, d.N) && unit(g2) && unit(u2) && unit(d2)) {
    auto h = torch::empty({d.A, d.Hp}, opt);
    nsw::ExpertFew f{};
    f.x = xu.data_ptr();
    f.wg = g2.data_ptr();
    f.wu = u2.data_ptr();
    f.wd = d2.data_ptr();
    f.weights = weights.data_ptr();
    f.residual = res ? res->data_ptr() : nullptr;
    f.experts = experts.data_ptr<int64_t>();
    f.h = h.data_ptr();
    f.y = y.data_ptr();
    f.ldx = xu.stride(0);
    f.ldwg = g2.stride(0);
    f.ldwu = u2.stride(0);
    f.ldwd = d2.stride(0);
    f.ldh = d.Hp;
    f.ldres = res ? res->stride(0) : 0;
    f.tokens = (int)d.M;
    f.k = (int)d.k;
    f.num_experts = (int)d.E;
    f.K = (int)d.K;
    f.H = (int)d.H;
    f.N = (int)d.N;
    f.act = (int)act;
    f.dtype = dtype;
    f.weight_dtype = wdt;
    check(nsw::expert_few(f, stream()), "expert_mlp");
    return {y};
  }
  if (!save) {
    d.tile = nsw::expert_tile(d.A, d.E, d.H, d.N);
    d.rows = d.tile * nsw::expert_tiles(d.A, d.E, d.tile);
  }
  Aligner al;
  const Rows ga = al.add(g2), ua = al.add(u2), da = al.add(d2);
  al.run();
  auto plan = torch::empty({plan_size(d)}, opt.dtype(at::kInt));
  const nsw::ExpertPlan p = plan_of(d, plan, experts.data_ptr<int64_t>());
  check(nsw::expert_plan(p, stream()), "expert_mlp plan");
  auto xs = torch::empty({d.rows, d.Kp}, opt);
  nsw::ExpertGather gather{};
  gather.plan = &p;
  gather.k = d.k;
  gather.n = d.K;
  gather.rows = xu.data_ptr();
  gather.ld_rows = xu.stride(0);
  gather.dst = xs.data_ptr();
  gather.ld_dst = d.Kp;
  gather.dtype = dtype;
  check(nsw::expert_gather(gather, true, stream()), "expert_mlp gather");
  const nsw::GatedGroups groups{d.E, p.tiles, p.rows, p.tile};
  auto h = torch::empty({d.rows, d.Hp}, opt);
  Tensor g, u;
  nsw::GatedArgs up{}, down{};
  up.mode = nsw::kGatedUp;
  down.mode = nsw::kGatedDown;
  up.dtype = down.dtype = dtype;
  up.act = (int)act;
  up.groups = down.groups = &groups;
  up.M = down.M = d.rows;
  up.N = d.H;
  up.K = d.K;
  up.a0 = xs.data_ptr();
  up.lda = d.Kp;
  up.b0 = ga.ptr();
  up.ldb0 = ga.ld;
  up.b1 = ua.ptr();
  up.ldb1 = ua.ld;
  up.out0 = h.data_ptr();
  up.ldout = d.Hp;
  if (save) {
    g = torch::empty({d.rows, d.Hp}, opt);
    u = torch::empty({d.rows, d.Hp}, opt);
    up.out1 = g.data_ptr();
    up.out2 = u.data_ptr();
    up.ldaux = d.Hp;
  }
  check(nsw::gated_product(up, d.tile < nsw::kExpertTile, stream()), "expert_mlp up");
  auto ys = torch::empty({d.rows, d.Np}, opt);
  down.N = d.N;
  down.K = d.H;
  down.a0 = h.data_ptr();
  down.lda = d.Hp;
  down.b0 = da.ptr();
  down.ldb0 = da.ld;
  down.out0 = ys.data_ptr();
  down.ldout = d.Np;
  check(nsw::gated_product(down, d.tile < nsw::kExpertTile, stream()), "expert_mlp down");
  nsw::ExpertCombine c{};
  c.row_of = p.row_of;
  c.tokens = d.M;
  c.k = d.k;
  c.n = d.N;
  c.rows = ys.data_ptr();
  c.ld_rows = d.Np;
  c.weights = weights.data_ptr();
  c.weight_dtype = wdt;
  c.residual = res ? res->data_ptr() : nullptr;
  c.ld_res = res ? res->stride(0) : 0;
  c.out = y.data_ptr();
  c.ld_out = d.N;
  c.dtype = dtype;
  check(nsw::expert_combine(c, true, stream()), "expert_mlp combine");
  if (!save) return {y};
  return {y, xs, g, u, h, ys, plan, ga.t, ua.t, da.t};
}

// {dx, dweights, dwg, dwu, dwd}, of which those with need set are computed; an entry is undefined where it is not
// needed or was added into its fp32 buffer in `into` (three weights).  types: of the three weights' parameters.
std::vector<Tensor> expert_mlp_bwd(const Tensor& dy, const Tensor& weights, int64_t E, int64_t K, const Tensor& xs,
                                   const Tensor& g, const Tensor& u, const Tensor& h, const Tensor& ys,
                                   const Tensor& plan, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act,
                                   const std::vector<bool>& need, const std::vector<OptTensor>& into,
                                   const std::vector<at::ScalarType>& types) {
  TORCH_CHECK(need.size() == 5 && into.size() == 3 && types.size() == 3, "expert_mlp backward: x, weights, three matrices");
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2 && dy.size(0) == weights.size(0) && dy.scalar_type() == wg.scalar_type() &&
                  E >= 1 && wg.dim() == 2 && wd.dim() == 2 && wg.size(0) % E == 0 && wd.size(0) % E == 0 &&
                  wg.size(1) == K && dy.size(1) == wd.size(0) / E && weights.is_contiguous(),
              "expert_mlp backward: arguments do not fit together");
  check_apart(into, "expert_mlp backward");
  const c10::cuda::CUDAGuard guard(dy.device());
  const auto opt = dy.options();
  ExpertShape d = expert_shape(dy, weights, E, wg.size(0) / E, wd.size(0) / E);
  d.K = K;
  d.Kp = round8(K);
  std::vector<Tensor> out(5);
  const std::vector<int64_t> sizes[3] = {{E, d.H, d.K}, {E, d.H, d.K}, {E, d.N, d.H}};
  if (d.M == 0) {
    if (need[0]) out[0] = torch::empty({0, d.K}, opt);
    if (need[1]) out[1] = torch::empty(weights.sizes(), weights.options());
    for (int i = 0; i < 3; ++i)
      if (need[2 + i] && !into[i]) out[2 + i] = torch::zeros(sizes[i], opt.dtype(types[i]));
    return out;
  }
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.numel() == plan_size(d) && xs.size(0) == d.rows &&
                  xs.size(1) == d.Kp && ys.size(1) == d.Np && g.size(1) == d.Hp && u.sizes() == g.sizes() &&
                  h.sizes() == g.sizes() && rows_aligned(wg) && rows_aligned(wu) && rows_aligned(wd),
              "expert_mlp backward: saved tensors must be as the forward returned them");
  const nsw::ExpertPlan p = plan_of(d, plan, nullptr);
  const nsw::GatedGroups groups{E, p.tiles, p.rows, p.tile};
  const int dtype = dt_code(dy, "dy"), wdt = dt_code(weights, "weights");
  const Tensor dyu = dy.stride(1) == 1 || dy.size(1) == 1 ? dy : dy.contiguous();
  GradOut grad[3];
  for (int i = 0; i < 3; ++i)
    if (need[2 + i]) grad[i] = GradOut(into[i], sizes[i], dy, types[i]);
  auto dys = torch::empty({d.rows, d.Np}, opt);
  nsw::ExpertGather gather{};
  gather.plan = &p;
  gather.k = d.k;
  gather.n = d.N;
  gather.rows = dyu.data_ptr();
  gather.ld_rows = dyu.stride(0);
  gather.dst = dys.data_ptr();
  gather.ld_dst = d.Np;
  gather.other = ys.data_ptr();
  gather.ld_other = d.Np;
  gather.weights = weights.data_ptr();
  gather.weight_dtype = wdt;
  gather.dtype = dtype;
  if (need[1]) {
    out[1] = torch::empty(weights.sizes(), weights.options());
    gather.dweights = out[1].data_ptr();
  }
  check(nsw::expert_gather(gather, false, stream()), "expert_mlp backward gather");
  const auto ld_of = [](const Tensor& t) { return t.size(0) == 1 ? round8(t.size(1)) : t.stride(0); };
  const bool need_hidden = need[0] || need[2] || need[3];
  Tensor dgu;
  char* du = nullptr;
  if (need_hidden) {
    dgu = torch::empty({d.rows, 2 * d.Hp}, opt);
    du = reinterpret_cast<char*>(dgu.data_ptr()) + 2 * d.Hp;
    nsw::GatedArgs a{};
    a.mode = nsw::kGatedDh;
    a.dtype = dtype;
    a.act = (int)act;
    a.groups = &groups;
    a.M = d.rows;
    a.N = d.H;
    a.K = d.N;
    a.a0 = dys.data_ptr();
    a.lda = d.Np;
    a.b0 = wd.data_ptr();
    a.ldb0 = ld_of(wd);
    a.in0 = g.data_ptr();
    a.in1 = u.data_ptr();
    a.ldin = d.Hp;
    a.out0 = dgu.data_ptr();
    a.out1 = du;
    a.ldout = a.ldaux = 2 * d.Hp;
    check(nsw::gated_product(a, false, stream()), "expert_mlp dh");
  }
  if (need[0]) {
    auto dxs = torch::empty({d.rows, d.Kp}, opt);
    nsw::GatedArgs b{};
    b.mode = nsw::kGatedDx;
    b.dtype = dtype;
    b.groups = &groups;
    b.M = d.rows;
    b.N = d.K;
    b.K = d.H;
    b.a0 = dgu.data_ptr();
    b.a1 = du;
    b.lda = 2 * d.Hp;
    b.b0 = wg.data_ptr();
    b.ldb0 = ld_of(wg);
    b.b1 = wu.data_ptr();
    b.ldb1 = ld_of(wu);
    b.out0 = dxs.data_ptr();
    b.ldout = d.Kp;
    check(nsw::gated_product(b, false, stream()), "expert_mlp dx");
    out[0] = torch::empty({d.M, d.K}, opt);
    nsw::ExpertCombine c{};
    c.row_of = p.row_of;
    c.tokens = d.M;
    c.k = d.k;
    c.n = d.K;
    c.rows = dxs.data_ptr();
    c.ld_rows = d.Kp;
    c.out = out[0].data_ptr();
    c.ld_out = d.K;
    c.dtype = dtype;
    check(nsw::expert_combine(c, true, stream()), "expert_mlp dx sum");
  }
  if (need[2] || need[3] || need[4]) {
    nsw::GatedDwArgs w{};
    w.dtype = dtype;
    w.T = d.rows;
    w.groups = &groups;
    const auto dst = [&](int i) { return need[2 + i] ? grad[i].t.data_ptr() : nullptr; };
    w.w[0] = {need_hidden ? dgu.data_ptr() : nullptr, xs.data_ptr(), 2 * d.Hp, d.Kp, d.H, d.K, dst(0), grad[0].f32,
              grad[0].into};
    w.w[1] = {du, xs.data_ptr(), 2 * d.Hp, d.Kp, d.H, d.K, dst(1), grad[1].f32, grad[1].into};
    w.w[2] = {dys.data_ptr(), h.data_ptr(), d.Np, d.Hp, d.N, d.H, dst(2), grad[2].f32, grad[2].into};
    check(nsw::gated_dw(w, stream()), "expert_mlp weight gradients");
    for (int i = 0; i < 3; ++i)
      if (need[2 + i]) out[2 + i] = grad[i].result(types[i]);
  }
  return out;
}

// The network of parameters in the compute type as one autograd node (fp32 master parameters, whose gradients may go
// straight into the optimizer's buffers, go through the Python node on the same two functions).
struct ExpertNode : public torch::autograd::Function<ExpertNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weights,
                        const Tensor& experts, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        const OptTensor& residual, int64_t act) {
    const Tensor w2 = flat(weights).contiguous();
    auto r = expert_mlp_fwd(flat(x), w2, flat(experts).contiguous(), wg, wu, wd, flat(residual), act, true);
    ctx->save_for_backward({w2, r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8], r[9]});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["weights"] = weights.sizes().vec();
    ctx->saved_data["experts"] = wg.size(0);
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = residual.has_value();
    return unflat(r[0], x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad) {
    once_differentiable("expert_mlp");
    const auto v = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    std::vector<bool> need(5);
    for (int i = 0; i < 5; ++i) need[i] = ctx->needs_input_grad(i < 2 ? i : i + 1);
    auto g = expert_mlp_bwd(flat(grad[0]), v[0], ctx->saved_data["experts"].toInt(), shape.back(), v[1], v[2], v[3], v[4],
                            v[5], v[6], v[7], v[8], v[9], ctx->saved_data["act"].toInt(), need, std::vector<OptTensor>(3),
                            std::vector<at::ScalarType>(3, v[7].scalar_type()));
    if (need[0]) g[0] = g[0].view(shape);
    if (need[1]) g[1] = g[1].view(ctx->saved_data["weights"].toIntVector());
    const bool need_res = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(6);
    return {g[0], g[1], Tensor(), g[2], g[3], g[4], need_res ? grad[0] : Tensor(), Tensor()};
  }
};

// x (..., K), weights and experts (int64) (..., k), residual (..., N); x, the matrices and residual in one 16-bit type
Tensor expert_mlp(const Tensor& x, const Tensor& weights, const Tensor& experts, const Tensor& wg, const Tensor& wu,
                  const Tensor& wd, const OptTensor& residual, int64_t act) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && wg.dim() == 3 && wd.dim() == 3 && wu.sizes() == wg.sizes() &&
                        wd.size(0) == wg.size(0) && wd.size(2) == wg.size(1) && x.size(-1) == wg.size(2),
                    "expert_mlp: x ", x.sizes(), ", w_gate ", wg.sizes(), ", w_up ", wu.sizes(), " and w_down ",
                    wd.sizes(), " do not fit together");
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK_VALUE(weights.sizes() == experts.sizes() && weights.dim() == x.dim() &&
                        weights.sizes().slice(0, x.dim() - 1) == lead,
                    "expert_mlp: weights ", weights.sizes(), " and experts ", experts.sizes(), " are not (", lead, ", k)");
  TORCH_CHECK_VALUE(weights.size(-1) >= 1, "expert_mlp: no experts a token");
  TORCH_CHECK_VALUE(!residual || (residual->dim() == x.dim() && residual->size(-1) == wd.size(1) &&
                                  residual->sizes().slice(0, x.dim() - 1) == lead),
                    "expert_mlp: residual ", residual->sizes(), " is not the output's shape");
  if (tangents()) {
    for (const Tensor* t : {&x, &weights, &wg, &wu, &wd}) no_tangent(*t, "expert_mlp");
    no_tangent(residual, "expert_mlp");
  }
  bool grad = false;
  if (at::GradMode::is_enabled()) {
    for (const Tensor* t : {&x, &weights, &wg, &wu, &wd}) grad = grad || t->requires_grad();
    grad = grad || (residual && residual->requires_grad());
  }
  if (grad) return ExpertNode::apply(x, weights, experts, wg, wu, wd, residual, act);
  return unflat(expert_mlp_fwd(flat(x), flat(weights).contiguous(), flat(experts).contiguous(), wg, wu, wd,
                               flat(residual), act, false)[0], x);
}

}  // namespace

void bind_experts(py::module& m) {
  m.def("route_tokens", &route_tokens);
  m.def("expert_mlp", &expert_mlp);
  m.def("expert_mlp_fwd", &expert_mlp_fwd);
  m.def("expert_mlp_bwd", &expert_mlp_bwd);
  m.def("expert_tile", &nsw::expert_tile);
}
