"""Routed experts and relative position bias on the CPU: the plain operators against their formulas, refusals, and the
model options that use them.

fp64 comparisons repeat the same sums in another order: below 1e-10 for the few hundred terms here.  fp32 ones have
2^-24 per rounding over chains of at most some hundred roundings: 1e-5 relative to the largest value."""

import math
import os

import pytest
import torch

from neural_scaling_weather_b200 import config as C
from neural_scaling_weather_b200 import ops
from neural_scaling_weather_b200.models import get_model
from neural_scaling_weather_b200.models.swin import RoutedMLP, SwinTransformer
from neural_scaling_weather_b200.utils.flops import FlopsCalculator
from neural_scaling_weather_b200.utils.misc import create_dummy_metadata
from tests.dist_utils import run

D = torch.float64


# --------------------------------------------------------------------------- router
@pytest.mark.parametrize("m,e,k,normalize", [(1, 1, 1, True), (5, 4, 2, True), (17, 9, 3, False), (3, 6, 6, False),
                                             (0, 4, 2, True)])
def test_route_is_its_formula(m, e, k, normalize):
    torch.manual_seed(0)
    z = torch.randn(m, e, dtype=D)
    w, idx, balance = ops.route_tokens(z, k, normalize)
    assert idx.dtype == torch.int64 and w.shape == idx.shape == (m, k)
    count, mean = [0] * e, [0.0] * e
    for t in range(m):
        row = z[t].tolist()
        order = sorted(range(e), key=lambda i: (-row[i], i))[:k]
        assert idx[t].tolist() == order
        total = sum(math.exp(v) for v in row)
        over = sum(math.exp(row[i]) for i in order) if normalize else total
        for j, i in enumerate(order):
            assert abs(w[t, j].item() - math.exp(row[i]) / over) < 1e-12
            count[i] += 1
        for i in range(e):
            mean[i] += math.exp(row[i]) / total / m
    want = e * sum(c / (m * k) * p for c, p in zip(count, mean)) if m else 0.0
    assert abs(balance.item() - want) < 1e-12


def test_route_ties_masks_and_shapes():
    z = torch.tensor([[1.0, 2.0, 2.0, 2.0], [-math.inf, 0.0, -math.inf, 1.0], [-math.inf] * 4], dtype=D)
    w, idx, balance = ops.route_tokens(z.view(3, 1, 4), 2)
    assert idx.view(3, 2)[:2].tolist() == [[1, 2], [3, 1]] and w.shape == (3, 1, 2)
    assert w[2].abs().max() == 0 and torch.isfinite(balance)
    assert torch.allclose(w[0], torch.full((1, 2), 0.5, dtype=D))
    even = ops.route_tokens(torch.zeros(8, 4, dtype=D), 4)[2]  # all chosen, all alike
    assert abs(even.item() - 1) < 1e-12


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient(normalize):
    torch.manual_seed(1)
    z = torch.randn(6, 5, dtype=D, requires_grad=True)
    assert torch.autograd.gradcheck(lambda v: ops.route_tokens(v, 2, normalize)[::2], z)


def test_route_refusals():
    z = torch.zeros(3, 4)
    for k in (0, 5, -1):
        with pytest.raises(ValueError, match="top_k"):
            ops.route_tokens(z, k)
    with pytest.raises(ValueError, match="top_k"):
        ops.route_tokens(torch.zeros(()), 1)


# --------------------------------------------------------------------------- experts
def _experts(m=7, k=2, e=3, kin=5, h=6, n=4, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=D)  # noqa: E731
    return (r(m, kin), torch.rand(m, k, generator=g, dtype=D), torch.randint(0, e, (m, k), generator=g),
            r(e, h, kin), r(e, h, kin), r(e, n, h), r(m, n))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_experts_are_their_formula(act):
    x, w, idx, wg, wu, wd, res = _experts()
    idx[0] = torch.tensor([1, 1])  # twice counts twice
    idx[1] = torch.tensor([-1, 3])  # outside: left out
    y = ops.expert_mlp(x, w, idx, wg, wu, wd, residual=res, activation=act)
    f = torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu
    for t in range(x.shape[0]):
        want = res[t].clone()
        for j in range(idx.shape[1]):
            e = int(idx[t, j])
            if 0 <= e < wg.shape[0]:
                want += w[t, j] * (wd[e] @ (f(wg[e] @ x[t]) * (wu[e] @ x[t])))
        assert torch.allclose(y[t], want, atol=1e-10)
    assert torch.equal(y[1], res[1])


def test_experts_gradient():
    x, w, idx, wg, wu, wd, res = _experts(m=4, kin=3, h=3, n=2)
    idx[0, 0] = -1
    leaves = [t.requires_grad_() for t in (x, w, wg, wu, wd, res)]
    assert torch.autograd.gradcheck(lambda x, w, a, b, c, r: ops.expert_mlp(x, w, idx, a, b, c, residual=r), leaves)


def test_expert_refusals():
    x, w, idx, wg, wu, wd, res = _experts()
    ok = lambda **k: ops.expert_mlp(**{**dict(x=x, weights=w, experts=idx, w_gate=wg, w_up=wu, w_down=wd), **k})  # noqa: E731
    ok()
    with pytest.raises(ValueError, match="activation"):
        ok(activation="relu")
    with pytest.raises(TypeError, match="integers"):
        ok(experts=idx.double())
    with pytest.raises(TypeError, match="integers"):
        ok(experts=idx > 0)
    for bad in (dict(w_up=wu[:, 1:]), dict(w_down=wd[1:]), dict(w_down=wd[:, :, 1:]), dict(x=x[:, 1:]),
                dict(w_gate=wg[0], w_up=wu[0])):
        with pytest.raises(ValueError, match="do not fit"):
            ok(**bad)
    for bad in (dict(weights=w[:, :1]), dict(weights=w[1:], experts=idx[1:]), dict(weights=w[None], experts=idx[None])):
        with pytest.raises(ValueError, match="must be"):
            ok(**bad)
    with pytest.raises(ValueError, match="residual"):
        ok(residual=res[:, 1:])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("lead", [(7,), (7, 1), (0,)])
def test_no_experts_a_token_is_refused(device, lead):
    dt = D if device == "cpu" else torch.bfloat16
    x = torch.zeros(*lead, 8, device=device, dtype=dt)
    none = torch.zeros(*lead, 0, device=device, dtype=dt)
    for master in (dt, torch.float32):
        w = [torch.zeros(2, 8, 8, device=device, dtype=master) for _ in range(3)]
        with pytest.raises(ValueError, match="no experts a token"):
            ops.expert_mlp(x, none, none.long(), *w)


def test_experts_under_autocast():
    """fp32 parameters under autocast, as the dense gated network takes them: products in bf16, gradients in fp32.  On the
    way to y about eight roundings (x, a weight, g or u, the activation, h, w_down, the expert's output, its weighted sum),
    each at most 2^-8 of its value: 2^-5 of the largest.  Gradients pass as many again twice (through y, whose error is in
    2 y, and back): 2^-3."""
    x, w, idx, wg, wu, wd, res = (t.float() if t.is_floating_point() else t for t in _experts(m=9, e=4))
    leaves = [t.requires_grad_() for t in (x, w, wg, wu, wd, res)]
    want = ops.expert_mlp(x, w, idx, wg, wu, wd, residual=res)
    exact = torch.autograd.grad(want.square().sum(), leaves)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        plain = ops.expert_mlp(x, w, idx, wg, wu, wd)
        y = ops.expert_mlp(x, w, idx, wg, wu, wd, residual=res)
        none = ops.expert_mlp(x, w, torch.full_like(idx, -1), wg, wu, wd)
        assert plain.dtype == none.dtype == ops.gated_mlp(x, wg[0], wu[0], wd[0]).dtype == torch.bfloat16
        assert none.abs().max() == 0
    assert (y - want).abs().max() < 2.0 ** -5 * want.abs().max()
    for a, b in zip(torch.autograd.grad(y.float().square().sum(), leaves), exact):
        assert a.dtype == torch.float32 and (a - b).abs().max() < 2.0 ** -3 * b.abs().max()


# --------------------------------------------------------------------------- relative position bias
def test_buckets_are_displacements():
    geom = ops.WindowGeometry(window=(3, 2))
    assert geom.num_buckets(2) == 3 * 5 * 3
    b = geom.relative_buckets(2)
    at = [(t, y, x) for t in range(2) for y in range(3) for x in range(2)]
    seen = {}
    for i, p in enumerate(at):
        for j, q in enumerate(at):
            d = tuple(a - c for a, c in zip(p, q))
            assert seen.setdefault(d, int(b[i, j])) == int(b[i, j])  # one bucket per displacement
    assert len(set(seen.values())) == len(seen) == geom.num_buckets(2)
    assert min(seen.values()) == 0 and max(seen.values()) == geom.num_buckets(2) - 1


def test_bias_joins_the_logits():
    torch.manual_seed(0)
    geom = ops.WindowGeometry(window=(2, 4), shift=(1, 2), mask=True, mask_shift=1, h_global=4)
    qkv, nh, hd = torch.randn(2, 1, 4, 8, 3 * 2 * 8), 2, 8
    one = torch.ones(hd)
    table = torch.randn(nh, geom.num_buckets(1))
    args = (one, one, nh, hd, geom, 0.3)
    y0 = ops.window_attention(qkv, *args)
    # a constant bias changes nothing, and zeros nothing at all
    assert torch.equal(ops.window_attention(qkv, *args, rel_bias=torch.zeros_like(table)), y0)
    assert torch.allclose(ops.window_attention(qkv, *args, rel_bias=torch.full_like(table, 2.0)), y0, atol=1e-5)
    assert not torch.allclose(ops.window_attention(qkv, *args, rel_bias=table), y0, atol=1e-2)
    # all displacements but zero masked: every query sees itself
    own = torch.full_like(table, -math.inf)
    own[:, geom.relative_buckets(1)[0, 0]] = 0.0
    v = qkv[..., 2 * nh * hd:]
    assert torch.allclose(ops.window_attention(qkv, *args, rel_bias=own), v, atol=1e-5)
    # no displacement left: zeros, with gradients of zero
    none = torch.full_like(table, -math.inf).requires_grad_()
    q = qkv.clone().requires_grad_()
    y = ops.window_attention(q, *args, rel_bias=none)
    assert y.abs().max() == 0
    y.sum().backward()
    assert torch.isfinite(q.grad).all()


def test_bias_refusals():
    geom = ops.WindowGeometry(window=(2, 4))
    qkv, one = torch.randn(1, 1, 4, 8, 3 * 2 * 8), torch.ones(8)
    n = geom.num_buckets(1)
    for bad in ((2, n - 1), (1, n), (n,), (2, 3, 5, 7)):
        with pytest.raises(ValueError, match="rel_bias"):
            ops.window_attention(qkv, one, one, 2, 8, geom, 1.0, rel_bias=torch.zeros(*bad))


# --------------------------------------------------------------------------- model options
ROUTED = dict(mlp_type="swiglu", num_experts=4, experts_per_token=2)


def _cfg(steps=1, **model):
    return C.create(dict(
        model=dict(arch="swin", embed_dim=32, patch_size=2, depth=2, window_size=[4, 8], num_heads=4, dropout=0.0,
                   mlp_ratio=2, coord_pos_embed=True, **model),
        data=dict(invariants=["a"]), train=dict(temporal_context_window=1, num_rollout_steps=steps),
        parallelism=dict(use_transformer_engine=False, micro_batch_size=1)))


@pytest.mark.parametrize("norm", ["pre", "sandwich"])
def test_routed_biased_block_is_its_formula(norm):
    torch.manual_seed(0)
    model = get_model(_cfg(rel_pos_bias=True, block_norm=norm, **ROUTED), create_dummy_metadata(16, 32, 4)).model
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.05 * torch.randn_like(p))
    x = torch.randn(2, 1, 5, 16, 32)
    s, total = model.prepare_tokens(x), 0.0
    for blk in model.blocks:
        at, m = blk.attn, blk.mlp
        assert at.rel_bias.shape == (4, 7 * 15) and isinstance(m, RoutedMLP)
        w, b = at.qkv_params()
        qkv = torch.nn.functional.linear(ops.rms_norm(s, blk.norm1.weight), torch.cat(w), torch.cat(b))
        a = ops.window_attention(qkv, at.q_norm.weight, at.k_norm.weight, 4, 8,
                                 blk.attention_geometry(blk.shift_size), at.scale, rel_bias=at.rel_bias)
        a = torch.nn.functional.linear(a, at.proj.weight, at.biasproj.bias)
        s = s + (a if norm == "pre" else blk.branch_gate1 * ops.rms_norm(a, blk.post_norm1.weight))
        h = ops.rms_norm(s, blk.norm2.weight)
        weights, experts, balance = ops.route_tokens(h @ m.router.weight.t(), 2)
        y = torch.zeros_like(h)
        for e in range(4):
            out = (torch.nn.functional.silu(h @ m.gate.weight[e].t()) * (h @ m.up.weight[e].t())) @ m.down.weight[e].t()
            y = y + out * (weights * (experts == e)).sum(-1, keepdim=True)
        s = s + (y if norm == "pre" else blk.branch_gate2 * ops.rms_norm(y, blk.post_norm2.weight))
        total = total + balance / 2
    got, balance = model(x, return_balance=True)
    assert torch.allclose(model.forward_head(s)[:, -1:], got, atol=1e-4)
    assert torch.allclose(balance, total, rtol=1e-5)
    assert torch.equal(got, model(x))  # asking for the balance changes nothing


def test_rollout_returns_the_mean_balance():
    torch.manual_seed(0)
    stepper = get_model(_cfg(steps=2, **ROUTED), create_dummy_metadata(16, 32, 4))
    x = torch.randn(1, 1, 5, 16, 32)
    out, balance = stepper(x, return_balance=True)
    first, b0 = stepper.model(x, return_balance=True)
    _, b1 = stepper.model(torch.cat([first, x[:, :, -1:]], 2), return_balance=True)
    assert out.shape[1] == 2 and torch.allclose(balance, (b0 + b1) / 2)
    balance.backward()
    assert stepper.model.blocks[0].mlp.router.weight.grad.abs().max() > 0


def test_options_validate_and_default_to_the_plain_block():
    md = create_dummy_metadata(16, 32, 4)
    names = lambda **k: set(dict(get_model(_cfg(**k), md).named_parameters()))  # noqa: E731
    assert names() == names(rel_pos_bias=False, num_experts=0)
    assert {n.split(".", 3)[-1] for n in names(rel_pos_bias=True) - names()} == {"attn.rel_bias"}
    extra = names(**ROUTED) - names(mlp_type="swiglu")
    assert {n.split(".", 3)[-1] for n in extra} == {"mlp.router.weight"}
    m = C.compose("default").model
    assert (m.rel_pos_bias, m.num_experts, m.experts_per_token) == (False, 0, 2)
    for bad in (dict(num_experts=4), dict(num_experts=4, mlp_type="gelu"), dict(num_experts=-1, mlp_type="swiglu")):
        with pytest.raises(ValueError, match="num_experts"):
            get_model(_cfg(**bad), md)
    for k in (0, 5):
        with pytest.raises(ValueError, match="experts_per_token"):
            get_model(_cfg(**{**ROUTED, "experts_per_token": k}), md)
    with pytest.raises(ValueError, match="dropout"):
        SwinTransformer(window_size=(4, 8), patch_size=2, in_chans=4, out_chans=4, embed_dim=64, depth=1, num_heads=4,
                        domain_metadata=md, mlp_type="swiglu", num_experts=2, drop_rate=0.1)
    with pytest.raises(ValueError, match="no experts"):
        get_model(_cfg(), md)(torch.randn(1, 1, 5, 16, 32), return_balance=True)


def test_flops_and_parameters_of_the_options():
    md = create_dummy_metadata(32, 64, 4)
    plain, gated = _cfg(), _cfg(mlp_type="swiglu")
    both = _cfg(rel_pos_bias=True, **ROUTED)
    count = lambda c: FlopsCalculator(c, 32, 64, 4, 4)  # noqa: E731
    tokens, e, h, L = 16 * 32, 32, 64, 32
    logits = tokens // L * 4 * L * L
    mlp = tokens * (2 * e * 4 + 5 * 4 + 2 * (6 * e * h + 9 * h + 2 * e))
    dense = tokens * (6 * e * h + 2 * h + e + 9 * h)
    got = (count(both).flops() - count(gated).flops()) * 1e12 / 2
    assert got == pytest.approx(mlp - dense + logits, rel=1e-6, abs=1.0)
    assert count(_cfg(rel_pos_bias=False, num_experts=0)).flops() == count(plain).flops()
    size = lambda c: sum(p.numel() for n, p in get_model(c, md).named_parameters() if "bias" not in n or "rel" in n)  # noqa: E731
    added = (count(both).param_count() - count(gated).param_count()) * 1e6
    assert added == pytest.approx(size(both) - size(gated), abs=1e-3)


# --------------------------------------------------------------------------- sharded
def _sharded_worker(rank, world, tp, sp1, sp2):
    import tests.test_distributed_cpu as base

    tiny = base._tiny_cfg

    def cfg():
        c = tiny()
        for name, value in dict(ROUTED, rel_pos_bias=True).items():
            c.model[name] = value
        return c

    base._tiny_cfg = cfg
    base._model_worker(rank, world, tp, sp1, sp2, 16, 32)


@pytest.mark.parametrize("tp,sp1,sp2", [(2, 1, 1), (1, 2, 1), (2, 1, 2)])
def test_routed_model_sharded_matches_single_rank(tp, sp1, sp2):
    run(_sharded_worker, tp * sp1 * sp2, tp, sp1, sp2)


def _balance_worker(rank, world):
    """Over tp every rank has the whole balance loss and its whole gradient."""
    from neural_scaling_weather_b200.parallel import comm

    torch.manual_seed(0)
    whole = RoutedMLP(16, 48, 4, 2)
    comm.init_model_parallel_info(tp=world, sp1=1, sp2=1, dp=1)
    part = RoutedMLP(16, 48, 4, 2)
    hl = 48 // world
    with torch.no_grad():
        part.router.weight.copy_(whole.router.weight)
        for a, b, dim in ((part.gate, whole.gate, 1), (part.up, whole.up, 1), (part.down, whole.down, 2)):
            a.weight.copy_(b.weight.narrow(dim, rank * hl, hl))
    x = torch.randn(2, 5, 16, requires_grad=True)
    y, balance = part(x, residual=2 * x)
    (y.square().sum() + 3 * balance).backward()
    comm_size, comm.get_size = comm.get_size, lambda *_: 1
    try:
        x1 = x.detach().clone().requires_grad_()
        y1, balance1 = whole(x1, residual=2 * x1)
        (y1.square().sum() + 3 * balance1).backward()
    finally:
        comm.get_size = comm_size
    assert torch.allclose(y, y1, atol=1e-5) and torch.equal(balance, balance1)
    assert torch.allclose(x.grad, x1.grad, atol=1e-5)
    assert torch.allclose(part.router.weight.grad, whole.router.weight.grad, atol=1e-5)


def test_router_over_tp_has_the_whole_gradient():
    run(_balance_worker, 2)


# --------------------------------------------------------------------------- trainer
OPTIONS = ["model.rel_pos_bias=true", "model.mlp_type=swiglu", "model.num_experts=4", "model.mlp_ratio=2",
           "optimizer.max_iterations=4", "train.log_every=2"]


def test_trainer_adds_the_balance_loss_and_resumes_older_runs(tmp_path):
    from neural_scaling_weather_b200.training.trainer import with_model_options
    from tests.test_trainer_cpu import _train

    weighted, free = str(tmp_path / "w.pt"), str(tmp_path / "f.pt")
    run(_train, 1, str(tmp_path / "a"), OPTIONS + ["model.router_balance_weight=10.0"], None, weighted)
    run(_train, 1, str(tmp_path / "b"), OPTIONS + ["model.router_balance_weight=0.0"], None, free)
    a, b = torch.load(weighted), torch.load(free)
    name = "module.model.blocks.0.mlp.router.weight"
    assert torch.isfinite(a[name]).all() and not torch.equal(a[name], b[name])
    lines = [r.split(",") for r in open(tmp_path / "a" / "logs.txt").read().strip().split("\n")]
    balance = [float(r[lines[0].index("router_balance")]) for r in lines[1:]]
    assert len(balance) == 2 and all(0.5 < v < 4 for v in balance)
    # a run saved before the options existed resumes, one with another value of them does not
    plain = ["optimizer.max_iterations=2", "train.log_every=2"]
    run(_train, 1, str(tmp_path / "c"), plain, None, None)
    path = os.path.join(tmp_path, "c", "hyperparameters.yaml")
    cfg = C.load(path)
    for key in ("rel_pos_bias", "num_experts", "experts_per_token", "router_balance_weight"):
        del cfg.model[key]
    C.save(cfg, path)
    run(_train, 1, str(tmp_path / "c"), plain, None, None)
    assert with_model_options({"model": {"num_experts": 2}}) != with_model_options({"model": {}})


def _logged_balance_worker(rank, world, exp_dir, options, out):
    """Trains, and keeps of each log what this rank's routers had and what was logged."""
    from neural_scaling_weather_b200.training.trainer import Trainer
    from tests.test_trainer_cpu import BASE

    t = Trainer(C.compose("default", BASE + [f"hydra.run.dir={exp_dir}"] + options))
    log, rows = t.validate_and_checkpoint, []

    def keep():
        own = (t.router_balance / max(1, t.n_mbs - t.n_mbs_last_log)).item()
        log()
        rows.append((own, t.logs["router_balance"]))

    t.validate_and_checkpoint = keep
    t.launch()
    torch.save(rows, f"{out}{rank}.pt")


@pytest.mark.parametrize("world,split", [(2, ["parallelism.sp2=2"]), (2, ["parallelism.sp1=2"]), (2, []),
                                         (4, ["parallelism.sp2=2"])])
def test_the_logged_balance_is_every_ranks(tmp_path, world, split):
    """The mean over the data-parallel (the ranks that are not split) and the spatial ranks: each routes its own tokens."""
    run(_logged_balance_worker, world, str(tmp_path / "a"), OPTIONS + split, str(tmp_path / "rank"))
    ranks = [torch.load(tmp_path / f"rank{r}.pt") for r in range(world)]
    assert len(ranks[0]) == 2
    for rows in zip(*ranks):
        own = [r[0] for r in rows]
        assert len(set(own)) == world
        for _, logged in rows:
            assert abs(logged - sum(own) / world) < 1e-5
