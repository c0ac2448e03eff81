"""Models with a relative position bias, routers and experts on the GPU: against the CPU, captured, without gradients."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import config as C  # noqa: E402
from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.models import get_model  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402
from neural_scaling_weather_b200.utils.misc import create_dummy_metadata  # noqa: E402

DEV = torch.device("cuda")
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


def build(md, rollout=1, window=(4, 8), **model):
    torch.manual_seed(0)
    return get_model(C.create(dict(
        model=dict(arch="swin", embed_dim=64, patch_size=2, depth=2, window_size=list(window), num_heads=4, dropout=0.0,
                   mlp_ratio=2, coord_pos_embed=True, mlp_type="swiglu", rel_pos_bias=True, **model),
        data=dict(invariants=["a"]), train=dict(temporal_context_window=1, num_rollout_steps=rollout),
        parallelism=dict(use_transformer_engine=False))), md)


@pytest.mark.parametrize("norm", ["pre", "sandwich"])
def test_model_matches_cpu(norm):
    """Every expert is chosen, so that no rounding changes a choice; the tolerances of the plain model's comparison
    (tests/test_model_gpu.py): bf16 activations through two blocks against fp32."""
    md = create_dummy_metadata(32, 64, 5)
    cpu = build(md, rollout=2, block_norm=norm, num_experts=3, experts_per_token=3)
    with torch.no_grad():
        for name, p in cpu.named_parameters():
            if "rel_bias" in name or "router" in name:
                p.add_(0.5 * torch.randn_like(p))
    gpu = build(md, rollout=2, block_norm=norm, num_experts=3, experts_per_token=3).cuda()
    gpu.load_state_dict(cpu.state_dict())
    x, y = torch.randn(2, 1, 6, 32, 64), torch.randn(2, 2, 5, 32, 64)
    out_c, bal_c = cpu(x, return_balance=True)
    (((out_c - y) ** 2).mean() + 0.01 * bal_c).backward()
    with torch.autocast("cuda", dtype=BF):
        out_g, bal_g = gpu(x.cuda(), return_balance=True)
    (((out_g.float() - y.cuda()) ** 2).mean() + 0.01 * bal_g).backward()
    assert rel(out_g.cpu(), out_c) < 3e-2
    assert abs(bal_g.item() - bal_c.item()) < 1e-5  # even shares, and probabilities that sum to one: 1 on either side
    grads = dict(cpu.named_parameters())
    for name, p in gpu.named_parameters():
        assert p.grad is not None and rel(p.grad.cpu(), grads[name].grad) < 8e-2, name


def test_block_is_its_operators_with_choices():
    """A block with two of six experts in bf16 parameters: bit for bit the public operators in a row, with gradients."""
    torch.manual_seed(1)
    model = build(create_dummy_metadata(16, 32, 4), num_experts=6, experts_per_token=2).model.to(DEV, BF)
    blk = model.blocks[1]
    x = torch.randn(2, 1, 8, 16, 64, device=DEV).to(BF).requires_grad_()
    got = blk(x)
    dout = torch.randn_like(got)
    params = list(blk.parameters())
    grads = torch.autograd.grad(got, [x, *params], dout)

    at, m = blk.attn, blk.mlp
    w, b = at.qkv_params()
    h = ops.rms_norm(x, blk.norm1.weight)
    a = ops.window_attention(ops.linear(h, w, b), at.q_norm.weight, at.k_norm.weight, 4, 16,
                             blk.attention_geometry(blk.shift_size), at.scale, rel_bias=at.rel_bias)
    s = ops.linear(a, at.proj.weight, at.biasproj.bias, residual=x)
    h = ops.rms_norm(s, blk.norm2.weight)
    weights, experts, _ = ops.route_tokens(ops.linear(h, m.router.weight), 2)
    want = ops.expert_mlp(h, weights, experts, m.gate.weight, m.up.weight, m.down.weight, residual=s)
    assert torch.equal(got, want)
    assert len(experts.unique()) > 1
    for p, g, e in zip([x, *params], grads, torch.autograd.grad(want, [x, *params], dout)):
        # the residual's two gradients may be summed in another order: a rounding of each (2 * 2^-8) and of the sums that
        # follow from it (as many again)
        assert rel(g, e) < 4 * 2.0 ** -8, p.shape


@pytest.mark.parametrize("tokens", ["few", "many"])
def test_rollout_without_gradients(tokens):
    """Two steps in inference mode, in a captured graph and out of it; the small grid's 8 tokens take the kernels for few assignments."""
    grid, window = ((4, 8), (2, 4)) if tokens == "few" else ((32, 64), (4, 8))
    model = build(create_dummy_metadata(*grid, 4), rollout=2, window=window, num_experts=5, experts_per_token=1).to(DEV, BF).eval()
    x = torch.randn(1, 1, 5, *grid, device=DEV).to(BF)
    with torch.no_grad():
        want = model(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph, static = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.stream(side):
            model(static)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            out = model(static)
        static.zero_()
        graph.replay()
        static.copy_(x)
        graph.replay()
    assert torch.isfinite(want).all() and torch.equal(out, want)
    with torch.inference_mode():
        assert torch.equal(model(x), want)


def test_trainer_with_experts_and_cuda_graphs(tmp_path):
    """Four training steps of the options through the trainer, from captured micro-batches."""
    import os

    from neural_scaling_weather_b200.training.trainer import Trainer

    os.environ["MASTER_PORT"] = "29542"
    t = Trainer(C.compose("default", [
        f"hydra.run.dir={tmp_path}", "parallelism.backend=nccl", "model.embed_dim=64", "model.depth=2",
        "model.num_heads=4", "model.window_size=[4,8]", "model.patch_size=2", "data.synthetic.nlat=32",
        "data.synthetic.nlon=64", "data.synthetic.n_samples=40", "data.levels=[500]", "data.batch_size=2",
        "optimizer=adamw", "optimizer.max_iterations=4", "train.log_every=2", "train.amp_dtype=bf16",
        "train.clip_grad_norm=1.0", "logging.log_to_wandb=false", "train.seed=1", "train.cuda_graphs=true",
        "model.mlp_type=swiglu", "model.mlp_ratio=2", "model.num_experts=4", "model.rel_pos_bias=true"]))
    t.launch()
    assert t.iters == 4 and t._graph is not None
    assert all(torch.isfinite(p).all() for p in t.model.parameters())
    assert 0.5 < t.logs["router_balance"] < 4
    import torch.distributed as dist

    t._graph = None
    dist.destroy_process_group()


def test_broadcast_inputs_are_their_copies():
    """Rows, experts, heads and gradients that share memory: bit for bit what their copies give."""
    torch.manual_seed(2)
    M, E, K, H, N = 300, 5, 72, 40, 64
    x, res, dy = (torch.randn(1, n, device=DEV).to(BF).expand(M, n) for n in (K, N, N))
    wg, wu = ((torch.randn(1, H, K, device=DEV) * 0.2).to(BF).expand(E, H, K) for _ in range(2))
    wd = (torch.randn(E, N, 1, device=DEV) * 0.2).to(BF).expand(E, N, H)
    z = torch.randn(1, E, device=DEV).expand(M, E)
    geom = ops.WindowGeometry(window=(4, 8), h_global=8)
    qkv, norm = torch.randn(1, 1, 8, 1, 3 * 2 * 64, device=DEV).to(BF).expand(2, 1, 8, 16, 384), torch.ones(64, device=DEV)
    table, da = torch.randn(1, geom.num_buckets(), device=DEV).expand(2, -1), torch.ones(1, device=DEV, dtype=BF).expand(2, 1, 8, 16, 128)

    def step(f):
        lx, lg, lu, ld, lz, lq, lt = leaves = [f(t).detach().requires_grad_() for t in (x, wg, wu, wd, z, qkv, table)]
        weights, experts, balance = ops.route_tokens(lz, 2)
        y = ops.expert_mlp(lx, weights, experts, lg, lu, ld, residual=f(res))
        a = ops.window_attention(lq, norm, norm, 2, 64, geom, 0.125, rel_bias=lt)
        with torch.no_grad():
            few = ops.expert_mlp(lx[:3], weights[:3], experts[:3], lg, lu, ld, residual=f(res)[:3])
            rows = ops.expert_mlp(lx, weights, experts, lg, lu, ld, residual=f(res))
        return [y, few, rows, a, balance, *torch.autograd.grad([y, a, balance], leaves, [f(dy), f(da), torch.ones_like(balance)])]

    for i, (got, want) in enumerate(zip(step(lambda t: t), step(lambda t: t.contiguous().clone()))):
        if i != 1:
            assert torch.equal(got, want)
        else:
            # w_down, whose columns are not adjacent, takes the kernels for rows sorted by expert where its copy takes
            # those for a few assignments: h, the experts' outputs and y are rounded there, h and y here, each by a
            # relative 2-norm of 2^-9, and one more for everything in fp32
            assert rel(got, want) < 6 * 2.0 ** -9


def test_two_graphs_at_once():
    """Two captured steps of attention, router and experts, replayed at the same time on two streams."""
    torch.manual_seed(3)
    model = build(create_dummy_metadata(16, 32, 4), num_experts=4, experts_per_token=2).model.to(DEV, BF)
    blk = model.blocks[1]
    params = list(blk.parameters())
    xs = [torch.randn(2, 1, 8, 16, 64, device=DEV).to(BF) for _ in range(4)]
    dout = torch.randn_like(xs[0])

    def step(x):
        x = x.detach().requires_grad_()
        y = blk(x)
        return [y.detach(), *torch.autograd.grad(y, [x, *params], dout)]

    want = [step(x) for x in xs]
    graphs = []
    for i in range(2):
        static, graph, side = xs[i].clone(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph, stream=side):
            out = step(static)
        graphs.append((static, graph, side, out))
    for use in (0, 2):
        torch.cuda.synchronize()
        for i, (static, graph, side, _) in enumerate(graphs):
            static.copy_(xs[use + i])
        torch.cuda.synchronize()
        for _ in range(5):
            for static, graph, side, _ in graphs:
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[use + i]))
