"""The transformer-block operators' plain forms, their checks, and the model options that use them (CPU)."""

import os
import subprocess
import sys

import pytest
import torch

from neural_scaling_weather_b200 import config as C
from neural_scaling_weather_b200 import ops
from neural_scaling_weather_b200.models import get_model
from neural_scaling_weather_b200.models.swin import SwinTransformer
from neural_scaling_weather_b200.ops import _ext
from neural_scaling_weather_b200.utils.flops import FlopsCalculator
from neural_scaling_weather_b200.utils.misc import create_dummy_metadata
from tests.dist_utils import run

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rand(*s):
    return torch.randn(*s, dtype=torch.float64, requires_grad=True)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_mlp_gradient_against_differences(act):
    torch.manual_seed(0)
    args = [_rand(3, 2, 5), _rand(7, 5), _rand(7, 5), _rand(4, 7), _rand(7), _rand(7), _rand(4), _rand(3, 2, 4)]
    f = lambda x, wg, wu, wd, bg, bu, bd, r: ops.gated_mlp(x, wg, wu, wd, bg, bu, bd, r, act)  # noqa: E731
    assert torch.autograd.gradcheck(f, args)
    x, wg, wu, wd = args[:4]
    g, u = x @ wg.t(), x @ wu.t()
    a = g * torch.sigmoid(g) if act == "silu" else g * torch.special.ndtr(g)
    assert torch.allclose(ops.gated_mlp(x, wg, wu, wd, activation=act), (a * u) @ wd.t())


@pytest.mark.parametrize("gate", ["none", "channel", "sample"])
def test_norm_gate_residual_definition(gate):
    """fp32 arithmetic of unit-scale values: a few roundings of 2^-24 each."""
    torch.manual_seed(0)
    y, skip = torch.randn(2, 3, 4, 6), torch.randn(2, 3, 4, 6)
    wp, wn = torch.rand(6) + 0.5, torch.rand(6) + 0.5
    g = {"none": None, "channel": torch.randn(6), "sample": torch.randn(2, 6)}[gate]
    s, n = ops.norm_gate_residual(y, skip, wp, g, wn, skip_scale=0.5)
    y, skip = y.double(), skip.double()
    eps = torch.finfo(torch.float32).eps
    rms = lambda v: v / (v.pow(2).mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    gg = 1.0 if g is None else (g if gate == "channel" else g[:, None, None, :])
    es = 0.5 * skip + gg * rms(y) * wp
    assert (s - es).abs().max() < 2e-6 and (n - rms(es) * wn).abs().max() < 5e-6
    assert ops.norm_gate_residual(y.float(), skip.float(), wp)[1] is None


def test_clip_grad_norm_in_place_and_out():
    grads = [torch.full((3, 2), 2.0), torch.full((4,), -1.0)]
    out = [torch.empty_like(g) for g in grads]
    norm = ops.clip_grad_norm(grads, 1.0, out=out)
    assert norm.item() == pytest.approx(28 ** 0.5, rel=1e-6) and grads[0][0, 0] == 2.0
    assert torch.cat([o.reshape(-1) for o in out]).norm().item() == pytest.approx(1.0, rel=1e-5)
    assert torch.equal(ops.clip_grad_norm(grads, 1.0), norm)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))
    before = [g.clone() for g in grads]
    ops.clip_grad_norm(grads, 100.0)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))


def test_refusals():
    x, w, wd = torch.zeros(2, 4), torch.zeros(6, 4), torch.zeros(4, 6)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_mlp(x, w, w, wd, activation="tanh")
    with pytest.raises(ValueError, match="fit together"):
        ops.gated_mlp(x, w, w[:5], wd)
    with pytest.raises(ValueError, match="residual"):
        ops.gated_mlp(x, w, w, wd, residual=torch.zeros(3, 4))
    with pytest.raises(ValueError, match="one shape"):
        ops.norm_gate_residual(x, x[:1], torch.ones(4))
    with pytest.raises(ValueError, match="w_post"):
        ops.norm_gate_residual(x, x, torch.ones(3))
    with pytest.raises(ValueError, match="gate"):
        ops.norm_gate_residual(x, x, torch.ones(4), torch.ones(3, 4))
    with pytest.raises(ValueError, match="no tensors"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grad_norm([x], -1.0)


def test_extension_refuses_with_numbers_in_the_message():
    """A refusal raised inside the extension (on tensors that claim a CUDA device but hold no memory, so nothing
    can run) reaches Python as an exception, also where the message is formatted from numbers."""
    ext = _ext.load()
    if ext is None:
        pytest.skip("extension not built")
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(4, 32, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(64, 64, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(ValueError, match=r"x \[4, 32\], w_gate \[64, 64\].* do not fit together"):
            ext.gated_mlp(x, w, w, w, None, None, None, None, 0)


@pytest.mark.parametrize("grad_mode", [False, True])
def test_extension_refuses_forward_mode_derivatives(grad_mode):
    """The kernels would return an output without a tangent, which counts as a zero derivative (on tensors that hold
    no memory, as above)."""
    ext = _ext.load()
    if ext is None:
        pytest.skip("extension not built")
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad as fw

    def dual(args, i):
        return [fw.make_dual(a, torch.zeros_like(a)) if j == i else a for j, a in enumerate(args)]

    with FakeTensorMode(), fw.dual_level(), torch.set_grad_enabled(grad_mode):
        half = lambda *s: torch.empty(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        gated = [half(4, 32), half(64, 32), half(64, 32), half(16, 64), half(64), half(64), half(16), half(4, 16)]
        for i in range(len(gated)):
            with pytest.raises(RuntimeError, match="gated_mlp: forward-mode"):
                ext.gated_mlp(*dual(gated, i), 0)
        norm = [half(2, 3, 16), half(2, 3, 16), *(torch.empty(16, device="cuda") for _ in range(3))]
        for i in range(len(norm)):
            with pytest.raises(RuntimeError, match="norm_gate_residual: forward-mode"):
                ext.norm_gate(*dual(norm, i), 1.0, 1e-6)
        with pytest.raises(RuntimeError, match="clip_grad_norm: forward-mode"):
            ext.clip_grads(dual(norm[2:], 1), 1.0, [])


@pytest.mark.parametrize("tied", [(0, 1), (1, 2), (3, 4), (0, 1, 2, 3, 4, 5), ()])
def test_in_place_gradients_of_tied_parameters(tied, monkeypatch):
    """The extension adds to all the buffers of a call at once, so no two of a call may be one parameter's: a
    parameter that is passed twice gets its gradients through autograd.  With a stand-in for the extension, whose
    forward and gradients are ones."""
    from neural_scaling_weather_b200.ops import fused, gradsink

    n, seen = 8, []

    class Ext:
        @staticmethod
        def gated_mlp_fwd(x, wg, wu, wd, *rest):
            return [torch.ones_like(x), x, x, x, x, wg, wu, wd]

        @staticmethod
        def gated_mlp_bwd(dy, x, wg, wu, wd, g, u, h, act, need, into, types):
            seen.append([t for t in into if t is not None])
            for t in seen[-1]:
                t.add_(1)
            return [None] + [None if t is not None else torch.ones(n, n) if i < 3 else torch.ones(n)
                             for i, t in enumerate(into)]

    monkeypatch.setattr(fused, "require", lambda: Ext)
    notices = []

    class Reducer:
        def notice(self, p):
            notices.append(p)

    reducer = Reducer()
    gradsink.register(reducer.notice)
    # one leaf for each place, or the same one in the tied places (a matrix cannot be a vector: ties across them none)
    ps = [torch.nn.Parameter(torch.ones(n, n)) for _ in range(3)] + [torch.nn.Parameter(torch.ones(n)) for _ in range(3)]
    for i in tied:
        ps[i] = ps[tied[0]] if (i < 3) == (tied[0] < 3) else ps[[j for j in tied if (j < 3) == (i < 3)][0]]
    for p in ps:
        p.grad = torch.zeros_like(p)
    y = fused._GatedMLP.apply(torch.ones(4, n), None, 0, *ps)
    y.sum().backward()
    gradsink.unregister(reducer.notice)
    assert len({t.data_ptr() for t in seen[0]}) == len(seen[0])
    for p in ps:
        uses = sum(q is p for q in ps)
        assert (p.grad == uses).all()
        # what autograd still has to add is not reported as written
        assert sum(q is p for q in notices) == (uses == 1)
        assert p._nsw_pending == 0


# --------------------------------------------------------------------------- model options
def _cfg(**model):
    return C.create(dict(
        model=dict(arch="swin", embed_dim=64, patch_size=2, depth=2, window_size=[4, 8], num_heads=4, dropout=0.0,
                   mlp_ratio=8 / 3, coord_pos_embed=True, **model),
        data=dict(invariants=["a"]), train=dict(temporal_context_window=1, num_rollout_steps=1),
        parallelism=dict(use_transformer_engine=False, micro_batch_size=1)))


@pytest.mark.parametrize("mlp_type", ["swiglu", "geglu"])
def test_sandwich_block_is_its_formula(mlp_type):
    torch.manual_seed(0)
    model = get_model(_cfg(mlp_type=mlp_type, block_norm="sandwich"), create_dummy_metadata(16, 32, 4)).model
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.05 * torch.randn_like(p))
    x = torch.randn(2, 1, 5, 16, 32)
    x0 = model.prepare_tokens(x)
    s = x0
    for blk in model.blocks:
        a = blk._shifted_window_attn(ops.rms_norm(s, blk.norm1.weight), None)
        s = s + blk.branch_gate1 * ops.rms_norm(a, blk.post_norm1.weight)
        h = ops.rms_norm(s, blk.norm2.weight)
        g = torch.nn.functional.linear(h, blk.mlp.gate.weight, blk.mlp.biasgate.bias)
        u = torch.nn.functional.linear(h, blk.mlp.up.weight, blk.mlp.biasup.bias)
        act = torch.nn.functional.silu if mlp_type == "swiglu" else torch.nn.functional.gelu
        m = torch.nn.functional.linear(act(g) * u, blk.mlp.down.weight, blk.mlp.biasdown.bias)
        s = s + blk.branch_gate2 * ops.rms_norm(m, blk.post_norm2.weight)
    assert torch.allclose(model.forward_head(s)[:, -1:], model(x), atol=1e-5)


def test_sandwich_blocks_are_called_as_modules():
    """Hooks on the blocks run, and a block by itself, given the stream alone, is the sandwich block."""
    torch.manual_seed(0)
    model = get_model(_cfg(mlp_type="swiglu", block_norm="sandwich"), create_dummy_metadata(16, 32, 4)).model
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.05 * torch.randn_like(p))
    streams = []
    for blk in model.blocks:
        blk.register_forward_pre_hook(lambda _, args: streams.append(args[0]))
        blk.register_forward_hook(lambda *a: streams.append(a[-1][0]))
    model(torch.randn(2, 1, 5, 16, 32))
    assert len(streams) == 2 * len(model.blocks)
    for i, blk in enumerate(model.blocks):
        before, after = streams[2 * i], streams[2 * i + 1]
        for hooks in (blk._forward_pre_hooks, blk._forward_hooks):
            hooks.clear()
        assert torch.allclose(blk(before), after, atol=1e-6)


def test_options_validate_and_default_to_the_plain_block():
    md = create_dummy_metadata(16, 32, 4)
    names = lambda **k: set(dict(get_model(_cfg(**k), md).named_parameters()))  # noqa: E731
    assert names() == names(mlp_type="gelu", block_norm="pre")
    extra = names(block_norm="sandwich") - names()
    assert {n.split(".")[-1] for n in extra} >= {"branch_gate1", "branch_gate2"}
    with pytest.raises(ValueError, match="mlp_type"):
        get_model(_cfg(mlp_type="relu"), md)
    with pytest.raises(ValueError, match="block_norm"):
        SwinTransformer(window_size=(4, 8), patch_size=2, in_chans=4, out_chans=4, embed_dim=64, depth=1, num_heads=4,
                        domain_metadata=md, block_norm="post")
    assert C.compose("default").model.mlp_type == "gelu" and C.compose("default").model.block_norm == "pre"


def test_flops_of_the_gated_network():
    """Three products of 2 embed hidden each instead of two of 2 embed 4 embed."""
    plain = FlopsCalculator(_cfg(), 32, 64, 4, 4)
    gated = FlopsCalculator(_cfg(mlp_type="swiglu"), 32, 64, 4, 4)
    tokens, e, hidden = 16 * 32, 64, int(64 * 8 / 3)
    got = (gated.flops() - plain.flops()) * 1e12 / 2
    main = tokens * (6 * e * hidden - 16 * e * e)
    small = tokens * (2 * hidden + e + 9 * hidden) - tokens * (4 * e + e + 8 * 4 * e)
    assert got == pytest.approx(main + small, rel=1e-6, abs=1.0)
    assert gated.param_count() - plain.param_count() == pytest.approx(2 * (3 * e * hidden - 8 * e * e) * 1e-6)


def _sharded_worker(rank, world, tp, sp1, sp2):
    import tests.test_distributed_cpu as base

    tiny = base._tiny_cfg

    def cfg():
        c = tiny()
        c.model["mlp_type"] = "swiglu"
        c.model["block_norm"] = "sandwich"
        return c

    base._tiny_cfg = cfg
    base._model_worker(rank, world, tp, sp1, sp2, 16, 32)


@pytest.mark.parametrize("tp,sp1,sp2", [(2, 1, 1), (1, 1, 2)])
def test_gated_sandwich_model_sharded_matches_single_rank(tp, sp1, sp2):
    run(_sharded_worker, tp * sp1 * sp2, tp, sp1, sp2)


def _all_reduces_worker(rank, world, drop):
    import torch.distributed as dist

    from neural_scaling_weather_b200.models.swin import GatedMLP
    from neural_scaling_weather_b200.parallel import comm

    comm.init_model_parallel_info(tp=world, sp1=1, sp2=1, dp=1)
    torch.manual_seed(0)
    mlp = GatedMLP(16, 48, "swiglu", drop)
    for p in mlp.parameters():
        torch.nn.init.normal_(p, std=0.2)
    x = torch.randn(2, 3, 16, requires_grad=True)
    y = mlp(x)
    plain, sizes = dist.all_reduce, []

    def counted(t, *a, **k):
        sizes.append(t.numel())
        return plain(t, *a, **k)

    dist.all_reduce = counted
    try:
        y.sum().backward()
    finally:
        dist.all_reduce = plain
    assert sizes == [x.numel()], sizes


@pytest.mark.parametrize("drop", [0.0, 0.5])
def test_gated_mlp_sums_its_input_gradient_once_over_tp(drop):
    run(_all_reduces_worker, 2, drop)


def test_example_trains_on_cpu():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "train_gated_block.py"), "--steps", "4",
                          "--dim", "64", "--depth", "1", "--grid", "36x72", "--channels", "2"], cwd=ROOT,
                         env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "rollout" in out.stdout
