"""The routed experts: which form a call takes, and what fp16 holds of small gradients."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402
from tests.test_expert_ops_gpu import BF, DEV, HF, U, expert_exact, expert_inputs, rel  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


# experts, width, hidden width, rows an expert, rows of a tile: by 5 % or more the fastest of the three where they were
# timed (the table beside expert_tile), on 148 SMs
TILES = [
    (2, 768, 1024, 512, 64), (2, 768, 1024, 1024, 256), (2, 1024, 4096, 128, 64), (2, 1024, 4096, 512, 256), (4, 128, 344, 512, 64),
    (4, 128, 344, 1024, 256), (1, 1024, 2736, 512, 64), (1, 1024, 2736, 1024, 256), (8, 1024, 2736, 8, 32), (8, 1024, 2736, 64, 64),
    (8, 1024, 2736, 96, 256), (8, 2048, 2736, 64, 64), (8, 2048, 2736, 96, 256), (32, 768, 512, 48, 64), (32, 768, 512, 96, 256),
    (64, 512, 680, 48, 64), (64, 512, 680, 64, 256), (64, 1024, 1368, 16, 32), (64, 1024, 1368, 64, 256), (128, 256, 344, 64, 256),
    (256, 512, 128, 64, 256),
]


@pytest.mark.parametrize("E,K,H,rows,tile", TILES)
def test_tiles_are_the_fastest_measured(E, K, H, rows, tile):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the rule counts SMs")
    assert _ext.require().expert_tile(rows * E, E, H, K) == tile


@pytest.mark.parametrize("M,E,K,H", [(64, 2, 128, 1024), (200, 2, 64, 4096), (700, 64, 64, 72)])
def test_forms_agree_about_the_rule(M, E, K, H):
    """Either side of the rule's borders, against 64 bits (4 u as in test_expert_ops_gpu.py)."""
    for m in (M, 3 * M, 6 * M):
        x, wt, chosen, w, res, _ = expert_inputs(m, 2, E, K, H, K, BF, seed=m)
        assert rel(ops.expert_mlp(x, wt, chosen, *w, residual=res), expert_exact(x, wt, chosen, w, res, "silu")) < 4 * U[BF]


def rounded_backward(x, wt, chosen, w, dy, dtype, scale=1.0):
    """The backward pass of SiLU experts in 64 bits, with what is said to be rounded to `dtype` rounded: g and u, the weighted
    dy, dg and du, h, an assignment's dx.  dy times `scale` goes in, the gradients come out divided by it."""
    r = lambda t: t.to(dtype).double()  # noqa: E731
    xd, wd = x.double(), wt.double()
    dx, grads = torch.zeros_like(xd), [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in w]
    for e in range(w[0].shape[0]):
        tok, slot = torch.nonzero(chosen == e, as_tuple=True)
        wg, wu, wdn = (t[e].double() for t in w)
        g, u = xd[tok] @ wg.t(), xd[tok] @ wu.t()
        h, g, u = r(g * torch.sigmoid(g) * u), r(g), r(u)
        sig = torch.sigmoid(g)
        dys = r(wd[tok, slot][:, None] * (dy.double() * scale)[tok])
        dh = dys @ wdn
        dg, du = r(dh * u * sig * (1 + g * (1 - sig))), r(dh * g * sig)
        dx = dx.index_add(0, tok, r(dg @ wg + du @ wu))
        for i, t in enumerate((dg.t() @ xd[tok], du.t() @ xd[tok], dys.t() @ h)):
            grads[i][e] = t
    return [t / scale for t in (dx, *grads)]


@pytest.mark.parametrize("small", [1.0, 1e-2, 1e-3, 1e-4])
def test_small_gradients_in_fp16(small):
    """dy and the weights of the second choice are `small`.  What is rounded to fp16 on the way, no more, limits the gradients:
    products below 6e-5 lose bits.  A loss scale that keeps them above it gives the definition's gradients again."""
    M, E, K, H = 800, 4, 64, 72
    x, wt, chosen, w, _, dy = expert_inputs(M, 2, E, K, H, K, HF, seed=11)
    wt[:, 1] = (wt[:, 1].float() * small).to(HF)
    dy = (dy.float() * small).to(HF)

    def run(scale):
        leaves = [t.clone().requires_grad_() for t in (x, *w)]
        y = ops.expert_mlp(leaves[0], wt, chosen, *leaves[1:])
        return [t.double() / scale for t in torch.autograd.grad(y, leaves, (dy.float() * scale).to(HF))]

    # dx has six roundings, the weights' gradients five (see test_expert_ops_gpu.py); both sides have them here
    for a, b in zip(run(1.0), rounded_backward(x, wt, chosen, w, dy, HF)):
        # the result's own rounding, below 2^-14 in steps of 2^-24
        step = 2.0 ** -24 * a.numel() ** 0.5
        assert (a - b).norm() < 6 * U[HF] * b.norm() + step
    scale = 2.0 ** round(-torch.tensor(small).log2().item())  # dy near one again
    want = expert_exact(x, wt, chosen, w, None, "silu", dy)[1]
    for a, b in zip(run(scale), [want[0], *want[2:]]):
        assert rel(a, b) < 6 * U[HF]


@pytest.mark.parametrize("master", [False, True])
def test_a_single_token_without_a_batch(master):
    """x (K,), weights and experts (k,), residual (N,): one token, with its gradients."""
    x, wt, chosen, w, res, dy = expert_inputs(1, 2, 4, 64, 40, 72, BF, seed=5)
    logits = torch.randn(4, device=DEV).requires_grad_()
    weights, experts, balance = ops.route_tokens(logits, 2)
    rows = ops.route_tokens(logits[None], 2)
    assert weights.shape == experts.shape == (2,) and torch.equal(weights, rows[0][0]) and torch.equal(experts, rows[1][0])
    got, want = (torch.autograd.grad([a.sum() + 2 * a.flatten()[0], b], logits, [torch.ones_like(b)] * 2)[0]
                 for a, b in ((weights, balance), (rows[0], rows[2])))
    assert torch.equal(got, want)
    if master:
        w = [torch.nn.Parameter(t.float()) for t in w]
    leaves = [x, wt, *w, res]
    leaves = [t if isinstance(t, torch.nn.Parameter) else t.detach().requires_grad_() for t in leaves]
    args = [leaves[0], leaves[1], chosen, *leaves[2:5], leaves[5]]
    y2 = ops.expert_mlp(*args[:6], residual=args[6])
    y1 = ops.expert_mlp(args[0][0], args[1][0], chosen[0], *args[3:6], residual=args[6][0])
    assert y1.shape == (72,) and torch.equal(y1, y2[0])
    for a, b in zip(torch.autograd.grad(y1, leaves, dy[0]), torch.autograd.grad(y2, leaves, dy)):
        assert a.shape == b.shape and torch.equal(a, b)
