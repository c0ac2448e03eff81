"""The transformer-block operators (gated feed-forward network, norms with gate and skip connection, gradient
clipping) against their definitions in 64 bits, on inputs that are exact in the tested type.

Tolerances are relative 2-norms, counted in unit roundoffs u of the 16-bit type (2^-9 for bf16, 2^-11 for fp16:
round to nearest): each value that a kernel rounds to 16 bits on the way to a result adds at most u to that
result's relative error (the operators are products and sums of such values; act' has relative condition at most
about one).  fp32 sums of up to 2^16 terms stay far below u."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402

DEV = torch.device("cuda")
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


# --------------------------------------------------------------------------- gated feed-forward network
def gated_inputs(M, K, H, N, dtype, bias, residual, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * std).to(dtype)

    w = [randn(H, K, std=K ** -0.5), randn(H, K, std=K ** -0.5), randn(N, H, std=H ** -0.5)]
    b = [randn(H, std=0.3), randn(H, std=0.3), randn(N, std=0.3)] if bias else [None] * 3
    return randn(M, K), w, b, (randn(M, N) if residual else None), randn(M, N)


def gated_exact(x, w, b, res, act, dy=None):
    ws = [t.detach().double().requires_grad_() for t in [x] + list(w)]
    bs = [None if t is None else t.detach().double().requires_grad_() for t in b]
    g = torch.nn.functional.linear(ws[0], ws[1], bs[0])
    u = torch.nn.functional.linear(ws[0], ws[2], bs[1])
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    y = torch.nn.functional.linear(a * u, ws[3], bs[2])
    if res is not None:
        y = y + res.double()
    if dy is None:
        return y.detach()
    leaves = ws + [t for t in bs if t is not None]
    return y.detach(), torch.autograd.grad(y, leaves, dy.double())


GATED_SIZES = [(1, 64, 64, 64), (1, 1024, 2736, 1024), (7, 96, 130, 40), (8, 33, 65, 31), (37, 128, 344, 128),
               (64, 100, 99, 101), (65, 64, 72, 64), (257, 200, 520, 136), (513, 129, 343, 127),
               (1000, 256, 682, 256), (128, 8, 8, 8), (300, 1, 1, 1)]


@pytest.mark.parametrize("M,K,H,N", GATED_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias,residual", [("silu", True, True), ("gelu", False, False), ("gelu", True, False)])
def test_gated_forward(M, K, H, N, dtype, act, bias, residual):
    """Rounded on the way: h and y.  The few-token and the general kernels at odd and aligned sizes."""
    x, w, b, res, _ = gated_inputs(M, K, H, N, dtype, bias, residual)
    y = ops.gated_mlp(x, *w, *b, residual=res, activation=act)
    assert y.shape == (M, N) and y.dtype == dtype and y.is_contiguous()
    assert rel(y, gated_exact(x, w, b, res, act)) < 2 * U[dtype]


@pytest.mark.parametrize("M,K,H,N", [s for s in GATED_SIZES if s[1] > 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False)])
def test_gated_backward(M, K, H, N, dtype, act, bias):
    """Rounded on the way to a gradient: g, u, one of h / dg / du, and the gradient itself."""
    x, w, b, res, dy = gated_inputs(M, K, H, N, dtype, bias, True)
    leaves = [t.requires_grad_() for t in [x] + w + [t for t in b if t is not None] + [res]]
    y = ops.gated_mlp(x, *w, *b, residual=res, activation=act)
    got = torch.autograd.grad(y, leaves, dy)
    ey, exact = gated_exact(x, w, b, res.detach(), act, dy)
    assert rel(y, ey) < 2 * U[dtype]
    assert torch.equal(got[-1], dy)
    for i, (a, e) in enumerate(zip(got[:-1], exact)):
        assert a.shape == e.shape and a.dtype == dtype
        assert rel(a, e) < 4 * U[dtype], i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False)])
def test_gated_backward_of_single_features(dtype, act, bias):
    """With one feature a weight's gradient is one sum over the tokens, which can cancel: the roundings are
    then relative to the sum of the terms' absolute values, not to the result."""
    x, w, b, res, dy = gated_inputs(300, 1, 1, 1, dtype, bias, True)
    leaves = [t.requires_grad_() for t in [x] + w + [t for t in b if t is not None]]
    got = torch.autograd.grad(ops.gated_mlp(x, *w, *b, residual=res, activation=act), leaves, dy)
    parts = [gated_exact(x[i:i + 1], w, b, None, act, dy[i:i + 1])[1] for i in range(300)]
    assert rel(got[0], torch.cat([p[0] for p in parts])) < 4 * U[dtype]
    for i in range(1, len(got)):
        terms = torch.stack([p[i].reshape(()) for p in parts])
        assert abs(got[i].double().sum() - terms.sum()) < 4 * U[dtype] * terms.abs().sum()


@pytest.mark.parametrize("M", [5, 300])
def test_gated_strides_and_batches(M):
    """Row slices, transposed weights, unaligned starts and leading dimensions give the contiguous result."""
    x, w, b, res, _ = gated_inputs(M, 96, 136, 64, torch.bfloat16, True, True)
    y = ops.gated_mlp(x, *w, *b, residual=res)
    wide = torch.zeros(M, 2, 100, device=DEV, dtype=x.dtype)
    wide[:, 1, 3:99] = x
    odd = torch.zeros(136 * 96 + 1, device=DEV, dtype=x.dtype)
    odd[1:] = w[0].reshape(-1)
    y2 = ops.gated_mlp(wide[:, 1, 3:99], odd[1:].view(136, 96), w[1].t().contiguous().t(), w[2], *b,
                       residual=res.t().contiguous().t())
    assert torch.equal(y, y2)
    y3 = ops.gated_mlp(x.view(M, 1, 1, 96), *w, *b, residual=res.view(M, 1, 1, 64))
    assert y3.shape == (M, 1, 1, 64) and torch.equal(y3.view(M, 64), y)


def test_gated_empty():
    x, w, b, res, _ = gated_inputs(3, 64, 128, 64, torch.bfloat16, True, False)
    for grad in (False, True):
        e = x[:0].clone().requires_grad_(grad)
        leaves = [t.requires_grad_(grad) for t in w + b]
        y = ops.gated_mlp(e, *w, *b)
        assert y.shape == (0, 64)
    got = torch.autograd.grad(y, [e] + leaves, torch.zeros_like(y))
    assert got[0].shape == e.shape
    assert all(t.shape == p.shape and not t.any() for t, p in zip(got[1:], leaves))


@pytest.mark.parametrize("M", [3, 400])
def test_gated_infinite_rows_stay_in_their_rows(M):
    """An inf or NaN token spoils its own output row only; large gates saturate without NaN."""
    x, w, b, _, _ = gated_inputs(M, 64, 72, 64, torch.bfloat16, True, False)
    y = ops.gated_mlp(x, *w, *b)
    bad = x.clone()
    bad[1, 5] = float("inf")
    bad[2, 7] = float("nan")
    yb = ops.gated_mlp(bad, *w, *b)
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(yb[keep], y[keep]) and not torch.isfinite(yb[2]).any()
    big = ops.gated_mlp(x * 2.0 ** 60, *w)
    assert not torch.isnan(ops.gated_mlp(x * 2.0 ** 10, *w)).any() and big.shape == y.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_fp32_parameters_and_in_place_gradients(dtype):
    """fp32 parameters under autocast: gradients of the parameters' type, added into an existing fp32
    ``.grad`` by the kernels, and the same on a second backward."""
    x, w, b, _, dy = gated_inputs(200, 64, 96, 64, dtype, True, False)
    params = [torch.nn.Parameter(t.float()) for t in w + b]
    with torch.autocast("cuda", dtype=dtype):
        got = torch.autograd.grad(ops.gated_mlp(x, *params), params, dy)
        _, exact = gated_exact(x, w, b, None, "silu", dy)
        for a, e in zip(got, exact[1:]):
            assert a.dtype == torch.float32 and rel(a, e) < 4 * U[dtype]
        for p in params:
            p.grad = torch.ones_like(p)
        for _ in range(2):
            ops.gated_mlp(x, *params).backward(dy)
    for p, a in zip(params, got):
        assert rel(p.grad, 1 + 2 * a.double()) < 1e-5


def test_gated_gradient_against_differences():
    """Directional derivative of sum(y dy) in 64 bits against the kernels' gradients."""
    x, w, b, _, dy = gated_inputs(130, 64, 136, 64, torch.float16, True, False)
    leaves = [t.requires_grad_() for t in [x] + w + b]
    got = torch.autograd.grad(ops.gated_mlp(x, *w, *b, activation="gelu"), leaves, dy)
    dirs = [torch.randn_like(t, dtype=torch.float64) for t in leaves]
    f = lambda s: (gated_exact(*(lambda v: (v[0], v[1:4], v[4:]))([t.detach().double() + s * d for t, d in  # noqa: E731
                                                                 zip(leaves, dirs)]), None, "gelu")
                   * dy.double()).sum()
    step = 1e-5
    diff = (f(step) - f(-step)) / (2 * step)
    dot = sum((g.double() * d).sum() for g, d in zip(got, dirs))
    scale = sum((g.double() * d).norm() for g, d in zip(got, dirs))
    assert abs(diff - dot) < 8 * U[torch.float16] * scale


@pytest.mark.parametrize("M", [9, 700])
def test_gated_is_deterministic_and_runs_on_the_current_stream(M):
    x, w, b, res, dy = gated_inputs(M, 128, 344, 128, torch.bfloat16, True, True)
    leaves = [t.requires_grad_() for t in [x] + w + b]

    def step():
        y = ops.gated_mlp(x, *w, *b, residual=res)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    first = step()
    with torch.no_grad():
        plain = ops.gated_mlp(x, *w, *b, residual=res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
        again_plain = ops.gated_mlp(x.detach(), *[t.detach() for t in w + b], residual=res)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(again, first))
    assert torch.equal(plain, again_plain)


def test_gated_refusals():
    x, w, b, res, _ = gated_inputs(4, 64, 72, 64, torch.bfloat16, True, True)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_mlp(x, *w, activation="relu")
    with pytest.raises(ValueError, match="fit together"):
        ops.gated_mlp(x[:, :32], *w)
    with pytest.raises(ValueError, match="residual"):
        ops.gated_mlp(x, *w, residual=res[:2])
    with pytest.raises(RuntimeError, match="b_gate"):
        ops.gated_mlp(x, *w, b[0][:8])
    with pytest.raises(RuntimeError, match="share a dtype"):
        ops.gated_mlp(x, *w, b[0], b[1].float())
    with pytest.raises(RuntimeError, match="device"):
        ops.gated_mlp(x, w[0].cpu(), w[1], w[2])
