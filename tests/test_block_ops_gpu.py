"""The transformer-block operators (gated feed-forward network, norms with gate and skip connection, gradient
clipping) against their definitions in 64 bits, on inputs that are exact in the tested type.

Tolerances are relative 2-norms, counted in u, 2^-9 for bf16 and 2^-11 for fp16 (the largest relative rounding
error is 2^-8 in bf16; over the spread of a tensor's significands its 2-norm is below 2^-9): each value that a kernel rounds to 16 bits on the way to a result adds at most u to that
result's relative error (the operators are products and sums of such values; act' has relative condition at most
about one).  fp32 sums of up to 2^16 terms stay far below u."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402
from neural_scaling_weather_b200.ops import weights as wcache  # noqa: E402

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


@pytest.mark.parametrize("rows", ["packed", "offset", "broadcast", "transposed"])
def test_gated_many_tokens_of_odd_widths(rows):
    """Results and residuals whose rows are not 16-byte aligned, with enough tokens for the tiled kernels."""
    M, K, H, N = 9003, 517, 1371, 519
    x, w, b, res, dy = gated_inputs(M, K, H, N, torch.bfloat16, True, True)
    if rows == "offset":
        res = torch.nn.functional.pad(res, (1, 2))[:, 1:-2]
    elif rows == "broadcast":
        res = res[:1].expand(M, N)
    elif rows == "transposed":
        res = res.t().contiguous().t()
    leaves = [t.requires_grad_() for t in [x] + w + b]
    y = ops.gated_mlp(x, *w, *b, residual=res)
    assert y.shape == (M, N) and y.is_contiguous()
    got = torch.autograd.grad(y, leaves, dy)
    ey, exact = gated_exact(x, w, b, res, "silu", dy)
    assert rel(y, ey) < 2 * U[torch.bfloat16]
    for i, (a, e) in enumerate(zip(got, exact)):
        assert rel(a, e) < 4 * U[torch.bfloat16], i
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(x, *w, *b, residual=res), y)


@pytest.mark.parametrize("M", [8, 40, 700, 12000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gated_tail_of_the_gate(M, dtype, act):
    """Every element of h, dg and du at gates of -6 to 6, with weights of ones that pick single features, so that
    the gates, the up projections and dh are exact.  An element's own rounding (2^-8 or 2^-11; half the spacing of
    fp16's subnormals) and 2e-5: the activation's approximations are below 1e-5 each, the slope's two terms cancel
    to no less than half of them except around its zero (an absolute 1e-6 of terms of at most one)."""
    H = 256
    eye, none = torch.eye(H, device=DEV, dtype=dtype), torch.zeros(H, H, device=DEV, dtype=dtype)
    w = [torch.cat([eye, none], 1), torch.cat([none, eye], 1), eye.clone()]
    gen = torch.Generator(device=DEV).manual_seed(1)
    gates = (torch.rand(M, H, generator=gen, device=DEV) * 12 - 6).to(dtype)
    g = gates.double().requires_grad_()
    a = torch.nn.functional.silu(g) if act == "silu" else g * torch.special.ndtr(g)
    (slope,) = torch.autograd.grad(a.sum(), g)
    a = a.detach()
    u, tiny = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype], 2.0 ** -25 * (dtype == torch.float16)
    for up, d in [(2.0 ** 13, 1.0), (1.0, 2.0 ** 13)]:  # large enough that fp16 holds the tail in normal numbers
        x = torch.cat([gates, torch.full_like(gates, up)], 1).requires_grad_()
        y = ops.gated_mlp(x, *w, activation=act)
        (dx,) = torch.autograd.grad(y, x, torch.full_like(y, d))
        with torch.no_grad():
            y2 = ops.gated_mlp(x, *w, activation=act)
        for got, exact in [(y, up * a), (y2, up * a), (dx[:, H:], d * a)]:
            assert ((got.double() - exact).abs() <= (u + 2e-5) * exact.abs() + tiny).all()
        exact = d * up * slope
        assert ((dx[:, :H].double() - exact).abs() <= (u + 2e-5) * exact.abs() + 1e-6 * d * up).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_many_tokens_of_aligned_widths(dtype, act):
    """The forms of a full grid: the pair kernel with residual and results by TMA, a wave of whole tiles of the weight
    gradients and the tiles that are left cut along the tokens (84 tiles for 74 pairs)."""
    M, K, H, N = 9001, 1024, 1600, 1024
    x, w, b, res, dy = gated_inputs(M, K, H, N, dtype, True, True)
    leaves = [t.requires_grad_() for t in [x] + w + b]
    y = ops.gated_mlp(x, *w, *b, residual=res, activation=act)
    got = torch.autograd.grad(y, leaves, dy)
    ey, exact = gated_exact(x, w, b, res, act, dy)
    assert rel(y, ey) < 2 * U[dtype]
    for i, (a, e) in enumerate(zip(got, exact)):
        assert rel(a, e) < 4 * U[dtype], i
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(x, *w, *b, residual=res, activation=act), y)


@pytest.mark.parametrize("M", [1, 2, 8, 9, 15, 16, 17])
@pytest.mark.parametrize("K,H,N", [(64, 72, 64), (1024, 2736, 1024), (1031, 2051, 517), (128, 4096, 24)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gated_few_tokens(M, K, H, N, dtype):
    """Up to 16 tokens without gradients: one and two groups of eight, whole and partly filled, one and several depth
    slices; 17 tokens, and any number with gradients: the tiled kernels.  Each token by itself (its 2-norm over the N
    outputs, of which there may be few: 4 u) and all of them."""
    x, w, b, res, _ = gated_inputs(M, K, H, N, dtype, True, True)
    exact = gated_exact(x, w, b, res, "silu")
    with torch.no_grad():
        y = ops.gated_mlp(x, *w, *b, residual=res)
    t = ops.gated_mlp(x.requires_grad_(), *w, *b, residual=res)
    for out in (y, t):
        assert rel(out, exact) < 2 * U[dtype]
        assert ((out.double() - exact).norm(dim=-1) < 4 * U[dtype] * exact.norm(dim=-1)).all()


@pytest.mark.parametrize("M", [3, 400])
def test_gated_large_gates(M):
    """Gates of 2^60: the sigmoid is 0 or 1, and the values are those of finite arithmetic."""
    x, w, b, _, _ = gated_inputs(M, 64, 72, 64, BF16, False, False)
    big = x * 2.0 ** 60
    y = ops.gated_mlp(big, *w)
    e = gated_exact(big, w, b, None, "silu")
    assert torch.isfinite(y).all() and rel(y, e) < 2 * U[BF16]


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


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_gated_strided_biases(M, dt):
    x, w, b, _, dy = gated_inputs(M, 64, 96, 64, BF16, True, False)
    b = [t.to(dt) for t in b]
    strided = [torch.stack([t, 0 * t], 1)[:, 0] for t in b]
    assert not any(t.is_contiguous() for t in strided)
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(x, *w, *strided), ops.gated_mlp(x, *w, *b))
    leaves = [[t.requires_grad_() for t in v] for v in (strided, b)]
    got, ref = (torch.autograd.grad(ops.gated_mlp(x, *w, *v), v, dy) for v in leaves)
    assert all(torch.equal(a, e) for a, e in zip(got, ref))


def test_gated_gradients_keep_their_own_types():
    """A bias in fp32 beside 16-bit ones gets its fp32 sums (of 300 terms: 1e-6 of their absolute values), and a weight
    in fp32 beside 16-bit ones the gradient that it has among fp32 ones."""
    x, w, b, _, dy = gated_inputs(300, 64, 96, 64, BF16, True, False)
    b = [b[0].requires_grad_(), b[1].requires_grad_(), b[2].float().requires_grad_()]
    got = torch.autograd.grad(ops.gated_mlp(x, *w, *b), b, dy)
    assert [t.dtype for t in got] == [BF16, BF16, F32]
    assert (got[2].double() - dy.double().sum(0)).norm() <= 1e-6 * dy.double().abs().sum(0).norm()
    for mixed in (0, 1, 2):  # one parameter in fp32 among 16-bit ones
        ps = [p.clone().float() if i == mixed else p.clone() for i, p in enumerate(w)]
        all32 = [p.float().requires_grad_() for p in w]
        ps = [p.requires_grad_() for p in ps]
        got = torch.autograd.grad(ops.gated_mlp(x, *ps), ps, dy)
        ref = torch.autograd.grad(ops.gated_mlp(x, *all32), all32, dy)
        for i, (a, e) in enumerate(zip(got, ref)):
            assert torch.equal(a, e if i == mixed else e.to(BF16))


@pytest.mark.parametrize("M,K,H,N", [(9001, 1024, 1600, 1024), (4003, 515, 1373, 517)])
def test_gated_in_place_gradients_of_many_tokens(M, K, H, N):
    """fp32 parameters with an existing ``.grad``: whole tiles add to it in the product's epilogue, cut ones in the
    kernel that adds their pieces.  Two backwards onto ones: the fp32 sums twice, exact to their roundings (1e-5)."""
    x, w, b, _, dy = gated_inputs(M, K, H, N, torch.bfloat16, True, False)
    params = [torch.nn.Parameter(t.float()) for t in w + b]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = torch.autograd.grad(ops.gated_mlp(x, *params), params, dy)
        for p in params:
            p.grad = torch.ones_like(p)
        at = [p.grad.data_ptr() for p in params]
        for _ in range(2):
            ops.gated_mlp(x, *params).backward(dy)
    _, exact = gated_exact(x, w, b, None, "silu", dy)
    for p, a, e, q in zip(params, got, exact[1:], at):
        assert p.grad.data_ptr() == q and rel(p.grad, 1 + 2 * a.double()) < 1e-5
        assert a.dtype == torch.float32 and rel(a, e) < 4 * U[torch.bfloat16]


def test_gated_tied_parameters_and_shared_gradient_buffers():
    """One parameter as both projections and one bias for both: their gradients add up in an existing fp32 ``.grad``
    as in separate ones (two fp32 sums in another order).  Buffers that overlap are refused."""
    x, w, b, _, dy = gated_inputs(1500, 256, 512, 256, torch.bfloat16, True, False)
    sep = [torch.nn.Parameter(t.float()) for t in (w[0], w[0], w[2], b[0], b[0], b[2])]
    got = torch.autograd.grad(ops.gated_mlp(x, *sep), sep, dy)
    tied = [torch.nn.Parameter(t.float()) for t in (w[0], w[2], b[0], b[2])]
    for p in tied:
        p.grad = torch.zeros_like(p)
    for _ in range(2):
        ops.gated_mlp(x, tied[0], tied[0], tied[1], tied[2], tied[2], tied[3]).backward(dy)
    for p, e in zip(tied, (got[0] + got[1], got[2], got[3] + got[4], got[5])):
        assert rel(p.grad, 2 * e) < 1e-6
    ext = _ext.require()
    _, *saved = ext.gated_mlp_fwd(x, *w, None, None, None, None, 0, True)
    x2, g, u, h, *ws = saved
    flat = torch.zeros(2 * 512 * 256, device=DEV)
    for at in (0, 512 * 256 - 4):
        into = [flat[:512 * 256].view(512, 256), flat[at:at + 512 * 256].view(512, 256)] + [None] * 4
        with pytest.raises(RuntimeError, match="overlap"):
            ext.gated_mlp_bwd(dy, x2, *ws, g, u, h, 0, [False] + [True] * 3 + [False] * 3, into, [torch.float32] * 6)
    assert not flat.any()


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


@pytest.mark.parametrize("M", [33, 600])
def test_gated_some_gradients_only(M):
    """Frozen weights, a frozen input, a single bias, and a residual alone: the asked gradients are the full
    call's, the others are not computed."""
    x, w, b, res, dy = gated_inputs(M, 64, 136, 64, torch.bfloat16, True, True)
    full = [t.clone().requires_grad_() for t in [x] + w + b + [res]]
    ref = torch.autograd.grad(ops.gated_mlp(*full[:7], residual=full[7]), full, dy)
    for pick in ([0], [2], [3, 6], [7], [0, 4]):
        args = [t.clone().requires_grad_(i in pick) for i, t in enumerate([x] + w + b + [res])]
        got = torch.autograd.grad(ops.gated_mlp(*args[:7], residual=args[7]), [args[i] for i in pick], dy)
        assert all(torch.equal(g, ref[i]) for g, i in zip(got, pick))
    one = [x, *w, None, b[1].clone().requires_grad_(), None]
    y = ops.gated_mlp(*one)
    (db,) = torch.autograd.grad(y, [one[5]], dy)
    _, exact = gated_exact(x, w, [None, b[1], None], None, "silu", dy)
    assert rel(db, exact[-1]) < 4 * U[torch.bfloat16]


@pytest.mark.parametrize("native", [True, False])
def test_gated_frozen_parameters_cost_no_gradient_memory(native):
    x, w, b, _, dy = gated_inputs(64, 1024, 2048, 1024, BF16, True, False)
    size = w[0].numel()
    ps = [torch.nn.Parameter(t if native else t.float(), requires_grad=False) for t in w + b]

    def peak(pick):
        for i, p in enumerate(ps):
            p.requires_grad_(i in pick)
        got = torch.autograd.grad(ops.gated_mlp(x, *ps), [ps[i] for i in pick], dy)
        del got
        y = ops.gated_mlp(x, *ps)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        at = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, [ps[i] for i in pick], dy)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - at

    each = size * (2 if native else 4)
    all3 = peak([0, 1, 2])
    for i in range(3):
        assert peak([i]) <= all3 - 1.9 * each, i


@pytest.mark.parametrize("M,K,H,N", [(40, 100, 72, 64), (3000, 256, 520, 264), (9001, 1024, 1600, 1024)])
@pytest.mark.parametrize("native", [True, False])
def test_gated_any_subset_of_gradients(M, K, H, N, native):
    """Each parameter's gradient by itself and several of them.  Another number of tiles may cut a weight's tokens into
    other pieces: fp32 sums in another order (1e-5), then the same rounding (half of u where some round apart)."""
    x, w, b, _, dy = gated_inputs(M, K, H, N, torch.bfloat16, True, False)
    make = lambda t: t.clone() if native else torch.nn.Parameter(t.float())  # noqa: E731
    full = [x.clone().requires_grad_()] + [make(t).requires_grad_() for t in w + b]
    ref = torch.autograd.grad(ops.gated_mlp(*full), full, dy)
    for pick in [[i] for i in range(7)] + [[1, 3], [2, 3], [0, 5], [3, 6], [1, 2, 4], [0, 2, 3, 6]]:
        args = [x.clone()] + [make(t) for t in w + b]
        for i, t in enumerate(args):
            t.requires_grad_(i in pick)
        got = torch.autograd.grad(ops.gated_mlp(*args), [args[i] for i in pick], dy)
        for a, i in zip(got, pick):
            assert a.dtype == ref[i].dtype
            assert rel(a, ref[i]) < (0.5 * U[torch.bfloat16] if a.dtype == torch.bfloat16 else 1e-5), (pick, i)


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


# --------------------------------------------------------------------------- norms, gate, skip
def norm_inputs(S, R, D, dtype, gate, nxt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s, std=1.0, mean=0.0, dt=dtype):
        return (torch.randn(*s, generator=g, device=DEV) * std + mean).to(dt)

    f = torch.float32
    gt = {"none": None, "channel": randn(D, std=0.5, dt=f), "sample": randn(S, D, std=0.5, dt=f)}[gate]
    return (randn(S, R, D), randn(S, R, D, std=2.0), randn(D, std=0.2, mean=1.0, dt=f), gt,
            randn(D, std=0.2, mean=1.0, dt=f) if nxt else None, randn(S, R, D), randn(S, R, D))


def norm_exact(y, skip, wp, gate, wn, c, ds=None, dn=None):
    """Outputs, and with gradients their values and the sums of the absolute terms of the vectors' gradients."""
    eps = torch.finfo(torch.float32).eps
    y, skip, wp = (t.detach().double().requires_grad_() for t in (y, skip, wp))
    S, D = y.shape[0], y.shape[-1]
    shape = (S,) + (1,) * (y.dim() - 2) + (D,)
    full = torch.ones(y.shape, dtype=torch.float64, device=DEV)
    gf = full if gate is None else full * (gate.double() if gate.dim() == 1 else gate.double().view(shape))
    gf = gf.requires_grad_()  # gradients of every row's gate; summed below
    wf = wp.expand(y.shape).detach().requires_grad_()
    rms = lambda v: v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)  # noqa: E731
    s = c * skip + gf * rms(y) * wf
    outs, grads, leaves = [s], [ds], [y, skip, wf, gf]
    if wn is not None:
        nf = wn.double().expand(y.shape).detach().requires_grad_()
        outs.append(rms(s) * nf)
        grads.append(dn)
        leaves.append(nf)
    res = [o.detach() for o in outs]
    if ds is None and dn is None:
        return res
    use = [(o, g.double()) for o, g in zip(outs, grads) if g is not None]
    got = torch.autograd.grad([o for o, _ in use], leaves, [g for _, g in use], allow_unused=True)
    got = [torch.zeros_like(t) if g is None else g for g, t in zip(got, leaves)]
    rows = tuple(range(y.dim() - 1))
    per = rows if gate is None or gate.dim() == 1 else rows[1:]
    vec = [(got[2].sum(rows), got[2].abs().sum(rows)), (got[3].sum(per), got[3].abs().sum(per))]
    if wn is not None:
        vec.append((got[4].sum(rows), got[4].abs().sum(rows)))
    return res, got[:2], vec


NORM_SIZES = [(1, 1, 1024), (1, 1, 1), (3, 5, 8), (2, 33, 96), (4, 257, 520), (3, 77, 1001), (2, 300, 1024),
              (1, 64, 1544), (2, 21, 4096), (1, 9, 6001), (1, 3, 16384), (300, 2, 64)]


@pytest.mark.parametrize("S,R,D", NORM_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gate,nxt", [("sample", True), ("channel", True), ("none", False)])
def test_norm_gate_residual(S, R, D, dtype, gate, nxt):
    """Tensors: one rounding at the end (u) of fp32 arithmetic.  Vectors (fp32): sums over the rows, each row's
    term a few fp32 roundings, relative to the sum of the terms' absolute values."""
    y, skip, wp, gt, wn, ds, dn = norm_inputs(S, R, D, dtype, gate, nxt)
    leaves = [t.requires_grad_() for t in (y, skip, wp, gt, wn) if t is not None]
    s, n = ops.norm_gate_residual(y, skip, wp, gt, wn, skip_scale=0.7)
    assert s.dtype == dtype and s.shape == y.shape and (n is None) == (not nxt)
    outs = [s] if n is None else [s, n]
    got = torch.autograd.grad(outs, leaves, [ds, dn][:len(outs)])
    exact, tens, vec = norm_exact(y, skip, wp, gt, wn, 0.7, ds, dn if nxt else None)
    with torch.no_grad():
        s2, n2 = ops.norm_gate_residual(y, skip, wp, gt, wn, skip_scale=0.7)
    assert torch.equal(s, s2) and (n is None or torch.equal(n, n2))
    for i, (a, e) in enumerate(zip(outs + list(got[:2]), exact + list(tens))):
        if y.numel() == 1 and i < len(outs):  # one number: the exact one, rounded
            assert torch.equal(a, e.to(dtype))
            continue
        # rows of one element: the gradient through a norm is 0 up to eps, a difference of equal numbers
        tol = (U[dtype] + 1e-5) * e.norm() + 1e-6 * ds.double().norm() * (D == 1)
        assert (a.double() - e).norm() <= tol
    if gt is None:
        vec.pop(1)
    for a, (e, terms) in zip(got[2:], vec):
        assert a.dtype == torch.float32 and a.shape == e.shape
        assert (a.double() - e).norm() <= 1e-5 * terms.norm()


@pytest.mark.parametrize("S,R,D", [(3, 1001, 131), (1, 2500, 2033), (37, 90, 515), (2, 1500, 250), (1, 1100, 1290),
                                   (2, 700, 1028), (5, 300, 3), (1, 70, 2045), (2, 2500, 768), (1, 900, 1536)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("start", [0, 1])
def test_norm_gate_residual_rows_anywhere(S, R, D, dtype, start):
    """Rows that begin anywhere in a 16-byte group, many for each block, also in tensors that begin off one.  Each
    element: its own rounding (2^-8 or 2^-11) and fp32 arithmetic, 1e-5 of the tensor's largest value.  An infinite
    row leaves its neighbours, which share its first and last groups, as they are."""
    y, skip, wp, gt, wn, ds, dn = norm_inputs(S, R, D, dtype, "sample", True)
    exact, tens, vec = norm_exact(y, skip, wp, gt, wn, 0.7, ds, dn)
    if start:
        y = torch.cat([y.new_zeros(1), y.reshape(-1)])[1:].view(S, R, D)
    leaves = [t.requires_grad_() for t in (y, skip, wp, gt, wn)]
    outs = ops.norm_gate_residual(y, skip, wp, gt, wn, skip_scale=0.7)
    got = torch.autograd.grad(outs, leaves, [ds, dn])
    for a, e in zip(list(outs) + list(got[:2]), exact + list(tens)):
        assert ((a.double() - e).abs() <= {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype] * e.abs()
                + 1e-5 * e.abs().max()).all()
    for a, (e, terms) in zip(got[2:], vec):
        assert (a.double() - e).norm() <= 1e-5 * terms.norm()
    with torch.no_grad():
        keep = torch.ones(S, R, dtype=torch.bool, device=DEV)
        keep[0, 1::3] = keep[-1, R - 1] = False
        y[~keep] = float("inf")
        again = ops.norm_gate_residual(y, skip, wp, gt, wn, skip_scale=0.7)
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(again, outs))


@pytest.mark.parametrize("D", [255, 256, 257, 513, 769, 1025, 1537, 2041, 2042, 2048, 2056, 4097, 6096, 6097, 6104, 6144,
                               6152, 8192, 8193, 12000, 12289, 16383])
def test_norm_gate_residual_widths_where_the_kernel_changes(D):
    """At each form's widest and narrowest rows, and where its shared memory passes the default limit."""
    y, skip, wp, gt, wn, ds, dn = norm_inputs(2, 11, D, torch.bfloat16, "sample", True)
    leaves = [t.requires_grad_() for t in (y, skip, wp, gt, wn)]
    outs = ops.norm_gate_residual(*leaves)
    got = torch.autograd.grad(outs, leaves, [ds, dn])
    exact, tens, vec = norm_exact(y, skip, wp, gt, wn, 1.0, ds, dn)
    for a, e in zip(list(outs) + list(got[:2]), exact + list(tens)):
        assert rel(a, e) < U[torch.bfloat16] + 1e-5
    for a, (e, terms) in zip(got[2:], vec):
        assert (a.double() - e).norm() <= 1e-5 * terms.norm()


@pytest.mark.parametrize("only", ["stream", "normed"])
def test_norm_gate_residual_with_one_output_used(only):
    y, skip, wp, gt, wn, ds, dn = norm_inputs(2, 19, 200, torch.bfloat16, "sample", True)
    leaves = [t.requires_grad_() for t in (y, skip, wp, gt, wn)]
    s, n = ops.norm_gate_residual(y, skip, wp, gt, wn)
    out, g = (s, ds) if only == "stream" else (n, dn)
    got = torch.autograd.grad(out, leaves, g, allow_unused=True)
    _, tens, vec = norm_exact(y, skip, wp, gt, wn, 1.0, ds if only == "stream" else None,
                              dn if only == "normed" else None)
    for a, e in zip(got[:2], tens):
        assert rel(a, e) < U[torch.bfloat16] + 1e-5
    for a, (e, terms) in zip(got[2:], vec):
        assert (a.double() - e).norm() <= 1e-5 * terms.norm()


@pytest.mark.parametrize("D", [512, 1001, 3000, 2301, 7001, 9000])
def test_norm_gate_residual_some_gradients_only(D):
    """Each input's gradient by itself and several of them are the full call's; what is not asked for takes no
    memory (in rows of up to 8192)."""
    y, skip, wp, gt, wn, ds, dn = norm_inputs(2, 500, D, torch.bfloat16, "sample", True)

    def step(pick):
        args = [t.clone().requires_grad_(i in pick) for i, t in enumerate((y, skip, wp, gt, wn))]
        outs = ops.norm_gate_residual(*args)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        at = torch.cuda.memory_allocated()
        got = torch.autograd.grad(outs, [args[i] for i in pick], [ds, dn])
        return got, torch.cuda.max_memory_allocated() - at

    ref, peak = step(range(5))
    ref, peak = step(range(5))
    size = y.numel() * y.element_size()
    for pick in ([0], [1], [2], [3], [4], [0, 3], [1, 4], [2, 3, 4]):
        got, used = step(pick)
        assert all(torch.equal(a, ref[i]) for a, i in zip(got, pick))
        if D <= 8192:
            assert used <= peak - 0.99 * size * sum(i not in pick for i in (0, 1)), pick


def test_norm_gate_residual_strides_zeros_and_infinities():
    """Non-contiguous inputs; a zero row and a zero branch stay finite; an infinite row spoils itself only."""
    y, skip, wp, gt, wn, _, _ = norm_inputs(2, 12, 136, torch.bfloat16, "sample", True)
    s, n = ops.norm_gate_residual(y, skip, wp, gt, wn)
    wide = torch.zeros(2, 12, 300, device=DEV, dtype=y.dtype)
    wide[..., 7:143] = y
    s2, n2 = ops.norm_gate_residual(wide[..., 7:143], skip.transpose(0, 1).contiguous().transpose(0, 1),
                                    wp.repeat_interleave(2)[::2], gt.t().contiguous().t(), wn)
    assert torch.equal(s, s2) and torch.equal(n, n2)
    y5 = y.view(2, 1, 3, 4, 136)
    s5, n5 = ops.norm_gate_residual(y5, skip.view_as(y5), wp, gt, wn)
    assert torch.equal(s5.view_as(s), s) and torch.equal(n5.view_as(n), n)
    y[0, 3], skip[0, 3] = 0, 0
    y[1, 4, 7] = float("inf")
    s3, n3 = ops.norm_gate_residual(y, skip, wp, gt, wn)
    assert not s3[0, 3].any() and not n3[0, 3].any()
    keep = torch.ones(2, 12, dtype=torch.bool, device=DEV)
    keep[0, 3] = keep[1, 4] = False
    assert torch.equal(s3[keep], s[keep]) and torch.equal(n3[keep], n[keep])
    assert torch.isnan(s3[1, 4]).any()


def test_norm_gate_residual_empty_and_refusals():
    y, skip, wp, gt, wn, _, _ = norm_inputs(2, 3, 64, torch.bfloat16, "sample", True)
    e = y[:, :0].clone().requires_grad_()
    w = wp.clone().requires_grad_()
    s, n = ops.norm_gate_residual(e, skip[:, :0], w, gt, wn)
    assert s.shape == (2, 0, 64) and n.shape == s.shape
    de, dw = torch.autograd.grad([s, n], [e, w], [s.detach(), n.detach()])
    assert de.shape == e.shape and not dw.any()
    with pytest.raises(ValueError, match="skip"):
        ops.norm_gate_residual(y, skip[:1], wp, gt, wn)
    with pytest.raises(ValueError, match="w_post"):
        ops.norm_gate_residual(y, skip, wp[:8], gt, wn)
    with pytest.raises(ValueError, match="gate"):
        ops.norm_gate_residual(y, skip, wp, gt[:1], wn)
    with pytest.raises(RuntimeError, match="width"):
        z = torch.zeros(1, 1, 16385, device=DEV, dtype=y.dtype)
        ops.norm_gate_residual(z, z, torch.ones(16385, device=DEV))


def test_norm_gate_residual_empty_batch():
    y, skip, wp, gt, wn, _, _ = norm_inputs(2, 3, 64, BF16, "sample", True)
    leaves = [t.clone().requires_grad_() for t in (y[:0], skip[:0], wp, gt[:0], wn)]
    s, n = ops.norm_gate_residual(*leaves)
    got = torch.autograd.grad([s, n], leaves, [torch.zeros_like(s), torch.zeros_like(n)])
    assert all(g.shape == t.shape and not g.any() for g, t in zip(got, leaves))


# --------------------------------------------------------------------------- gradient clipping
def clip_inputs(shapes, dtypes, std=0.1):
    g = torch.Generator(device=DEV).manual_seed(3)
    return [(torch.randn(s, generator=g, device=DEV) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("shapes,dtypes", [
    ([(1,)], [F32]), ([(7,), (0,), (1, 1)], [BF16]), ([(64, 64), (64,), (8193,), (3, 5, 7)], [F32, BF16, F16]),
    ([(8192,), (8191,), (16385,)], [F16]), ([(1000, 1001), (17,)], [F32]), ([(i % 13 + 1, 9) for i in range(1300)], [F32, BF16]),
])
@pytest.mark.parametrize("max_norm", [0.05, 1e9])
def test_clip_grad_norm(shapes, dtypes, max_norm):
    """The norm: fp32 sums of positive terms.  Scaled tensors: bit for bit the fp32 factor of that norm times
    the element, rounded once."""
    grads = clip_inputs(shapes, dtypes)
    before = [g.clone() for g in grads]
    exact = torch.cat([g.double().reshape(-1) for g in grads]).norm()
    out = [torch.full_like(g, 9.0) for g in grads]
    norm = ops.clip_grad_norm(grads, max_norm, out=out)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(norm.item() / exact.item() - 1) < 1e-5
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    norm2 = ops.clip_grad_norm(grads, max_norm)
    assert torch.equal(norm, norm2)
    limit = torch.full_like(norm, max_norm)  # tensor / tensor: one rounding (scalar / tensor has two)
    coef = torch.where(norm > limit, limit / (norm + 1e-6), torch.ones_like(norm))
    for g, b, o in zip(grads, before, out):
        assert torch.equal(g, o) and torch.equal(o, (b.float() * coef).to(b.dtype))


def test_clip_grad_norm_unaligned_and_non_finite():
    flat = clip_inputs([(5000,)], [BF16])[0]
    views = [flat[1:100], flat[101:4000], flat[4001:]]
    exact = torch.cat([v.double() for v in views]).norm()
    out = torch.zeros_like(flat)
    norm = ops.clip_grad_norm(views, 0.5, out=[out[1:100], out[101:4000], out[4001:]])
    assert abs(norm.item() / exact.item() - 1) < 1e-5
    assert not out[0] and not out[100] and not out[4000]
    assert rel(out[101:4000], views[1].double() * (0.5 / (exact + 1e-6))) < U[BF16] + 1e-5
    g = [torch.ones(10, device=DEV), torch.tensor([float("nan")], device=DEV)]
    assert torch.isnan(ops.clip_grad_norm(g, 1.0)) and torch.equal(g[0], torch.ones(10, device=DEV))
    g = [torch.ones(10, device=DEV), torch.tensor([float("inf")], device=DEV)]
    assert torch.isinf(ops.clip_grad_norm(g, 1.0)) and not g[0].any() and torch.isnan(g[1]).all()


def test_clip_grad_norm_counts_as_an_in_place_write():
    """What is written has a new version, so that a node that saved it refuses to use it, and cached copies of it are
    made anew."""
    g = clip_inputs([(64,), (0,), (5, 7)], [F32, BF16, F16])
    before = [t._version for t in g]
    ops.clip_grad_norm(g, 0.01)
    assert all(t._version > v for t, v in zip(g, before))
    before = [t._version for t in g]
    out = [torch.empty_like(t) for t in g]
    seen = [t._version for t in out]
    ops.clip_grad_norm(g, 0.01, out=out)
    assert all(t._version > v for t, v in zip(out, seen)) and [t._version for t in g] == before
    x = torch.randn(64, device=DEV, requires_grad=True)
    z = x.exp()  # saves its result
    ops.clip_grad_norm([z.detach()], 0.01)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    p = torch.nn.Parameter(torch.randn(8, 8, device=DEV))
    stale = wcache.get(p, BF16).clone()
    ops.clip_grad_norm([torch.ones(8, 8, device=DEV)], 1.0, out=[p.detach()])
    assert torch.equal(wcache.get(p, BF16), p.detach().bfloat16()) and not torch.equal(stale, wcache.get(p, BF16))
    with torch.inference_mode():
        t = torch.ones(8, device=DEV)
        assert ops.clip_grad_norm([t], 1.0) > 2 and t.norm() < 1.001


def test_clip_grad_norm_refusals():
    g = [torch.ones(4, 4, device=DEV)]
    with pytest.raises(ValueError, match="no tensors"):
        ops.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="positive"):
        ops.clip_grad_norm(g, 0.0)
    with pytest.raises(ValueError, match="outputs"):
        ops.clip_grad_norm(g, 1.0, out=[])
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.clip_grad_norm([torch.ones(4, 6, device=DEV).t()], 1.0)
    with pytest.raises(RuntimeError, match="device"):
        ops.clip_grad_norm([g[0], torch.ones(3)], 1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.clip_grad_norm([torch.ones(3, device=DEV, dtype=torch.float64)], 1.0)


def test_second_derivatives_are_refused():
    x, w, _, _, dy = gated_inputs(4, 64, 72, 64, BF16, False, False)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(ops.gated_mlp(x, *w), x, dy, create_graph=True)
    s, _ = ops.norm_gate_residual(x, x.detach(), torch.ones(64, device=DEV))
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(s, x, dy, create_graph=True)


def test_clip_grad_norm_refuses_tensors_that_overlap():
    """All tensors are scaled at the same time: one that is given twice, or an output on another's input, would be
    read and written at once."""
    flat = torch.ones(3000, device=DEV)
    a, b = flat[:1000], flat[1000:2000]
    out = torch.empty_like(flat)
    for grads, outs in [([a, b, a], None), ([a, flat[999:1500]], None), ([a, b], [out[:1000], out[500:1500]]),
                        ([a, b], [b, out[:1000]]), ([a], [flat[1:1001]]), ([a, b], [b, a]), ([flat, b], [flat, out[:1000]])]:
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_grad_norm(grads, 0.5, out=outs)
    assert torch.equal(flat, torch.ones_like(flat))
    norm = ops.clip_grad_norm([a, a, b], 1e9, out=[out[:1000], out[1000:2000], b])  # read twice, written once
    assert abs(norm.item() - 3000 ** 0.5) < 1e-3 and torch.equal(out[:2000], flat[:2000])
    assert not ops.clip_grad_norm([flat[:0], flat[:0]], 1.0)


@pytest.mark.parametrize("frozen", [True, False])
def test_forward_mode_derivatives_are_refused(frozen):
    """Under no_grad or with frozen parameters the output would have no tangent, which counts as zero."""
    from torch.autograd import forward_ad as fw

    x, w, b, _, _ = gated_inputs(4, 64, 72, 64, BF16, True, False)
    y, skip, wp, gt, wn, _, _ = norm_inputs(2, 3, 64, BF16, "sample", True)
    with fw.dual_level(), torch.set_grad_enabled(not frozen):
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_mlp(fw.make_dual(x, x), *w, *b)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_mlp(x, *w, b[0], fw.make_dual(b[1], b[1]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_mlp(x, fw.make_dual(w[0].float(), w[0].float()), w[1].float(), w[2].float())
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.norm_gate_residual(y, fw.make_dual(skip, skip), wp, gt, wn)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.norm_gate_residual(y, skip, wp, fw.make_dual(gt, gt), wn)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.clip_grad_norm([fw.make_dual(wp, wp)], 1.0)


# --------------------------------------------------------------------------- in the model
def test_model_with_gated_networks_and_sandwich_norms_matches_cpu():
    """The tolerances of the plain model's comparison (tests/test_model_gpu.py): bf16 activations through two
    blocks against fp32."""
    from neural_scaling_weather_b200 import config as C
    from neural_scaling_weather_b200.models import get_model
    from neural_scaling_weather_b200.utils.misc import create_dummy_metadata

    torch.manual_seed(0)
    cfg = C.create(dict(
        model=dict(arch="swin", embed_dim=64, patch_size=2, depth=2, window_size=[4, 8], num_heads=4, dropout=0.0,
                   mlp_ratio=8 / 3, coord_pos_embed=True, mlp_type="swiglu", block_norm="sandwich"),
        data=dict(invariants=["a"]), train=dict(temporal_context_window=1, num_rollout_steps=2),
        parallelism=dict(use_transformer_engine=False)))
    md = create_dummy_metadata(32, 64, 5)
    cpu = get_model(cfg, md)
    gpu = get_model(cfg, md).cuda()
    gpu.load_state_dict(cpu.state_dict())
    x, y = torch.randn(2, 1, 6, 32, 64), torch.randn(2, 2, 5, 32, 64)
    out_c = cpu(x)
    ((out_c - y) ** 2).mean().backward()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out_g = gpu(x.cuda())
    ((out_g.float() - y.cuda()) ** 2).mean().backward()
    assert rel(out_g.cpu(), out_c) < 3e-2
    grads = dict(cpu.named_parameters())
    for name, p in gpu.named_parameters():
        assert p.grad is not None and rel(p.grad.cpu(), grads[name].grad) < 8e-2, name


def test_trainer_with_gated_blocks_and_cuda_graphs(tmp_path):
    """Four training steps of the options through the trainer, from captured micro-batches."""
    import os

    from neural_scaling_weather_b200 import config as C
    from neural_scaling_weather_b200.training.trainer import Trainer

    os.environ["MASTER_PORT"] = "29541"
    t = Trainer(C.compose("default", [
        f"hydra.run.dir={tmp_path}", "parallelism.backend=nccl", "model.embed_dim=64", "model.depth=2",
        "model.num_heads=4", "model.window_size=[4,8]", "model.patch_size=2", "data.synthetic.nlat=32",
        "data.synthetic.nlon=64", "data.synthetic.n_samples=40", "data.levels=[500]", "data.batch_size=2",
        "optimizer=adamw", "optimizer.max_iterations=4", "train.log_every=2", "train.amp_dtype=bf16",
        "train.clip_grad_norm=1.0", "logging.log_to_wandb=false", "train.seed=1", "train.cuda_graphs=true",
        "model.mlp_type=swiglu", "model.block_norm=sandwich", "model.mlp_ratio=2.6667"]))
    t.launch()
    assert t.iters == 4 and all(torch.isfinite(p).all() for p in t.model.parameters())
    import torch.distributed as dist

    dist.destroy_process_group()


def test_example_training_step_on_gpu():
    import os
    import sys

    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import train_gated_block as ex

    torch.manual_seed(0)
    model = ex.build(128, 2, (36, 72), 4, DEV, torch.bfloat16)
    losses, norms = ex.train(model, 8, (36, 72), 4)
    assert torch.isfinite(losses).all() and torch.isfinite(norms).all() and losses[-1] < losses[0]
    out = ex.rollout(model, torch.randn(1, 1, 4, 36, 72, device=DEV).bfloat16(), 2)
    assert torch.isfinite(out).all()
