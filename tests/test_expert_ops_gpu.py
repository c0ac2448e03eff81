"""The router and the routed experts against their definitions in 64 bits, on inputs that are exact in the tested type.

Tolerances are relative 2-norms, counted in u, 2^-9 for bf16 and 2^-11 for fp16 (the 2-norm of the rounding to 16 bits
over the spread of a tensor's significands is below that): each value that a kernel rounds to 16 bits on the way to a
result adds at most u to its relative error.  The output passes h, the experts' outputs and itself; dx the weighted dy,
g and u, dg and du, the experts' dx and itself; the weights' gradients of gate and up the same without the fourth, that
of down the weighted dy, h and itself, the combining weights' h, the experts' outputs and themselves.  One more u is
left for everything in fp32 (sums of up to 2^16 terms, exponentials with relative errors below 1e-5)."""

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
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


# --------------------------------------------------------------------------------------------------- router
def route_exact(z, k, normalize, dw=None, db=None):
    """fp64, with the selection by repeated maxima (the lowest index among equals)."""
    m, e = z.shape
    zd = z.detach().double().requires_grad_()
    left, at, chosen = zd.detach().clone(), torch.arange(e, device=DEV).expand(m, e), []
    taken = torch.zeros(m, e, dtype=torch.bool, device=DEV)
    for _ in range(k):
        top = torch.where(taken, -torch.inf, left).amax(1, keepdim=True)
        best = torch.where((left == top) & ~taken, at, e).amin(1, keepdim=True)
        taken.scatter_(1, best, True)
        chosen.append(best)
    chosen = torch.cat(chosen, 1)
    dead = (zd == -torch.inf).all(1, keepdim=True)
    safe = zd.masked_fill(dead, 0.0)
    p = torch.softmax(safe, 1).masked_fill(dead, 0.0)
    w = torch.softmax(safe.gather(1, chosen), 1).masked_fill(dead, 0.0) if normalize else p.gather(1, chosen)
    share = torch.bincount(chosen.reshape(-1), minlength=e).double() / (m * k)
    balance = e * (share * p.mean(0)).sum()
    out = w.detach(), chosen, balance.detach()
    if dw is None:
        return out
    return out, torch.autograd.grad([w, balance], [zd], [dw.double(), db.double()])[0]


# |z - max| is below 16 here, so rounding it to fp32 changes an exponential by 2^-20 at most, and sums and quotients by
# less than as much again
ROUTE_TOL = 2.0 ** -19


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("m,e,k,normalize", [
    (1, 1, 1, True), (1, 8, 2, True), (3, 8, 8, False), (33, 9, 1, False), (257, 16, 16, True), (1000, 31, 5, False),
    (4050, 61, 3, False), (2049, 64, 2, True), (515, 65, 4, True), (700, 129, 9, False), (90, 300, 16, True),
    (19, 512, 7, False), (40000, 8, 2, True), (300, 128, 16, True), (301, 150, 16, False), (67, 256, 9, True)])
def test_route_matches_definition(dtype, m, e, k, normalize):
    g = torch.Generator(device=DEV).manual_seed(m + e)
    z = (torch.randn(m, e, generator=g, device=DEV) * 2).to(dtype).requires_grad_()
    dw, db = torch.randn(m, k, generator=g, device=DEV), torch.full((), 2.0 * m, device=DEV)
    w, chosen, balance = ops.route_tokens(z, k, normalize)
    (we, ce, be), dz = route_exact(z, k, normalize, dw, db)
    assert chosen.dtype == torch.int64 and torch.equal(chosen, ce)
    assert rel(w, we) < ROUTE_TOL and abs(balance.item() - be.item()) < ROUTE_TOL * abs(be.item())
    got, = torch.autograd.grad([w, balance], [z], [dw, db])
    assert got.dtype == dtype and rel(got, dz) < ROUTE_TOL + U.get(dtype, 0.0) + (1e-6 if e == 1 else 0)
    with torch.no_grad():
        again = ops.route_tokens(z, k, normalize)
    assert all(torch.equal(a, b) for a, b in zip(again, (w, chosen, balance)))


def test_route_gradient_against_differences():
    g = torch.Generator(device=DEV).manual_seed(5)
    z = torch.randn(6, 9, generator=g, device=DEV).requires_grad_()
    dw, db = torch.randn(6, 3, generator=g, device=DEV), torch.full((), 3.0, device=DEV)
    for normalize in (True, False):
        w, _, b = ops.route_tokens(z, 3, normalize)
        got, = torch.autograd.grad([w, b], [z], [dw, db])

        def f(v):
            (we, _, be) = route_exact(v, 3, normalize)
            return ((we * dw).sum() + be * db).item()

        step = 1e-6  # central differences in fp64: error step^2 + eps / step
        for i in range(6):
            for j in range(9):
                v = z.detach().double()
                hi, lo = v.clone(), v.clone()
                hi[i, j] += step
                lo[i, j] -= step
                assert abs((f(hi) - f(lo)) / (2 * step) - got[i, j].item()) < 1e-5


def test_route_ties_masks_and_strange_values():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(F32).min
    z = torch.tensor([[1, 1, 1, 1], [0.0, -0.0, 0, -0.0], [-inf, 2, -inf, -inf], [-inf] * 4, [low] * 4,
                      [low, low, 5, low]], device=DEV).requires_grad_()
    w, chosen, balance = ops.route_tokens(z, 2)
    assert chosen.tolist() == [[0, 1], [0, 1], [1, 0], [0, 1], [0, 1], [2, 0]]
    assert w.tolist() == [[0.5, 0.5], [0.5, 0.5], [1, 0], [0, 0], [0.5, 0.5], [1, 0]]
    assert torch.isfinite(balance)
    d, = torch.autograd.grad([w, balance], [z], [torch.ones_like(w) + w.detach(), torch.ones_like(balance)])
    assert torch.isfinite(d).all() and (d[3] == 0).all() and d[2, 0] == 0
    # a NaN is the row's own matter (and the balance's), and is above every number in the choice
    w, chosen, balance = ops.route_tokens(torch.tensor([[0, nan, 9.0], [1, 2, 3]], device=DEV), 1, normalize=False)
    assert chosen.tolist() == [[1], [2]] and w[0].isnan() and abs(w[1].item() - 0.6652410) < 1e-6
    e, m = 61, 700
    same = torch.zeros(m, e, device=DEV, dtype=BF)
    w, chosen, balance = ops.route_tokens(same, 16)
    assert torch.equal(chosen, torch.arange(16, device=DEV).expand(m, 16)) and abs(balance.item() - 1) < 1e-6


def test_route_shapes_strides_and_refusals():
    z = torch.randn(3, 5, 40, device=DEV)
    for v in (z[..., 3:20], z[..., ::2], z.transpose(0, 1)):
        w, chosen, b = ops.route_tokens(v, 3)
        w2, chosen2, b2 = ops.route_tokens(v.contiguous(), 3)
        assert w.shape == chosen.shape == (*v.shape[:-1], 3)
        assert torch.equal(w, w2) and torch.equal(chosen, chosen2) and torch.equal(b, b2)
    w, chosen, b = ops.route_tokens(torch.empty(0, 8, device=DEV).requires_grad_(), 2)
    assert w.shape == chosen.shape == (0, 2) and b.item() == 0
    for bad in (lambda: ops.route_tokens(z, 0), lambda: ops.route_tokens(z, 41), lambda: ops.route_tokens(z, 17),
                lambda: ops.route_tokens(torch.zeros(2, 513, device=DEV), 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.route_tokens(torch.zeros(2, 8, device=DEV, dtype=torch.float64), 2)
    leaf = z.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(ops.route_tokens(leaf, 2)[0].sum(), leaf, create_graph=True)[0].sum(), leaf)


# --------------------------------------------------------------------------------------------------- experts
def expert_inputs(M, k, E, K, H, N, dtype, seed=0, skew=1.0, wdtype=None, drop=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=DEV) * std).to(dtype)

    z = torch.randn(M, E, generator=g, device=DEV) + skew * torch.randn(E, generator=g, device=DEV)
    top = z.topk(k, dim=1)
    chosen = top.indices
    if drop:
        out = torch.rand(M, k, generator=g, device=DEV)
        chosen = torch.where(out < drop / 2, -1, torch.where(out < drop, E, chosen))
    w = [randn(E, H, K, std=K ** -0.5), randn(E, H, K, std=K ** -0.5), randn(E, N, H, std=H ** -0.5)]
    return randn(M, K), torch.softmax(top.values, 1).to(wdtype or dtype), chosen, w, randn(M, N), randn(M, N)


def expert_exact(x, weights, chosen, w, res, act, dy=None):
    leaves = [t.detach().double().requires_grad_() for t in (x, weights, *w)]
    xd, wt, wg, wu, wd = leaves
    y = torch.zeros(x.shape[0], wd.shape[1], dtype=torch.float64, device=DEV) if res is None else res.double()
    for e in range(wg.shape[0]):
        tok, slot = torch.nonzero(chosen == e, as_tuple=True)
        g = xd[tok] @ wg[e].t()
        a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
        y = y.index_add(0, tok, (a * (xd[tok] @ wu[e].t())) @ wd[e].t() * wt[tok, slot][:, None])
    if dy is None:
        return y.detach()
    return y.detach(), torch.autograd.grad(y, leaves, dy.double(), allow_unused=True)


SIZES = [  # M, k, E, K, H, N
    (1, 1, 1, 8, 8, 8), (1, 2, 8, 64, 40, 64), (8, 2, 4, 128, 344, 128), (16, 1, 16, 72, 24, 80), (5, 3, 3, 33, 17, 9),
    (17, 1, 4, 128, 344, 128), (37, 2, 16, 256, 136, 256), (300, 2, 5, 100, 60, 92), (255, 1, 1, 64, 128, 64),
    (257, 3, 7, 65, 31, 129), (4096, 1, 8, 64, 72, 64), (4097, 1, 3, 64, 72, 64), (2049, 2, 61, 96, 200, 104),
    (1000, 16, 40, 64, 64, 64), (700, 2, 512, 64, 8, 64)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,k,E,K,H,N", SIZES)
def test_experts_forward(M, k, E, K, H, N, act, dtype):
    x, wt, chosen, w, res, _ = expert_inputs(M, k, E, K, H, N, dtype, seed=M + E, drop=0.2 if M > 8 else 0.0)
    for r in (None, res):
        y = ops.expert_mlp(x, wt, chosen, *w, residual=r, activation=act)
        assert y.dtype == dtype and rel(y, expert_exact(x, wt, chosen, w, r, act)) < 4 * U[dtype]


@pytest.mark.parametrize("dtype,act", [(BF, "silu"), (HF, "gelu")])
@pytest.mark.parametrize("M,k,E,K,H,N", SIZES)
def test_experts_gradients(M, k, E, K, H, N, act, dtype):
    x, wt, chosen, w, res, dy = expert_inputs(M, k, E, K, H, N, dtype, seed=M + E, drop=0.2 if M > 8 else 0.0)
    leaves = [t.clone().requires_grad_() for t in (x, wt, *w, res)]
    y = ops.expert_mlp(leaves[0], leaves[1], chosen, *leaves[2:5], residual=leaves[5], activation=act)
    ye, exact = expert_exact(x, wt, chosen, w, res, act, dy)
    assert rel(y, ye) < 4 * U[dtype]
    got = torch.autograd.grad(y, leaves, dy)
    for name, a, b, tol in zip(("dx", "dweights", "dgate", "dup", "ddown"), got, exact, (6, 4, 5, 5, 4)):
        assert a.dtype == dtype and a.shape == b.shape and rel(a, b) < tol * U[dtype], name
    assert torch.equal(got[5], dy)
    none = ~(chosen[..., None] == torch.arange(E, device=DEV)).any(1).any(0)
    for a in got[2:5]:  # experts without tokens
        assert (a[none] == 0).all()
    assert (got[1][(chosen < 0) | (chosen >= E)] == 0).all()


def test_experts_gradient_against_differences():
    x, wt, chosen, w, _, dy = expert_inputs(6, 2, 3, 16, 24, 16, HF, seed=9)
    leaves = [t.clone().requires_grad_() for t in (x, wt, *w)]
    got = torch.autograd.grad(ops.expert_mlp(leaves[0], leaves[1], chosen, *leaves[2:]), leaves, dy)
    args = [t.double() for t in (x, wt, *w)]

    def f(a):
        return (expert_exact(a[0], a[1], chosen, a[2:], None, "silu") * dy.double()).sum().item()

    gen = torch.Generator(device=DEV).manual_seed(3)
    for i in range(5):  # along a random direction: the derivative is <gradient, direction>
        d = torch.randn(args[i].shape, generator=gen, device=DEV, dtype=torch.float64)
        hi, lo = ([t + s * 1e-5 * d if j == i else t for j, t in enumerate(args)] for s in (1, -1))
        # error of the inner product: the gradient's (6 u) times the direction's norm
        bound = 6 * U[HF] * got[i].double().norm() * d.norm() / d.numel() ** 0.5 * 4
        assert abs((f(hi) - f(lo)) / 2e-5 - (got[i].double() * d).sum()) < bound


def test_experts_uneven_choices():
    """Every token to one expert, to none, and the same expert twice."""
    x, wt, chosen, w, res, dy = expert_inputs(600, 2, 6, 64, 40, 72, BF, seed=1)
    for c in (torch.full_like(chosen, 5), torch.full_like(chosen, -1), torch.full_like(chosen, 2 ** 40), chosen[:, :1].expand(600, 2)):
        leaves = [t.clone().requires_grad_() for t in (x, wt, *w)]
        y = ops.expert_mlp(leaves[0], leaves[1], c, *leaves[2:], residual=res)
        ye, exact = expert_exact(x, wt, c, w, res, "silu", dy)
        assert rel(y, ye) < 4 * U[BF]
        for a, b in zip(torch.autograd.grad(y, leaves, dy), exact):
            b = torch.zeros_like(a) if b is None else b
            assert rel(a, b) < 6 * U[BF] if b.norm() > 0 else (a == 0).all()
        few = ops.expert_mlp(x[:7], wt[:7], c[:7], *w, residual=res[:7])
        assert rel(few, expert_exact(x[:7], wt[:7], c[:7], w, res[:7], "silu")) < 4 * U[BF]


@pytest.mark.parametrize("M,E,H", [(3, 4, 64), (30, 2, 64), (300, 5, 136), (3000, 3, 1024)])
def test_experts_all_left_out(M, E, H):
    """No assignment inside the experts: the residual, with gradients of zero, whichever kernels run."""
    x, weights, _, w, res, dy = expert_inputs(M, 2, E, 64, H, 72, BF)
    chosen = torch.where(torch.rand(M, 2, device=DEV) < 0.5, -1, E)
    with torch.no_grad():
        assert torch.equal(ops.expert_mlp(x, weights, chosen, *w, residual=res), res)
        assert ops.expert_mlp(x, weights, chosen, *w).abs().max() == 0
    leaves = [t.requires_grad_() for t in (x, weights, *w)]
    y = ops.expert_mlp(x, weights, chosen, *w, residual=res)
    assert torch.equal(y, res)
    assert all(g.abs().max() == 0 for g in torch.autograd.grad(y, leaves, dy))


def test_experts_non_finite_tokens_stay_apart():
    x, wt, chosen, w, _, _ = expert_inputs(300, 2, 4, 64, 72, 64, BF, seed=2)
    x[17] = float("nan")
    x[101, 3] = float("inf")
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[[17, 101]] = False
    y = ops.expert_mlp(x, wt, chosen, *w)
    assert torch.isfinite(y[keep]).all() and y[17].isnan().all()
    # a token that is left out with an infinite weight does not reach the output
    chosen[5] = -1
    wt[5] = float("inf")
    y = ops.expert_mlp(x, wt, chosen, *w)
    assert (y[5] == 0).all()
    # an expert with non-finite weights touches its own tokens alone, next to the others in memory
    keep &= ~(chosen == 1).any(1)
    w[0][1], w[1][1], w[2][1] = float("nan"), float("inf"), float("nan")
    assert torch.isfinite(ops.expert_mlp(x, wt, chosen, *w)[keep]).all()
    few = ops.expert_mlp(x[:8], wt[:8], chosen[:8], *w)
    assert torch.isfinite(few[keep[:8]]).all()


@pytest.mark.parametrize("M", [6, 500])
def test_experts_strides_types_and_shapes(M):
    x, wt, chosen, w, res, dy = expert_inputs(M, 2, 4, 64, 40, 64, BF, seed=4)
    want = ops.expert_mlp(x, wt, chosen, *w, residual=res)
    wide = torch.zeros(M, 131, device=DEV, dtype=BF)
    wide[:, 3:67] = x
    assert torch.equal(ops.expert_mlp(wide[:, 3:67], wt, chosen, *w, residual=res), want)
    assert torch.equal(ops.expert_mlp(x.t().contiguous().t(), wt, chosen.int(), *w, residual=res), want)
    r2 = torch.zeros(M, 77, device=DEV, dtype=BF)
    r2[:, 5:69] = res
    assert torch.equal(ops.expert_mlp(x, wt, chosen.to(torch.uint8), *w, residual=r2[:, 5:69]), want)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in w]
    assert rel(ops.expert_mlp(x, wt, chosen, *turned, residual=res), want) < 2 * U[BF]
    spaced = [torch.zeros(4, 2 * t.shape[1], t.shape[2], device=DEV, dtype=BF)[:, ::2].copy_(t) for t in w]
    assert rel(ops.expert_mlp(x, wt, chosen, *spaced, residual=res), want) < 2 * U[BF]
    y = ops.expert_mlp(x.view(2, -1, 64), wt.view(2, -1, 2), chosen.view(2, -1, 2), *w, residual=res.view(2, -1, 64))
    assert torch.equal(y.view(M, 64), want)
    leaves = [wide[:, 3:67].detach().requires_grad_(), wt.float().requires_grad_(), *(t.detach().requires_grad_() for t in turned)]
    y = ops.expert_mlp(leaves[0], leaves[1], chosen, *leaves[2:])
    exact = expert_exact(x, wt, chosen, w, None, "silu", dy)[1]
    turned_dy = dy.t().contiguous().t()
    for a, b, leaf in zip(torch.autograd.grad(y, leaves, turned_dy), exact, leaves):
        assert a.dtype == leaf.dtype and rel(a, b) < 6 * U[BF]


def test_experts_empty_batch_and_refusals():
    x, wt, chosen, w, res, _ = expert_inputs(4, 2, 4, 64, 40, 64, BF)
    leaves = [t.clone().requires_grad_() for t in (x[:0], wt[:0], *w)]
    y = ops.expert_mlp(leaves[0], leaves[1], chosen[:0], *leaves[2:])
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, leaves, y.detach())
    assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, leaves))
    for bad in (lambda: ops.expert_mlp(x, wt, chosen, w[0], w[1][:3], w[2]), lambda: ops.expert_mlp(x, wt[:3], chosen, *w),
                lambda: ops.expert_mlp(x[:, :60], wt, chosen, *w), lambda: ops.expert_mlp(x, wt, chosen, *w, residual=res[:3]),
                lambda: ops.expert_mlp(x, wt, chosen, *w, activation="relu"),
                lambda: ops.expert_mlp(x, wt.repeat(1, 9), chosen.repeat(1, 9), *w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.expert_mlp(x, wt, chosen.float(), *w)
    with pytest.raises(RuntimeError):
        ops.expert_mlp(x, wt.cpu(), chosen, *w)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(ops.expert_mlp(leaf, wt, chosen, *w).sum(), leaf, create_graph=True)
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError):
            ops.expert_mlp(dual, wt, chosen, *w)


def test_experts_partial_gradients():
    x, wt, chosen, w, _, dy = expert_inputs(400, 2, 4, 64, 40, 64, BF, seed=6)
    full = [t.clone().requires_grad_() for t in (x, wt, *w)]
    want = torch.autograd.grad(ops.expert_mlp(full[0], full[1], chosen, *full[2:]), full, dy)
    for i in range(5):
        args = [t.detach() for t in full]
        args[i] = args[i].clone().requires_grad_()
        got, = torch.autograd.grad(ops.expert_mlp(args[0], args[1], chosen, *args[2:]), [args[i]], dy)
        assert torch.equal(got, want[i])


def test_experts_master_parameters_in_place():
    """fp32 parameters under autocast: gradients are added into their fp32 buffers; repeated backward passes add up."""
    x, wt, chosen, w, _, dy = expert_inputs(500, 2, 4, 64, 40, 64, BF, seed=7, wdtype=F32)
    params = [torch.nn.Parameter(t.float()) for t in w]
    for p in params:
        p.grad = torch.ones_like(p)
    xl, wl = x.float().requires_grad_(), wt.clone().requires_grad_()
    with torch.autocast("cuda", dtype=BF):
        for _ in range(2):
            y = ops.expert_mlp(xl, wl, chosen, *params)
            y.backward(dy)
    exact = expert_exact(x, wt, chosen, w, None, "silu", dy)[1]
    for p, e in zip(params, exact[2:]):
        assert rel(p.grad - 1, 2 * e) < 5 * U[BF]
    assert xl.grad.dtype == F32 and rel(xl.grad, 2 * exact[0]) < 6 * U[BF] and rel(wl.grad, 2 * exact[1]) < 4 * U[BF]
    # gate and up are one parameter: its shares meet in autograd
    tied = torch.nn.Parameter(w[0].float())
    tied.grad = torch.zeros_like(tied)
    with torch.autocast("cuda", dtype=BF):
        ops.expert_mlp(x, wt, chosen, tied, tied, params[2]).backward(dy)
    exact = expert_exact(x, wt, chosen, [w[0], w[0], w[2]], None, "silu", dy)[1]
    assert rel(tied.grad, exact[2] + exact[3]) < 6 * U[BF]
    wcache.clear()


def test_expert_block_repeats_and_replays():
    """Router and experts together, twice, on another stream, and captured with their backward and replayed on new
    inputs."""
    M, k, E, K, H = 3000, 2, 8, 128, 96
    x, _, _, w, res, dy = expert_inputs(M, k, E, K, H, K, BF, seed=8)
    wr = (torch.randn(E, K, device=DEV) * K ** -0.5).to(BF)
    leaves = [t.clone().requires_grad_() for t in (x, wr, *w)]

    def step(inp):
        wt, chosen, balance = ops.route_tokens(inp @ leaves[1].t(), k)
        y = ops.expert_mlp(inp, wt, chosen, *leaves[2:], residual=res)
        return [y.detach(), *torch.autograd.grad([y, balance], [inp, *leaves[1:]], [dy, torch.full_like(balance, 0.01)])]

    first = step(leaves[0])
    assert all(torch.equal(a, b) for a, b in zip(first, step(leaves[0])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(leaves[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    static = x.clone().requires_grad_()
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    new = torch.randn_like(x)
    with torch.no_grad():
        static.copy_(new)
    graph.replay()
    want = step(new.clone().requires_grad_())
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.no_grad():
        static.copy_(x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, first))
