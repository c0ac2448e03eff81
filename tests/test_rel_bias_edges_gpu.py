"""Window attention with a relative position bias where numbers are large, small, masked or nearly cancel, against its
definition in 64 bits.

u is 2^-9 for bf16 and 2^-11 for fp16 (the 2-norm of the rounding to 16 bits over the spread of a tensor's significands is
below that).  As in test_rel_bias_gpu.py 6 u are the output's, 10 u the gradients' of q, k and v, 24 u those of sums
with changing signs.  dS = P (dP - D) may be what remains of a difference: D_i = <dO_i, O_i> has the rounding of O, u times
the root sum of squares of its terms, g_i, and P, whose values were rounded before they were divided by their sum, adds up
to one but for u (sum_j P_ij^2)^1/2.  Both are one number a row, eta_i = u (g_i^2 + D_i^2 sum_j P_ij^2)^1/2, of no sign:
rows add up like their squares.  Three times that is allowed, `eta` below without its u."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402
from tests.test_rel_bias_gpu import BF, DEV, EPS, F32, HF, U, inputs, rel  # noqa: E402

INF = float("inf")


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


def definition(qkv, qw, kw, table, geom, nh, hd, dout=None):
    """-> out, or {out, grads of qkv / qw / kw / table, slack: the same gradients of eta P in dS's place, noise: of each head's
    table (the root sum of squares of eta P)}; fp64, windows gathered token by token."""
    B, T, H, W, _ = qkv.shape
    (wh, ww), (sh, sw) = geom.window, geom.shift
    leaves = [t.detach().double().requires_grad_() for t in (qkv, qw, kw, table)]
    x, qwd, kwd, tab = leaves
    at = [(t, y, c) for t in range(T) for y in range(wh) for c in range(ww)]
    token, far = [], []
    for b in range(B):
        for y0 in range(0, H, wh):
            for x0 in range(0, W, ww):
                token.append([((b * T + t) * H + (y0 + y + sh) % H) * W + (x0 + c + sw) % W for t, y, c in at])
                far.append([bool(geom.mask) and y0 + y >= H - geom.mask_shift for _, y, _ in at])
    token, far = torch.tensor(token, device=DEV), torch.tensor(far, device=DEV)
    bucket = torch.tensor([[((t - t2 + T - 1) * (2 * wh - 1) + y - y2 + wh - 1) * (2 * ww - 1) + c - c2 + ww - 1
                            for t2, y2, c2 in at] for t, y, c in at], device=DEV)
    q, k, v = x.reshape(-1, 3, nh, hd)[token].permute(2, 0, 3, 1, 4)
    norm = lambda a, w: a * torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    s = norm(q, qwd) @ norm(k, kwd).transpose(-1, -2) * hd ** -0.5 + tab[:, bucket]
    s = s - 100.0 * (far[:, None, :, None] != far[:, None, None, :])
    none = (s == -INF).all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
    o = p @ v
    out = torch.zeros(B * T * H * W, nh * hd, dtype=torch.float64, device=DEV)
    out = out.index_copy(0, token.reshape(-1), o.transpose(1, 2).reshape(-1, nh * hd)).view(B, T, H, W, nh * hd)
    if dout is None:
        return out.detach()
    grads = torch.autograd.grad(out, leaves, dout.double(), retain_graph=True)
    with torch.no_grad():
        do = dout.double().reshape(-1, nh, hd)[token].transpose(1, 2)
        d = (do * o).sum(-1, keepdim=True)
        eta = ((do * o).square().sum(-1, keepdim=True) + d.square() * p.square().sum(-1, keepdim=True)).sqrt()
        noise = (p * eta).square().sum((0, 2, 3)).sqrt()
        weight = p * eta
    slack = torch.autograd.grad((s.masked_fill(weight == 0, 0.0) * weight).sum(), leaves, allow_unused=True)
    return {"out": out.detach(), "grads": grads, "slack": slack, "noise": noise}


def call(qkv, qw, kw, table, geom, nh, hd, dout):
    leaves = [t.clone().requires_grad_() for t in (qkv, qw, kw, table)]
    out = ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3])
    return out.detach(), torch.autograd.grad(out, leaves, dout)


# ------------------------------------------------------------------------------------------------ range of the values
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("size", [1e18, 3e30, 3e38, 1e-30])
def test_equal_tokens_give_their_value(hd, size):
    """One window of equal tokens: every weight is 1 / 162, the output is v, whatever its size in bf16."""
    nh, geom = 2, ops.WindowGeometry(window=(9, 18))
    qkv = torch.ones(1, 1, 9, 18, 3 * nh * hd, device=DEV, dtype=BF)
    qkv[..., 2 * nh * hd:] = size
    one = torch.ones(hd, device=DEV)
    for bias in (0.0, -3e6):
        table = torch.full((nh, geom.num_buckets(1)), bias, device=DEV)
        out = ops.window_attention(qkv, one, one, nh, hd, geom, hd ** -0.5, rel_bias=table)
        assert rel(out, qkv[..., 2 * nh * hd:]) < 2 * U[BF]  # (it is itself a bf16 number: at most one rounding)


@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("weight", [1.0, 4.0, 6.0, 12.0])
@pytest.mark.parametrize("power", [-100, -60, -40, 0, 20, 40, 100])
def test_values_of_any_scale(hd, weight, power):
    """v times a power of two scales the output and all gradients but v's.  weight: of one feature's norms alone, so that most
    logits are far below what the weights allow."""
    nh = 2
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, 9, 18, nh, hd, BF, True, seed=hd)
    qkv[..., 2 * nh * hd:] *= 2.0 ** power
    qw[3] = kw[3] = weight
    qkv[..., 3:2 * nh * hd:hd] *= 0.05  # that feature is small in every token
    out, grads = call(qkv, qw, kw, table, geom, nh, hd, dout)
    want = definition(qkv, qw, kw, table, geom, nh, hd, dout)
    c = nh * hd
    assert rel(out, want["out"]) < 6 * U[BF]
    for part in (slice(0, c), slice(c, 2 * c), slice(2 * c, 3 * c)):
        assert rel(grads[0][..., part], want["grads"][0][..., part]) < 10 * U[BF]
    assert rel(grads[3], want["grads"][3]) < 24 * U[BF]


# ------------------------------------------------------------------------------------------------ rows that add up
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("weight,spread", [(1.0, 1.0), (2.0, 0.3), (3.0, 1.0), (3.0, 0.3)])
def test_the_backwards_weights_add_up_to_one(hd, dtype, weight, spread):
    """With dout one for a single query of each window, dv is that query's weights.  Aligned q and k, whose logits are large, at
    norm weights of one to three.  Rounded on the way: the weights (in the forward, whose sum divides them, and here) and
    dv, each u of a root sum of squares that is at most one: 3^1/2 u."""
    nh = 2
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 8, 8, 9, 18, nh, hd, dtype, True, seed=7)
    c = nh * hd
    common = torch.randn(c, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    qkv = torch.cat([spread * qkv[..., :c] + common, spread * qkv[..., c:2 * c] + common, qkv[..., 2 * c:]], -1).to(dtype)
    dout = torch.zeros_like(dout)
    sh, sw = geom.shift
    dout[:, :, (4 + sh) % 9::9, (7 + sw) % 18::18] = 1.0  # token (4, 7) of every window
    _, grads = call(qkv, (qw * weight).to(dtype), (kw * weight).to(dtype), table, geom, nh, hd, dout)
    dv = torch.roll(grads[0][..., 2 * c:].double(), (-sh, -sw), (2, 3))
    total = dv.view(8, 9, 8, 18, nh, hd).sum((1, 3))
    assert (total - 1).square().mean().sqrt() < 3 ** 0.5 * U[dtype]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("weight", [1.0, 2.0, 3.0])
def test_common_offset_of_dp_cancels(hd, dtype, weight):
    """Aligned q and k, and dout and v with a common offset: dP is nearly one number in a row, and dS what remains of it less
    D.  Weights that do not add up to one leave a part of the offset."""
    nh = 2
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, 9, 18, nh, hd, dtype, True, seed=7)
    c = nh * hd
    g = torch.Generator(device=DEV).manual_seed(1)
    common, of_v = (torch.randn(c, generator=g, device=DEV) for _ in range(2))
    qkv = torch.cat([0.3 * qkv[..., :c] + common, 0.3 * qkv[..., c:2 * c] + common, 0.25 * qkv[..., 2 * c:] + of_v], -1).to(dtype)
    qw, kw = (qw * weight).to(dtype), (kw * weight).to(dtype)
    dout = (0.25 * dout + of_v).to(dtype)
    out, grads = call(qkv, qw, kw, table, geom, nh, hd, dout)
    want = definition(qkv, qw, kw, table, geom, nh, hd, dout)
    u = U[dtype]
    for name, part in (("dq", slice(0, c)), ("dk", slice(c, 2 * c))):
        got, g, s = grads[0][..., part].double(), want["grads"][0][..., part], want["slack"][0][..., part]
        assert (got - g).norm() < 10 * u * g.norm() + 3 * u * s.norm(), name
    for h in range(nh):
        assert (grads[3][h].double() - want["grads"][3][h]).norm() < 24 * u * want["grads"][3][h].norm() + 3 * u * want["noise"][h]


@pytest.mark.parametrize("dtype,hd", [(BF, 16), (BF, 32), (BF, 64), (BF, 128), (HF, 32), (HF, 64), (HF, 128)])
def test_each_heads_gradient(dtype, hd):
    """The table's gradient head by head, each against its own size, at offsets, wide ranges, the types' lowest values and
    infinities."""
    nh, wh, ww = 3, 9, 18
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, wh, ww, nh, hd, dtype, True, seed=4)
    g = torch.Generator(device=DEV).manual_seed(9)
    low = torch.finfo(F32).min
    b = geom.relative_buckets().to(DEV)
    cases = {"plain": table.float(), "offset": table.float() + 1000.0, "wide": table.float() * 60,
             "far below": table.float() - 3e6, "all lowest": torch.full_like(table, low, dtype=F32)}
    cases["masked"] = table.float().masked_fill(torch.rand(table.shape, generator=g, device=DEV) < 0.4, -INF)
    cases["masked"][:, b[0, 0]] = 1.0
    apart = table.float().clone()
    apart[1] = -INF
    apart[2] = low
    apart[2, b[0, 1]] = 3.0
    cases["heads apart"] = apart
    half = table.float().clone()  # the lowest value of fp16, with one displacement left of the second head
    half[1:] = torch.finfo(HF).min
    half[1, b[0, 1]] = 3.0
    cases["lowest of fp16"] = half
    u = U[dtype]
    for name, t in cases.items():
        out, grads = call(qkv, qw, kw, t, geom, nh, hd, dout)
        want = definition(qkv, qw, kw, t, geom, nh, hd, dout)
        assert rel(out, want["out"]) < 6 * u, name
        c = nh * hd
        for part in (slice(0, c), slice(c, 2 * c), slice(2 * c, 3 * c)):
            got, e, s = grads[0][..., part].double(), want["grads"][0][..., part], want["slack"][0][..., part]
            assert (got - e).norm() < 10 * u * e.norm() + 3 * u * s.norm(), name
        for h in range(nh):
            got, e = grads[3][h].double(), want["grads"][3][h]
            allowed = 24 * u * e.norm() + 3 * u * want["noise"][h]
            assert (got - e).norm() <= allowed, (name, h)
            assert allowed < 0.75 * e.norm() or not e.any(), (name, h)  # a gradient of zeros does not pass


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("T,wh,ww", [(4, 6, 8), (8, 4, 6), (6, 5, 6), (192, 1, 1)])
def test_windows_of_three_dimensions(T, wh, ww, hd, dtype):
    """The most displacements that 192 tokens can have, 7 x 11 x 15, in any order of the dimensions: the largest tables."""
    nh = 2
    qkv, qw, kw, table, geom, dout = inputs(1, T, 2, 2, wh, ww, nh, hd, dtype, True, seed=T)
    out, grads = call(qkv, qw, kw, table, geom, nh, hd, dout)
    want = definition(qkv, qw, kw, table, geom, nh, hd, dout)
    u, c = U[dtype], nh * hd
    assert rel(out, want["out"]) < 6 * u
    for part in (slice(0, c), slice(c, 2 * c), slice(2 * c, 3 * c)):
        assert rel(grads[0][..., part], want["grads"][0][..., part]) < 10 * u
    assert all(rel(a, b) < 24 * u for a, b in zip(grads[1:], want["grads"][1:]))


# ------------------------------------------------------------------------------------------------ calls
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype,hd", [(BF, 16), (BF, 64), (BF, 128), (HF, 32), (HF, 128)])
def test_results_repeat(dtype, hd, bias):
    nh = 3
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 3, 3, 9, 18, nh, hd, dtype, True, seed=2)
    leaves = [t.clone().requires_grad_() for t in (qkv, qw, kw, table)][:4 if bias else 3]

    def step():
        out = ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3] if bias else None)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    first = step()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def shifted(t, by):
    """The same contiguous tensor, `by` elements into a packed buffer."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
    v = flat[by:by + t.numel()].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (HF, 64), (BF, 128), (HF, 32)])
@pytest.mark.parametrize("master", [False, True])
def test_inputs_of_any_alignment(dtype, hd, master, bias):
    nh = 2
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, 9, 18, nh, hd, dtype, True, seed=3)
    if master:
        qw, kw, table = (torch.nn.Parameter(t.float()) for t in (qw, kw, table))

    def step(x, d):
        leaves = [x.detach().requires_grad_(), *(t.detach().requires_grad_() if not master else t for t in (qw, kw, table))]
        out = ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3] if bias else None)
        return [out.detach(), *torch.autograd.grad(out, leaves[:4 if bias else 3], d)]

    want = step(qkv, dout)
    for by in (1, 3, 4):
        got = step(shifted(qkv, by), shifted(dout, 8 - by))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
