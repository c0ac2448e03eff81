"""Window attention with a learned relative position bias against its definition in 64 bits.

Tolerances are relative 2-norms, counted in u, 2^-9 for bf16 and 2^-11 for fp16 (the 2-norm of the rounding to 16 bits
over the spread of a tensor's significands is below that), on inputs that are exact in the tested type.  Rounded to 16
bits on the way to the output: the normalised q and k, whose errors reach a logit as sums of head_dim products, 2 u
times at most the root of the mean square of the logits (they have it below 2 here), the probabilities and the output:
2 * 2 + 2 = 6 u.  The gradients add those of dS (from the rounded probabilities) and of the result, and the norms' weights
and the bias sum them with changing signs, which leaves a sum's error below the terms' root sum of squares while the sum
itself may cancel to about a third of it: 3 (6 + 2) u = 24 u there, 10 u for q, k and v."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402

DEV = torch.device("cuda")
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = torch.finfo(F32).eps


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


def inputs(B, T, gh, gw, wh, ww, nh, hd, dtype, shift, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, generator=g, device=DEV) * std + mean).to(dtype)

    sh, sw = (wh // 2, ww // 2) if shift else (0, 0)
    geom = ops.WindowGeometry(window=(wh, ww), shift=(sh, sw), mask=shift, mask_shift=sh, h_global=gh * wh)
    qkv = randn(B, T, gh * wh, gw * ww, 3 * nh * hd)
    return qkv, randn(hd, std=0.2, mean=1.0), randn(hd, std=0.2, mean=1.0), randn(nh, geom.num_buckets(T), std=std), geom, \
        randn(B, T, gh * wh, gw * ww, nh * hd)


def exact(qkv, qw, kw, table, geom, nh, hd, dout=None):
    """Pairs of tokens by their grid positions, in fp64; a query without a finite logit is zero."""
    B, T, H, W, _ = qkv.shape
    (wh, ww), (sh, sw) = geom.window, geom.shift
    leaves = [t.detach().double().requires_grad_() for t in (qkv, qw, kw, table)]
    x, qwd, kwd, tab = leaves
    t, y, xx = (v.reshape(-1) for v in torch.meshgrid(torch.arange(T), torch.arange(wh), torch.arange(ww), indexing="ij"))
    bucket = ((t[:, None] - t + T - 1) * (2 * wh - 1) + y[:, None] - y + wh - 1) * (2 * ww - 1) + xx[:, None] - xx + ww - 1
    bucket = bucket.to(DEV)
    norm = lambda v, w: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    out = torch.zeros(B, T, H, W, nh * hd, dtype=torch.float64, device=DEV)
    for wy in range(H // wh):
        rows = (wy * wh + y + sh) % H
        far = ((wy * wh + y) >= H - geom.mask_shift).to(DEV) if geom.mask else torch.zeros_like(y, dtype=torch.bool).to(DEV)
        cols = (torch.arange(W // ww)[:, None] * ww + xx + sw) % W  # (windows across, L)
        v = x[:, t[None].expand_as(cols), rows[None].expand_as(cols), cols].view(B, cols.shape[0], -1, 3, nh, hd)
        q, k, val = v.permute(3, 0, 1, 4, 2, 5)
        s = norm(q, qwd) @ norm(k, kwd).transpose(-1, -2) * hd ** -0.5 + tab[:, bucket]
        s = s - 100.0 * (far[:, None] != far)
        none = (s == -torch.inf).all(-1, keepdim=True)
        p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
        o = (p @ val).transpose(2, 3).reshape(B, cols.shape[0], -1, nh * hd)
        out = out.index_put((torch.arange(B, device=DEV)[:, None, None], t[None, None].to(DEV),
                             rows[None, None].to(DEV), cols[None].to(DEV)), o)
    if dout is None:
        return out.detach()
    return out.detach(), torch.autograd.grad(out, leaves, dout.double())


SHAPES = [  # B, T, window rows, window columns, wh, ww, heads, head_dim
    (1, 1, 1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 9, 18, 2, 64), (2, 1, 3, 2, 9, 18, 3, 64), (1, 1, 3, 3, 4, 4, 4, 64),
    (1, 2, 2, 2, 7, 9, 3, 64), (1, 3, 2, 3, 3, 5, 2, 64), (1, 1, 2, 2, 13, 13, 2, 64), (1, 1, 2, 3, 1, 37, 5, 64),
    (1, 1, 3, 2, 88, 2, 1, 64), (1, 1, 7, 9, 8, 8, 16, 64), (3, 1, 5, 5, 5, 6, 7, 64), (1, 1, 2, 1, 16, 11, 1, 64),
    (1, 1, 2, 2, 16, 12, 2, 64), (1, 2, 2, 2, 7, 9, 3, 32), (1, 1, 3, 2, 9, 18, 3, 16), (2, 1, 2, 2, 9, 18, 2, 128),
    (1, 1, 2, 2, 12, 16, 1, 128), (1, 4, 2, 2, 3, 4, 2, 32), (1, 1, 2, 2, 2, 3, 3, 16), (1, 12, 2, 2, 2, 8, 2, 32)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("B,T,gh,gw,wh,ww,nh,hd", SHAPES)
def test_bias_matches_definition(B, T, gh, gw, wh, ww, nh, hd, shift, dtype):
    qkv, qw, kw, table, geom, dout = inputs(B, T, gh, gw, wh, ww, nh, hd, dtype, shift, seed=wh * ww + nh)
    leaves = [t.clone().requires_grad_() for t in (qkv, qw, kw, table)]
    out = ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3])
    want, grads = exact(qkv, qw, kw, table, geom, nh, hd, dout)
    assert out.dtype == dtype and rel(out, want) < 6 * U[dtype]
    got = torch.autograd.grad(out, leaves, dout)
    c = nh * hd
    for name, a, b, tol in (("dq", got[0][..., :c], grads[0][..., :c], 10), ("dk", got[0][..., c:2 * c], grads[0][..., c:2 * c], 10),
                            ("dv", got[0][..., 2 * c:], grads[0][..., 2 * c:], 10), ("dqw", got[1], grads[1], 24),
                            ("dkw", got[2], grads[2], 24), ("dtable", got[3], grads[3], 24)):
        assert a.dtype == dtype and a.shape == b.shape
        if T * wh * ww == 1 and name != "dv":  # one token: the softmax is one
            assert a.float().abs().max() < 1e-3, name
        else:
            assert rel(a, b) < tol * U[dtype], name
    with torch.no_grad():
        assert torch.equal(ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3]), out)
    again = torch.autograd.grad(ops.window_attention(*leaves[:3], nh, hd, geom, hd ** -0.5, rel_bias=leaves[3]), leaves, dout)
    assert torch.equal(got[3], again[3]) and torch.equal(got[0], again[0])


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (HF, 64)])
def test_bias_against_differences(dtype, hd):
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, 4, 5, 2, hd, dtype, True, seed=3)
    leaf = table.clone().requires_grad_()
    got, = torch.autograd.grad(ops.window_attention(qkv, qw, kw, 2, hd, geom, hd ** -0.5, rel_bias=leaf), [leaf], dout)

    def f(t):
        return (exact(qkv, qw, kw, t, geom, 2, hd) * dout.double()).sum()

    d = torch.randn(table.shape, device=DEV, dtype=torch.float64)
    slope = (f(table.double() + 1e-5 * d) - f(table.double() - 1e-5 * d)) / 2e-5
    # an inner product of the gradient's error (24 u) with a direction that is not correlated with it, four times over
    assert abs(slope - (got.double() * d).sum()) < 4 * 24 * U[dtype] * got.double().norm()


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (HF, 64), (BF, 32)])
def test_bias_of_any_size(dtype, hd):
    """Offsets, wide ranges, the lowest value, infinities."""
    nh, wh, ww = 3, 9, 18
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, wh, ww, nh, hd, dtype, True, seed=4)
    low, inf = torch.finfo(F32).min, float("inf")
    b = geom.relative_buckets().to(DEV)
    cases = {"offset": table.float() + 1000.0, "wide": table.float() * 60, "far below": table.float() - 3e6}
    cases["one displacement left"] = torch.full_like(table, low, dtype=F32).index_fill_(1, b[0, 0], 0.0)
    cases["masked"] = table.float().masked_fill(torch.rand(table.shape, device=DEV) < 0.4, -inf)
    cases["masked"][:, b[0, 0]] = 1.0
    cases["all lowest"] = torch.full_like(table, low, dtype=F32)
    some = table.float().clone()
    some[1] = -inf  # a head without any
    some[2] = low
    some[2, b[0, 1]] = 3.0  # rows that look left have one finite-sized logit, the others the lowest throughout
    cases["heads apart"] = some
    for name, t in cases.items():
        leaves = [v.clone().requires_grad_() for v in (qkv, t)]
        out = ops.window_attention(leaves[0], qw, kw, nh, hd, geom, hd ** -0.5, rel_bias=leaves[1])
        want, grads = exact(qkv, qw, kw, t, geom, nh, hd, dout)
        assert torch.isfinite(out).all(), name
        assert rel(out, want) < 6 * U[dtype], name
        got = torch.autograd.grad(out, leaves, dout)
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all(), name
        # probabilities near one: dS is what remains of a difference of two rounded numbers, its error u of them
        scale = dout.double().norm() * qkv.double().std()
        assert (got[0].double() - grads[0]).norm() < 10 * U[dtype] * max(grads[0].norm(), scale), name
        assert (got[1].double() - grads[3]).norm() < 24 * U[dtype] * max(grads[3].norm(), scale), name


def test_bias_of_zero_is_none_and_types_are_kept():
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 2, 2, 9, 18, 4, 64, BF, True, seed=5)
    plain = ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125)
    # two kernels that share no rounding, each within 6 u of the definition: 6 + 6
    assert rel(ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=torch.zeros_like(table)), plain) < 12 * U[BF]
    want = ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=table)
    turned = table.t().contiguous().t()
    assert torch.equal(ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=turned), want)
    grads = []
    for dt in (F32, torch.float64, HF, BF):
        leaf = turned.to(dt).detach().requires_grad_()
        out = ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=leaf)
        grads.append(torch.autograd.grad(out, [leaf], dout)[0])
        assert grads[-1].dtype == dt and rel(grads[-1], grads[0]) < U[BF]
    # an fp32 parameter whose gradient buffer is added to
    param = torch.nn.Parameter(table.float())
    param.grad = torch.ones_like(param)
    for _ in range(2):
        ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=param).backward(dout)
    assert rel(param.grad - 1, 2 * grads[0]) < 1e-5


def test_bias_refusals():
    qkv, qw, kw, table, geom, _ = inputs(1, 1, 2, 2, 4, 4, 4, 64, BF, False)
    for bad in (table[:3], table[:, 1:], table[0], table.t()):
        with pytest.raises(ValueError):
            ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=bad)
    with pytest.raises(RuntimeError):
        ops.window_attention(qkv, qw, kw, 4, 64, geom, 0.125, rel_bias=table.cpu())
    big = ops.WindowGeometry(window=(16, 16), h_global=16)
    x = torch.zeros(1, 1, 16, 16, 3 * 64, device=DEV, dtype=BF)
    with pytest.raises(ValueError):
        ops.window_attention(x, qw, kw, 1, 64, big, 0.125, rel_bias=torch.zeros(1, big.num_buckets(), device=DEV))


def test_bias_replays():
    qkv, qw, kw, table, geom, dout = inputs(1, 1, 4, 4, 9, 18, 4, 64, BF, True, seed=6)
    leaves = [t.clone().requires_grad_() for t in (qkv, qw, kw, table)]

    def step(*args):
        out = ops.window_attention(*args[:3], 4, 64, geom, 0.125, rel_bias=args[3])
        return [out.detach(), *torch.autograd.grad(out, args, dout)]

    first = step(*leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = [t.detach().clone().requires_grad_() for t in leaves]
    with torch.cuda.stream(side):
        for _ in range(2):
            other = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    new = [torch.randn_like(t) for t in leaves]
    with torch.no_grad():
        for s, n in zip(static, new):
            s.copy_(n)
    graph.replay()
    want = step(*(n.clone().requires_grad_() for n in new))
    assert all(torch.equal(a, b) for a, b in zip(out, want))
