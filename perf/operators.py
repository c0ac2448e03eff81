"""Operators of a transformer block with a gated feed-forward network: cases, plain forms and exact values.

Three operators that one training step of such a block uses together, and that its rollout uses without
gradients:

* ``gated``: the gated feed-forward network ``y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd + residual``,
  and its backward pass (gradients of the input, of the three weights and of the three biases);
* ``norm``: what stands between two branches of the block: the branch's output is normalised, gated per
  sample and channel and added to the scaled skip connection, and the new stream is normalised for the next
  branch, ``s = c * skip + gate * rms(y) * w_post``, ``n = rms(s) * w_next``; and its backward pass;
* ``clip``: the global norm of many gradient tensors, and the tensors scaled to at most ``max_norm``.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = float(torch.finfo(torch.float32).eps)  # the framework's RMSNorm epsilon

# the largest gated case (also the bound of the drawn ones): a 720 x 1440 grid in patches of 4 at width 1024
GRID_TOKENS, WIDTH = 180 * 360, 1024
MOST_MACS = GRID_TOKENS * WIDTH * 2736


def listed():
    return [
        # one token through a trained block: what a single call costs when nothing amortises the weights
        {"name": "gated_one_token", "op": "gated", "tokens": 1, "dim": 1024, "hidden": 2736, "act": "silu",
         "dtype": "bf16", "bias": True, "residual": True, "train": False},
        # a few tokens (a column of patches), exact GELU as the gate, half precision
        {"name": "gated_few_tokens", "op": "gated", "tokens": 37, "dim": 1024, "hidden": 4096, "act": "gelu",
         "dtype": "fp16", "bias": True, "residual": False, "train": False},
        # a 45 x 90 patch grid (patches of 16); hidden = int(1024 * 8 / 3), whose rows are not 16-byte aligned
        {"name": "gated_unaligned", "op": "gated", "tokens": 4050, "dim": 1024, "hidden": 2730, "act": "silu",
         "dtype": "bf16", "bias": True, "residual": True, "train": False},
        # one rollout step of the 720 x 1440 grid: the largest forward pass
        {"name": "gated_rollout", "op": "gated", "tokens": GRID_TOKENS, "dim": 1024, "hidden": 2736, "act": "silu",
         "dtype": "bf16", "bias": True, "residual": True, "train": False},
        # training on a small test grid (72 x 144 in patches of 4, width 128): latency of the whole step
        {"name": "gated_train_small", "op": "gated", "tokens": 648, "dim": 128, "hidden": 344, "act": "silu",
         "dtype": "bf16", "bias": True, "residual": True, "train": True},
        # training the wide model on the coarse grid, half precision, GELU gate, no biases
        {"name": "gated_train_wide", "op": "gated", "tokens": 4050, "dim": 2048, "hidden": 5464, "act": "gelu",
         "dtype": "fp16", "bias": False, "residual": False, "train": True},
        # training on the 720 x 1440 grid: the largest case
        {"name": "gated_train_grid", "op": "gated", "tokens": GRID_TOKENS, "dim": 1024, "hidden": 2736,
         "act": "silu", "dtype": "bf16", "bias": True, "residual": True, "train": True},
        # the norms, gate and skip connection of one token without gradients
        {"name": "norm_one_token", "op": "norm", "samples": 1, "rows": 1, "dim": 1024, "dtype": "bf16",
         "skip_scale": 1.0, "train": False},
        # three samples of a cropped grid at an odd width, half precision, with gradients
        {"name": "norm_train_odd", "op": "norm", "samples": 3, "rows": 677, "dim": 1001, "dtype": "fp16",
         "skip_scale": 0.7071, "train": True},
        # the 720 x 1440 grid at width 1024 as two half grids, with gradients
        {"name": "norm_train_grid", "op": "norm", "samples": 2, "rows": GRID_TOKENS // 2, "dim": 1024,
         "dtype": "bf16", "skip_scale": 1.0, "train": True},
        # the gradients of a one-block test model in bf16: many tiny tensors
        {"name": "clip_small", "op": "clip", "depth": 1, "dim": 128, "hidden": 344, "dtype": "bf16",
         "max_norm": 1.0},
        # the gradients of sixteen blocks at width 1024 in fp32
        {"name": "clip_model", "op": "clip", "depth": 16, "dim": 1024, "hidden": 2736, "dtype": "fp32",
         "max_norm": 1.0},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gated", "gated", "gated", "norm", "norm", "clip"])
    if op == "gated":
        dim = _spread(rng, 96, 2048)
        hidden = int(dim * rng.choice([2.0, 8 / 3, 3.5, 4.0]))
        if rng.random() < 0.7:  # most models keep their widths at multiples of 8
            dim, hidden = 8 * (dim // 8), 8 * max(1, hidden // 8)
        train = rng.random() < 0.5
        tokens = _spread(rng, 1, max(1, min(GRID_TOKENS, MOST_MACS // (dim * hidden))))
        return {"op": "gated", "tokens": tokens, "dim": dim, "hidden": hidden, "act": rng.choice(["silu", "gelu"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "train": train}
    if op == "norm":
        dim = _spread(rng, 96, 2048)
        if rng.random() < 0.7:
            dim = 8 * (dim // 8)
        samples = rng.randint(1, 4)
        rows = _spread(rng, 1, max(1, GRID_TOKENS * WIDTH // (dim * samples)))
        return {"op": "norm", "samples": samples, "rows": rows, "dim": dim,
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "skip_scale": rng.choice([1.0, 0.7071]),
                "train": rng.random() < 0.6}
    dim = 8 * (_spread(rng, 96, 1024) // 8)
    return {"op": "clip", "depth": rng.randint(1, 16), "dim": dim, "hidden": int(dim * rng.choice([8 / 3, 4.0])),
            "dtype": rng.choice(["fp32", "bf16"]), "max_norm": rng.choice([1.0, 32.0, 1e9])}


# ------------------------------------------------------------------------------------------- inputs
def _block_shapes(case):
    """Shapes of the parameters (hence gradients) of the blocks: q, k, v, proj with biases, the gated
    feed-forward network's three products with biases, the norms and the gates."""
    d, h = case["dim"], case["hidden"]
    block = [(d, d)] * 4 + [(d,)] * 4 + [(h, d), (h,), (h, d), (h,), (d, h), (d,)] + [(d,)] * 4 + [(64,), (64,)]
    return block * case["depth"]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "gated":
        m, d, h = case["tokens"], case["dim"], case["hidden"]
        s["x"] = randn(m, d)  # a normalised stream
        s["w"] = [randn(h, d, std=d ** -0.5), randn(h, d, std=d ** -0.5), randn(d, h, std=h ** -0.5)]
        s["b"] = [randn(h, std=0.1), randn(h, std=0.1), randn(d, std=0.1)] if case["bias"] else [None] * 3
        s["residual"] = randn(m, d, std=2.0) if case["residual"] else None
        s["leaves"] = []
        if case["train"]:
            s["dy"] = randn(m, d, std=0.1)
            s["leaves"] = [s["x"]] + s["w"] + [b for b in s["b"] if b is not None]
    elif case["op"] == "norm":
        b, r, d = case["samples"], case["rows"], case["dim"]
        s["y"], s["skip"] = randn(b, r, d, std=0.5), randn(b, r, d, std=2.0)
        # parameters and the conditioning gate are fp32, as the framework keeps them
        s["w_post"] = randn(d, std=0.1, mean=1.0, dtype=torch.float32)
        s["w_next"] = randn(d, std=0.1, mean=1.0, dtype=torch.float32)
        s["gate"] = randn(b, d, std=0.3, mean=0.5, dtype=torch.float32)
        s["leaves"] = []
        if case["train"]:
            s["ds"], s["dn"] = randn(b, r, d, std=0.1), randn(b, r, d, std=0.1)
            s["leaves"] = [s["y"], s["skip"], s["w_post"], s["gate"], s["w_next"]]
    else:
        shapes = _block_shapes(case)
        s["grads"] = [randn(*shape, std=0.01) for shape in shapes]
        # the clipped gradients go to views of one buffer, so that a pass can be repeated on its inputs
        s["flat"] = torch.zeros(sum(8 * -(-g.numel() // 8) for g in s["grads"]), dtype=dt, device=DEVICE)
        s["out"], at = [], 0
        for g in s["grads"]:
            s["out"].append(s["flat"][at:at + g.numel()].view(g.shape))
            at += 8 * -(-g.numel() // 8)
    for t in s.get("leaves", []):
        t.requires_grad_()
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _act_and_slope(g, act):
    if act == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_gated(s):
    case = s["case"]
    dt = s["x"].dtype
    x = s["x"].detach().float()
    wg, wu, wd = (w.detach().float() for w in s["w"])
    bg, bu, bd = (0.0 if b is None else b.detach().float() for b in s["b"])
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    a, slope = _act_and_slope(g, case["act"])
    h = a * u
    y = h @ wd.t() + bd
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dw"] = [(dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)]
        if case["bias"]:
            out["db"] = [dg.sum(0).to(dt), du.sum(0).to(dt), dy.sum(0).to(dt)]
    return out


def _plain_norm(s):
    case = s["case"]
    dt = s["y"].dtype
    y, skip = s["y"].detach().float(), s["skip"].detach().float()
    wp, wn, gate = s["w_post"].detach(), s["w_next"].detach(), s["gate"].detach()[:, None, :]
    ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    yh = y * ry
    st = case["skip_scale"] * skip + gate * (yh * wp)
    rs = torch.rsqrt((st * st).mean(-1, keepdim=True) + EPS)
    sh = st * rs
    out = {"stream": st.to(dt), "normed": (sh * wn).to(dt)}
    if case["train"]:
        dn, ds = s["dn"].float(), s["ds"].float()
        dsh = dn * wn
        ds = ds + rs * (dsh - sh * (dsh * sh).mean(-1, keepdim=True))
        dp = ds * gate
        dyh = dp * wp
        out["dy"] = (ry * (dyh - yh * (dyh * yh).mean(-1, keepdim=True))).to(dt)
        out["dskip"] = (case["skip_scale"] * ds).to(dt)
        out["dw_post"] = (dp * yh).sum((0, 1))
        out["dgate"] = (ds * yh * wp).sum(1)
        out["dw_next"] = (dn * sh).sum((0, 1))
    return out


def _plain_clip(s):
    limit = s["case"]["max_norm"]
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = torch.where(norm > limit, limit / (norm + 1e-6), torch.ones_like(norm))
    [o.copy_(g.float() * coef) for o, g in zip(s["out"], s["grads"])]
    return {"norm": norm, "clipped": s["flat"]}


def _own_gated(s):
    from neural_scaling_weather_b200 import ops

    case = s["case"]
    (wg, wu, wd), (bg, bu, bd) = s["w"], s["b"]
    y = ops.gated_mlp(s["x"], wg, wu, wd, bg, bu, bd, residual=s["residual"], activation=case["act"])
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, s["leaves"], s["dy"])
        out["dx"], out["dw"] = grads[0], list(grads[1:4])
        if case["bias"]:
            out["db"] = list(grads[4:])
    return out


def _own_norm(s):
    from neural_scaling_weather_b200 import ops

    case = s["case"]
    st, n = ops.norm_gate_residual(s["y"], s["skip"], s["w_post"], s["gate"], s["w_next"],
                                   skip_scale=case["skip_scale"])
    out = {"stream": st.detach(), "normed": n.detach()}
    if case["train"]:
        out["dy"], out["dskip"], out["dw_post"], out["dgate"], out["dw_next"] = torch.autograd.grad(
            [st, n], s["leaves"], [s["ds"], s["dn"]])
    return out


def _own_clip(s):
    from neural_scaling_weather_b200 import ops

    return {"norm": ops.clip_grad_norm(s["grads"], s["case"]["max_norm"], out=s["out"]), "clipped": s["flat"]}


def run(state):
    op = state["case"]["op"]
    if op == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_clip(state) if own else _plain_clip(state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "gated":
        m, d, h = case["tokens"], case["dim"], case["hidden"]
        weights = 3 * d * h + (2 * h + d if case["bias"] else 0)
        acts = m * d * (2 + (1 if case["residual"] else 0))
        if case["train"]:
            return {"bytes": 2 * (2 * weights + acts + 2 * m * d), "flops": 18 * m * d * h}
        return {"bytes": 2 * (weights + acts), "flops": 6 * m * d * h}
    if case["op"] == "norm":
        n, d = case["samples"] * case["rows"], case["dim"]
        vecs = 4 * d * (2 + case["samples"])
        if case["train"]:
            return {"bytes": 2 * 8 * n * d + 2 * vecs, "flops": 40 * n * d}
        return {"bytes": 2 * 4 * n * d + vecs, "flops": 12 * n * d}
    n = sum(math.prod(shape) for shape in _block_shapes(case))
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": 2 * size * n, "flops": 3 * n}


# ------------------------------------------------------------------------------------------- exact values
def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by differentiation of the definition."""
    s = prepare(case, seed)
    wide = lambda t: None if t is None else t.detach().double()  # noqa: E731
    with torch.enable_grad():
        if case["op"] == "gated":
            x, w, b = wide(s["x"]), [wide(t) for t in s["w"]], [wide(t) for t in s["b"]]
            leaves = [x] + w + [t for t in b if t is not None]
            for t in leaves:
                t.requires_grad_(case["train"])
            pre = [torch.nn.functional.linear(x, w[i], b[i]) for i in (0, 1)]
            gate = pre[0] * torch.sigmoid(pre[0]) if case["act"] == "silu" else pre[0] * torch.special.ndtr(pre[0])
            y = torch.nn.functional.linear(gate * pre[1], w[2], b[2])
            if s["residual"] is not None:
                y = y + wide(s["residual"])
            out = {"y": y.detach()}
            if case["train"]:
                grads = torch.autograd.grad(y, leaves, wide(s["dy"]))
                out["dx"], out["dw"] = grads[0], list(grads[1:4])
                if case["bias"]:
                    out["db"] = list(grads[4:])
            return out
        if case["op"] == "norm":
            y, skip, wp, gate, wn = (wide(s[k]) for k in ("y", "skip", "w_post", "gate", "w_next"))
            leaves = [y, skip, wp, gate, wn]
            for t in leaves:
                t.requires_grad_(case["train"])
            rms = lambda v: v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)  # noqa: E731
            stream = skip * case["skip_scale"] + rms(y) * wp * gate.unsqueeze(1)
            normed = rms(stream) * wn
            out = {"stream": stream.detach(), "normed": normed.detach()}
            if case["train"]:
                names = ("dy", "dskip", "dw_post", "dgate", "dw_next")
                out.update(zip(names, torch.autograd.grad([stream, normed], leaves, [wide(s["ds"]), wide(s["dn"])])))
            return out
    norm = torch.linalg.vector_norm(torch.cat([g.reshape(-1).double() for g in s["grads"]]))
    coef = case["max_norm"] / (norm + 1e-6) if float(norm) > case["max_norm"] else norm.new_ones(())
    flat = torch.zeros(s["flat"].numel(), dtype=torch.float64, device=DEVICE)
    at = 0
    for g in s["grads"]:
        flat[at:at + g.numel()] = g.reshape(-1).double() * coef
        at += 8 * -(-g.numel() // 8)
    return {"norm": norm, "clipped": flat}
