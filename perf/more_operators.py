"""Operators of a Swin block with a learned relative position bias and routed experts: cases, plain forms, exact values.

Three operators that one training step of such a block uses one after the other, and its rollout without gradients:

* ``attn``: shifted-window attention with QK-RMSNorm, the latitude-wrap mask and a learned bias for each head and
  displacement of query and key, ``softmax(scale q k^T + table[bucket(i, j)] + mask) v``; and its backward pass
  (gradients of q / k / v, of the two norm weights and of the table);
* ``route``: the router's choice of ``k`` of ``E`` experts for each token from its logits, their weights (a softmax
  over the chosen ones, or the full softmax's values) and the balance ``E sum_e f_e P_e`` (share of the choices times
  mean probability); and its backward pass;
* ``experts``: ``y_t = sum_j w_tj MLP_e(t,j)(x_t) + residual_t`` with gated networks as experts, products grouped by
  expert over ragged numbers of tokens; and its backward pass (gradients of the input, of the combining weights and of
  the three stacked weight matrices).
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = float(torch.finfo(torch.float32).eps)  # the framework's RMSNorm epsilon

# the largest cases (also the bounds of the drawn ones): a 720 x 1440 grid in patches of 4, windows of 9 x 18
GRID_TOKENS, WIDTH, WINDOW = 180 * 360, 1024, 162
MOST_SCORES = GRID_TOKENS * 16 * WINDOW
MOST_MACS = 2 * GRID_TOKENS * WIDTH * 1368
MOST_WEIGHTS = 64 * WIDTH * 1368


def listed():
    return [
        # one window of a regional cut-out in a rollout: what a single call costs
        {"name": "attn_one_window", "op": "attn", "batch": 1, "steps": 1, "rows": 1, "cols": 1, "wh": 9, "ww": 18,
         "heads": 2, "head_dim": 64, "shift": False, "dtype": "bf16", "train": False},
        # training on two time steps of a small grid, odd windows, narrow heads, half precision
        {"name": "attn_train_odd", "op": "attn", "batch": 2, "steps": 2, "rows": 5, "cols": 7, "wh": 7, "ww": 9,
         "heads": 3, "head_dim": 32, "shift": True, "dtype": "fp16", "train": True},
        # one rollout step of the 720 x 1440 grid, a shifted block
        {"name": "attn_rollout_grid", "op": "attn", "batch": 1, "steps": 1, "rows": 20, "cols": 20, "wh": 9, "ww": 18,
         "heads": 16, "head_dim": 64, "shift": True, "dtype": "bf16", "train": False},
        # training on the 720 x 1440 grid, a shifted block: the largest attention
        {"name": "attn_train_grid", "op": "attn", "batch": 1, "steps": 1, "rows": 20, "cols": 20, "wh": 9, "ww": 18,
         "heads": 16, "head_dim": 64, "shift": True, "dtype": "bf16", "train": True},
        # one token's choice of 2 of 8 experts
        {"name": "route_one_token", "op": "route", "tokens": 1, "experts": 8, "k": 2, "normalize": True,
         "dtype": "bf16", "train": False},
        # a 45 x 90 patch grid (patches of 16), an odd number of experts, fp32 logits, unnormalised weights
        {"name": "route_train_odd", "op": "route", "tokens": 4050, "experts": 61, "k": 3, "normalize": False,
         "dtype": "fp32", "train": True},
        # training on the 720 x 1440 grid with 64 experts
        {"name": "route_train_grid", "op": "route", "tokens": GRID_TOKENS, "experts": 64, "k": 2, "normalize": True,
         "dtype": "bf16", "train": True},
        # one token through two of eight experts: latency, and the weights that it reads
        {"name": "experts_one_token", "op": "experts", "tokens": 1, "dim": 1024, "hidden": 1368, "experts": 8, "k": 2,
         "act": "silu", "dtype": "bf16", "residual": True, "train": False, "skew": 1.0},
        # a few tokens (a column of patches) over sixteen experts, GELU gate, half precision
        {"name": "experts_few_tokens", "op": "experts", "tokens": 37, "dim": 1024, "hidden": 1368, "experts": 16,
         "k": 2, "act": "gelu", "dtype": "fp16", "residual": False, "train": False, "skew": 1.0},
        # a 45 x 90 patch grid; hidden = int(1024 * 4 / 3), whose rows are not 16-byte aligned; uneven experts
        {"name": "experts_unaligned", "op": "experts", "tokens": 4050, "dim": 1024, "hidden": 1365, "experts": 8,
         "k": 2, "act": "silu", "dtype": "bf16", "residual": True, "train": False, "skew": 1.5},
        # training on a small test grid (72 x 144 in patches of 4, width 128): latency of the whole step
        {"name": "experts_train_small", "op": "experts", "tokens": 648, "dim": 128, "hidden": 344, "experts": 4,
         "k": 1, "act": "silu", "dtype": "bf16", "residual": True, "train": True, "skew": 0.5},
        # training on the 720 x 1440 grid, two of eight experts a token: the largest case
        {"name": "experts_train_grid", "op": "experts", "tokens": GRID_TOKENS, "dim": 1024, "hidden": 1368,
         "experts": 8, "k": 2, "act": "silu", "dtype": "bf16", "residual": True, "train": True, "skew": 0.5},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "route", "experts", "experts", "experts"])
    if op == "attn":
        steps = rng.choice([1, 1, 1, 2])
        wh = rng.randint(1, 12)
        ww = rng.randint(1, max(1, min(24, 176 // (steps * wh))))
        heads, hd = rng.randint(1, 16), rng.choice([64, 64, 64, 32, 16, 128])
        scores = heads * (steps * wh * ww) ** 2
        windows = _spread(rng, 1, max(1, min(4096, MOST_SCORES // scores, MOST_SCORES // (8 * heads * hd * wh * ww))))
        batch = rng.choice([1, 1, 2, 3])
        nwh = max(1, int(math.sqrt(windows / batch) * rng.uniform(0.5, 1.0)))
        nww = max(1, windows // (batch * nwh))
        return {"op": "attn", "batch": batch, "steps": steps, "rows": nwh, "cols": nww, "wh": wh, "ww": ww, "heads": heads,
                "head_dim": hd, "shift": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
                "train": rng.random() < 0.5}
    if op == "route":
        experts = _spread(rng, 2, 256)
        k = rng.randint(1, min(8, experts))
        tokens = _spread(rng, 1, max(1, GRID_TOKENS * 64 // max(experts, 16 * k)))
        return {"op": "route", "tokens": tokens, "experts": experts, "k": k, "normalize": rng.random() < 0.6,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "train": rng.random() < 0.5}
    dim = _spread(rng, 96, 2048)
    hidden = max(8, int(dim * rng.choice([2 / 3, 4 / 3, 2.0, 8 / 3])))
    if rng.random() < 0.7:  # most models keep their widths at multiples of 8
        dim, hidden = 8 * (dim // 8), 8 * (hidden // 8)
    experts = _spread(rng, 2, max(2, min(64, MOST_WEIGHTS // (dim * hidden))))
    k = rng.randint(1, min(4, experts))
    tokens = _spread(rng, 1, max(1, min(GRID_TOKENS, MOST_MACS // (k * dim * hidden))))
    return {"op": "experts", "tokens": tokens, "dim": dim, "hidden": hidden, "experts": experts, "k": k,
            "act": rng.choice(["silu", "gelu"]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "residual": rng.random() < 0.5, "train": rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.5])}


# ------------------------------------------------------------------------------------------- inputs
def _grid(case):
    """Windows down and across the token grid, and the window's rows and columns."""
    return case["rows"], case["cols"], case["wh"], case["ww"]


def _buckets(case):
    """Bucket of query token i and key token j of a window: its displacement in time, latitude and longitude."""
    t, wh, ww = case["steps"], case["wh"], case["ww"]
    at = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(wh), torch.arange(ww), indexing="ij")).reshape(3, -1)
    d = at[:, :, None] - at[:, None, :] + torch.tensor([t - 1, wh - 1, ww - 1])[:, None, None]
    return ((d[0] * (2 * wh - 1) + d[1]) * (2 * ww - 1) + d[2]).to(DEVICE)


def _shifts(case):
    return [case["wh"] // 2, case["ww"] // 2] if case["shift"] else [0, 0]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * std + mean).to(dtype)

    s = {"case": case, "leaves": []}
    if case["op"] == "attn":
        (gh, gw, wh, ww), nh, hd = _grid(case), case["heads"], case["head_dim"]
        h, w, t = gh * wh, gw * ww, case["steps"]
        s["qkv"] = randn(case["batch"], t, h, w, 3 * nh * hd)
        s["qw"], s["kw"] = randn(hd, std=0.2, mean=1.0), randn(hd, std=0.2, mean=1.0)
        s["table"] = randn(nh, (2 * t - 1) * (2 * wh - 1) * (2 * ww - 1))  # a trained table: a few units of logit
        if own:
            from neural_scaling_weather_b200 import ops

            sh, sw = _shifts(case)
            s["geom"] = ops.WindowGeometry(window=(wh, ww), shift=(sh, sw), mask=case["shift"], mask_shift=sh,
                                           h_global=h)
        else:
            s["buckets"] = _buckets(case)
        if case["train"]:
            s["dout"] = randn(case["batch"], t, h, w, nh * hd, std=0.1)
            s["leaves"] = [s["qkv"], s["qw"], s["kw"], s["table"]]
    elif case["op"] == "route":
        m, e, k = case["tokens"], case["experts"], case["k"]
        s["logits"] = randn(m, e)
        if case["train"]:
            s["dweights"] = randn(m, k, std=0.1, dtype=torch.float32)
            # the balance's weight in the loss (in half precision the loss is scaled: the gradient of each logit is
            # the balance's divided by the number of tokens)
            s["dbalance"] = torch.full((), 1.0 * m if dt == torch.float16 else 0.01, device=DEVICE)
            s["leaves"] = [s["logits"]]
    else:
        m, d, h, e, k = case["tokens"], case["dim"], case["hidden"], case["experts"], case["k"]
        s["x"] = randn(m, d)  # a normalised stream
        s["w"] = [randn(e, h, d, std=d ** -0.5), randn(e, h, d, std=d ** -0.5), randn(e, d, h, std=h ** -0.5)]
        # a router's choices: some experts are liked more than others
        logits = randn(m, e, dtype=torch.float32) + case["skew"] * randn(e, dtype=torch.float32)
        top = logits.topk(k, dim=1)
        s["experts"] = top.indices
        s["weights"] = torch.softmax(top.values, 1).to(dt)
        s["residual"] = randn(m, d, std=2.0) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(m, d, std=0.1)
            s["leaves"] = [s["x"], s["weights"]] + s["w"]
    for t in s["leaves"]:
        t.requires_grad_()
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _to_windows(t, case, heads):
    """(B, T, H, W, heads * hd) -> (windows, heads, L, hd) of the shifted grid, fp32."""
    b, (gh, gw, wh, ww), steps = case["batch"], _grid(case), case["steps"]
    sh, sw = _shifts(case)
    t = torch.roll(t.detach().float(), (-sh, -sw), (2, 3))
    t = t.reshape(b, steps, gh, wh, gw, ww, heads, case["head_dim"]).permute(0, 2, 4, 6, 1, 3, 5, 7)
    return t.reshape(b * gh * gw, heads, steps * wh * ww, case["head_dim"])


def _from_windows(t, case):
    b, (gh, gw, wh, ww), steps = case["batch"], _grid(case), case["steps"]
    sh, sw = _shifts(case)
    n = t.shape[1] * t.shape[3]
    t = t.reshape(b, gh, gw, t.shape[1], steps, wh, ww, t.shape[3]).permute(0, 4, 1, 5, 2, 6, 3, 7)
    return torch.roll(t.reshape(b, steps, gh * wh, gw * ww, n), (sh, sw), (2, 3))


def _wrap_mask(case):
    """-100 between tokens on the two sides of the latitude wrap: (window rows, L, L)."""
    gh, _, wh, ww = _grid(case)
    far = (torch.arange(gh * wh, device=DEVICE) >= gh * wh - _shifts(case)[0]).reshape(gh, 1, wh, 1)
    far = far.expand(gh, case["steps"], wh, ww).reshape(gh, -1)
    return torch.where(far[:, :, None] != far[:, None, :], -100.0, 0.0)


def _plain_attn(s):
    case = s["case"]
    dt, nh, hd = s["qkv"].dtype, case["heads"], case["head_dim"]
    scale = hd ** -0.5
    q, k, v = (_to_windows(t, case, nh) for t in s["qkv"].chunk(3, -1))
    qw, kw = s["qw"].detach().float(), s["kw"].detach().float()
    rq, rk = (torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS) for t in (q, k))
    qh, kh = q * rq, k * rk
    qn, kn = qh * qw, kh * kw
    p = (qn @ kn.transpose(-1, -2)) * scale + s["table"].detach().float()[:, s["buckets"]]
    if case["shift"]:
        gh, gw = case["rows"], case["cols"]
        p = (p.view(case["batch"], gh, gw, nh, *p.shape[2:]) + _wrap_mask(case)[:, None, None]).view(p.shape)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = {"out": _from_windows(p @ v, case).to(dt)}
    if case["train"]:
        g = _to_windows(s["dout"], case, nh)
        dv = p.transpose(-1, -2) @ g
        ds = g @ v.transpose(-1, -2)
        ds = p * (ds - (p * ds).sum(-1, keepdim=True))
        member = s["buckets"].reshape(-1, 1) == torch.arange(s["table"].shape[1], device=DEVICE)
        table = ds.sum(0).reshape(nh, -1) @ member.float()
        dqn, dkn = (ds @ kn) * scale, (ds.transpose(-1, -2) @ qn) * scale
        grads = []
        for d, hat, r, w in ((dqn, qh, rq, qw), (dkn, kh, rk, kw)):
            dh = d * w
            grads.append(r * (dh - hat * (dh * hat).mean(-1, keepdim=True)))
        out["dqkv"] = torch.cat([_from_windows(t, case) for t in (*grads, dv)], -1).to(dt)
        out["dqw"], out["dkw"] = (dqn * qh).sum((0, 1, 2)).to(dt), (dkn * kh).sum((0, 1, 2)).to(dt)
        out["dtable"] = table.to(dt)
    return out


def _plain_route(s):
    case = s["case"]
    m, e, k = case["tokens"], case["experts"], case["k"]
    z = s["logits"].detach().float()
    p = torch.exp(z - z.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    order = torch.sort(z, dim=1, descending=True, stable=True)  # equal logits: the lower index first
    chosen = order.indices[:, :k]
    w = p.gather(1, chosen)
    if case["normalize"]:
        w = torch.exp(order.values[:, :k] - order.values[:, :1])
        w = w / w.sum(1, keepdim=True)
    share = torch.zeros(e, device=DEVICE).index_add_(0, chosen.reshape(-1), torch.ones(m * k, device=DEVICE))
    share = share * (e / (m * k))
    out = {"weights": w, "experts": chosen, "balance": (share * p.sum(0)).sum() / m}
    if case["train"]:
        g = s["dweights"]
        d = p * (share - (p * share).sum(1, keepdim=True)) * (s["dbalance"] / m)
        if case["normalize"]:
            d = d.scatter_add(1, chosen, w * (g - (w * g).sum(1, keepdim=True)))
        else:
            d = d - p * (w * g).sum(1, keepdim=True)
            d = d.scatter_add(1, chosen, w * g)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _act_and_slope(g, act):
    if act == "silu":
        sig = 1 / (1 + torch.exp(-g))
        return g * sig, sig * (1 + g * (1 - sig))
    cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_experts(s):
    case = s["case"]
    dt, k = s["x"].dtype, case["k"]
    x, w = s["x"].detach().float(), s["weights"].detach().float()
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].float()
    train = case["train"]
    if train:
        dy, dx, dw = s["dy"].float(), torch.zeros_like(x), torch.zeros_like(w)
        dws = [torch.zeros_like(t) for t in s["w"]]
    order = torch.sort(s["experts"].reshape(-1), stable=True).indices
    counts = torch.bincount(s["experts"].reshape(-1), minlength=case["experts"]).tolist()
    at = 0
    for e, n in enumerate(counts):
        rows = order[at:at + n]
        at += n
        if n == 0:
            continue
        tok, slot = rows // k, rows % k
        wg, wu, wd = (t.detach()[e].float() for t in s["w"])
        xe, we = x[tok], w[tok, slot][:, None]
        g, u = xe @ wg.t(), xe @ wu.t()
        a, slope = _act_and_slope(g, case["act"])
        h = a * u
        ye = h @ wd.t()
        y = y.index_add(0, tok, we * ye)
        if train:
            dye = dy[tok]
            dw[tok, slot] = (dye * ye).sum(1)
            dye = we * dye
            dh = dye @ wd
            dg, du = dh * u * slope, dh * a
            dx = dx.index_add(0, tok, dg @ wg + du @ wu)
            for i, t in enumerate((dg.t() @ xe, du.t() @ xe, dye.t() @ h)):
                dws[i][e] = t.to(dt)
    out = {"y": y.to(dt)}
    if train:
        out["dx"], out["dweights"], out["dw"] = dx.to(dt), dw.to(s["weights"].dtype), dws
    return out


# ------------------------------------------------------------------------------------------- the framework's calls
def _own_attn(s):
    from neural_scaling_weather_b200 import ops

    case = s["case"]
    out = ops.window_attention(s["qkv"], s["qw"], s["kw"], case["heads"], case["head_dim"], s["geom"],
                               case["head_dim"] ** -0.5, rel_bias=s["table"])
    res = {"out": out.detach()}
    if case["train"]:
        res["dqkv"], res["dqw"], res["dkw"], res["dtable"] = torch.autograd.grad(out, s["leaves"], s["dout"])
    return res


def _own_route(s):
    from neural_scaling_weather_b200 import ops

    case = s["case"]
    w, chosen, balance = ops.route_tokens(s["logits"], case["k"], normalize=case["normalize"])
    res = {"weights": w.detach(), "experts": chosen, "balance": balance.detach()}
    if case["train"]:
        res["dlogits"], = torch.autograd.grad([w, balance], s["leaves"], [s["dweights"], s["dbalance"]])
    return res


def _own_experts(s):
    from neural_scaling_weather_b200 import ops

    case = s["case"]
    y = ops.expert_mlp(s["x"], s["weights"], s["experts"], *s["w"], residual=s["residual"], activation=case["act"])
    res = {"y": y.detach()}
    if case["train"]:
        res["dx"], res["dweights"], *res["dw"] = torch.autograd.grad(y, s["leaves"], s["dy"])
    return res


def run(state):
    op = state["case"]["op"]
    if op == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    if op == "route":
        return _own_route(state) if own else _plain_route(state)
    return _own_experts(state) if own else _plain_experts(state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attn":
        (gh, gw, wh, ww), t = _grid(case), case["steps"]
        n, length = case["batch"] * t * gh * wh * gw * ww, t * wh * ww
        c = case["heads"] * case["head_dim"]
        table = case["heads"] * (2 * t - 1) * (2 * wh - 1) * (2 * ww - 1)
        if case["train"]:  # q k^T, p v; dv, dp, dq, dk
            return {"bytes": size * (8 * n * c + 2 * table), "flops": 12 * n * length * c}
        return {"bytes": size * (4 * n * c + table), "flops": 4 * n * length * c}
    if case["op"] == "route":
        m, e, k = case["tokens"], case["experts"], case["k"]
        if case["train"]:
            return {"bytes": m * (2 * size * e + 16 * k), "flops": m * (15 * e + 10 * k)}
        return {"bytes": m * (size * e + 12 * k), "flops": m * (5 * e + 4 * k)}
    m, d, h, e, k = case["tokens"], case["dim"], case["hidden"], case["experts"], case["k"]
    weights = 3 * d * h * min(e, m * k)  # experts that no token chooses need not be read
    acts = m * d * (2 + (1 if case["residual"] else 0)) + m * k
    ids = 8 * m * k
    if case["train"]:  # (every expert's gradient is written)
        return {"bytes": size * (weights + 3 * d * h * e + acts + 2 * m * d + m * k) + ids, "flops": 18 * m * k * d * h}
    return {"bytes": size * (weights + acts) + ids, "flops": 6 * m * k * d * h}


# ------------------------------------------------------------------------------------------- exact values
def _exact_attn(s, case):
    b, steps, (gh, gw, wh, ww) = case["batch"], case["steps"], _grid(case)
    nh, hd, length = case["heads"], case["head_dim"], steps * wh * ww
    h, w = gh * wh, gw * ww
    sh, sw = _shifts(case)
    leaves = [s[n].detach().double().requires_grad_(case["train"]) for n in ("qkv", "qw", "kw", "table")]
    qkv, qw, kw, table = leaves
    # the grid token of each window's tokens
    wy, wx, t, iy, ix = (torch.arange(n, device=DEVICE) for n in (gh, gw, steps, wh, ww))
    row = ((wy[:, None] * wh + iy + sh) % h)[:, None, None, :, None]
    col = ((wx[:, None] * ww + ix + sw) % w)[None, :, None, None, :]
    token = (t[None, None, :, None, None] * h + row) * w + col
    token = token.expand(gh, gw, steps, wh, ww).reshape(1, gh * gw, length)
    token = (token + steps * h * w * torch.arange(b, device=DEVICE)[:, None, None]).reshape(-1, length)
    far = (wy[:, None] * wh + iy >= h - sh)[:, None, None, :, None].expand(gh, gw, steps, wh, ww).reshape(-1, length)
    far = far.repeat(b, 1) & case["shift"]
    rows = qkv.reshape(-1, 3, nh, hd)[token].permute(2, 0, 3, 1, 4)
    norm = lambda v, wt: v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS) * wt  # noqa: E731
    scores = torch.einsum("bhid,bhjd->bhij", norm(rows[0], qw), norm(rows[1], kw)) / math.sqrt(hd)
    scores = scores + table[:, _buckets(case)] - 100.0 * (far[:, None, :, None] != far[:, None, None, :])
    o = torch.einsum("bhij,bhjd->bihd", torch.softmax(scores, -1), rows[2])
    out = torch.zeros(b * steps * h * w, nh * hd, dtype=torch.float64, device=DEVICE)
    out = out.index_copy(0, token.reshape(-1), o.reshape(-1, nh * hd)).view(*qkv.shape[:4], nh * hd)
    res = {"out": out.detach()}
    if case["train"]:
        res.update(zip(("dqkv", "dqw", "dkw", "dtable"), torch.autograd.grad(out, leaves, s["dout"].double())))
    return res


def _exact_route(s, case):
    m, e, k = case["tokens"], case["experts"], case["k"]
    z = s["logits"].detach().double().requires_grad_(case["train"])
    left, index, chosen = z.detach().clone(), torch.arange(e, device=DEVICE).expand(m, e), []
    for _ in range(k):  # the largest that is left, the lowest index among equals
        best = torch.where(left == left.amax(1, keepdim=True), index, e).amin(1, keepdim=True)
        chosen.append(best)
        left.scatter_(1, best, -math.inf)
    chosen = torch.cat(chosen, 1)
    p = torch.softmax(z, 1)
    w = torch.softmax(z.gather(1, chosen), 1) if case["normalize"] else p.gather(1, chosen)
    share = torch.bincount(chosen.reshape(-1), minlength=e).double() / (m * k)
    balance = e * (share * p.mean(0)).sum()
    res = {"weights": w.detach(), "experts": chosen, "balance": balance.detach()}
    if case["train"]:
        res["dlogits"], = torch.autograd.grad([w, balance], [z], [s["dweights"].double(), s["dbalance"].double()])
    return res


def _exact_experts(s, case):
    leaves = [t.detach().double().requires_grad_(case["train"]) for t in (s["x"], s["weights"], *s["w"])]
    x, w, wg, wu, wd = leaves
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    for e in range(case["experts"]):
        tok, slot = torch.nonzero(s["experts"] == e, as_tuple=True)
        pre = torch.nn.functional.linear(x[tok], wg[e])
        gate = pre * torch.sigmoid(pre) if case["act"] == "silu" else pre * torch.special.ndtr(pre)
        hidden = gate * torch.nn.functional.linear(x[tok], wu[e])
        y = y.index_add(0, tok, torch.nn.functional.linear(hidden, wd[e]) * w[tok, slot].unsqueeze(1))
    res = {"y": y.detach()}
    if case["train"]:
        res["dx"], res["dweights"], *res["dw"] = torch.autograd.grad(y, leaves, s["dy"].double())
    return res


def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by differentiation of the definition."""
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"attn": _exact_attn, "route": _exact_route, "experts": _exact_experts}[case["op"]](s, case)
