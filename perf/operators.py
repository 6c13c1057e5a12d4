"""Operators of a mixture-of-experts layer around the grouped GEMMs, as they are measured: routing (scores, group-limited
top-k, weights, their gradient), the padded layout tables that follow from the routing, the gradient of the weighted
combine, and the dense matrix product with bias, activation and residual, forward and backward.

`run` computes them in plain torch where `own` is false and through the public entry points of `asymgemm_b200` where it
is true. Layer sizes are those of this repository's own layer workload (hidden 7168, intermediate 2048, 256 experts,
top-8) or generic ones.
"""
import math

import torch

own = False

ALIGN = 128          # rows every expert's segment is padded to
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_FLOPS = 2.0 * 8192 * 4096 * 7168
MOST_BYTES = 4.0 * 8192 * 8 * 7168


# ------------------------------------------------------------------------------------------------------------- cases
def route(name, tokens, experts, top_k, scoring, bias, groups, top_groups, renormalize, scale, dtype, pad, grad):
    case = dict(op="route", tokens=tokens, experts=experts, top_k=top_k, scoring=scoring, bias=bias, groups=groups,
                top_groups=top_groups, renormalize=renormalize, scale=scale, dtype=dtype, pad=pad, grad=grad)
    return dict(case, name=name) if name else case


def layout(name, tokens, experts, top_k, max_rows, pad):
    case = dict(op="layout", tokens=tokens, experts=experts, top_k=top_k, max_rows=max_rows, pad=pad)
    return dict(case, name=name) if name else case


def combine(name, tokens, experts, top_k, hidden, dtype, pad, rows_grad):
    case = dict(op="combine_grad", tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, dtype=dtype, pad=pad, rows_grad=rows_grad)
    return dict(case, name=name) if name else case


def linear(name, m, n, k, activation, bias, residual, dtype, out, grad):
    case = dict(op="linear", m=m, n=n, k=k, activation=activation, bias=bias, residual=residual, dtype=dtype, out=out, grad=grad)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token of a decode step through the router: sigmoid scores, balance bias, 4 of 8 groups; all latency
        route("route_one_token", 1, 256, 8, "sigmoid", True, 8, 4, True, 2.5, "fp32", 0, False),
        # the router of a whole prompt batch of the layer workload
        route("route_prompt", 65536, 256, 8, "sigmoid", True, 8, 4, True, 2.5, "fp32", 0, False),
        # a training step of a softmax router over an odd number of experts, the batch padded at its end; bf16 logits, with gradient
        route("route_train_softmax", 20000, 60, 4, "softmax", False, 1, 1, True, 1.0, "bf16", 37, True),
        # tables of a decode batch
        layout("layout_decode", 64, 256, 8, 0, 0),
        # tables of the layer workload's 65536 tokens
        layout("layout_prompt", 65536, 256, 8, 0, 0),
        # gradient of the combine of a small layer, a few padding tokens
        combine("combine_grad_small", 500, 16, 4, 2048, "bf16", 11, True),
        # gradient of the combine at the layer workload's width
        combine("combine_grad_wide", 8192, 256, 8, 7168, "bf16", 0, True),
        # router logits of a few decode tokens: fp32 out, the weights are all there is to read
        linear("gate_decode", 4, 256, 7168, "none", False, False, "bf16", "fp32", False),
        # router logits of a prompt batch: as many bytes as a narrow product has flops
        linear("gate_prompt", 16384, 256, 7168, "none", True, False, "bf16", "fp32", False),
        # down projection of a shared expert for a decode batch, the routed experts' sum as residual
        linear("down_decode_residual", 48, 7168, 2048, "none", False, True, "bf16", "bf16", False),
        # up projection of a shared expert for a prompt batch
        linear("up_prompt_silu", 8192, 4096, 7168, "silu", True, False, "bf16", "bf16", False),
        # a training step of a projection with everything in its epilogue, ragged rows and columns: output and all gradients
        linear("train_gelu_ragged", 3990, 2050, 2048, "gelu", True, True, "fp16", "fp16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "layout", "combine_grad", "linear", "linear", "linear"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 8 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        grad, renormalize = rng.random() < 0.5, rng.random() < 0.7
        # one renormalised weight is the scale whatever the logits are: its gradient is 0
        top_k = rng.randint(2 if grad and renormalize else 1, min(16, top_groups * experts // groups))
        tokens = _log(rng, 1, 65536 * 256 // max(256, experts))
        return route(None, tokens, experts, top_k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups, top_groups,
                     renormalize, rng.choice([1.0, 1.5, 2.5]), rng.choice(["bf16", "fp16", "fp32"]), rng.randint(0, tokens // 4), grad)
    if op == "layout":
        experts = _log(rng, 4, 512)
        top_k = rng.randint(1, min(8, experts))
        tokens = _log(rng, 1, 65536)
        rows = 0 if rng.random() < 0.6 else 8 + 2 * tokens * top_k // experts
        return layout(None, tokens, experts, top_k, rows, rng.randint(0, tokens // 4))
    if op == "combine_grad":
        experts = _log(rng, 4, 256)
        top_k = rng.randint(1, min(8, experts))
        hidden = 8 * _log(rng, 16, 896)
        tokens = _log(rng, 1, MOST_BYTES / (4.0 * hidden * top_k))
        return combine(None, min(tokens, 16384), experts, top_k, hidden, rng.choice(["bf16", "fp32"]) if tokens < 2048 else "bf16",
                       rng.randint(0, min(tokens, 16384) // 4), rng.random() < 0.6)
    grad = rng.random() < 0.4
    n, k = _log(rng, 64, 8192), 8 * _log(rng, 32, 1024)
    m = _log(rng, 64 if grad else 1, max(128, min(16384, MOST_FLOPS / (2.0 * n * k * (3 if grad else 1)))))
    dtype = rng.choice(["bf16", "fp16"])
    return linear(None, m, n, k, rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.5, rng.random() < 0.4, dtype,
                  dtype if grad else rng.choice([dtype, dtype, "fp32"]), grad)


# ------------------------------------------------------------------------------------------------------------ inputs
def _routing(tokens, experts, top_k, pad, gen):
    """Distinct experts per token, popular ones more often; the last `pad` tokens have none (-1)."""
    popularity = torch.randn(experts, device="cuda", generator=gen)
    noise = torch.empty((tokens, experts), device="cuda").exponential_(generator=gen)
    ids = torch.topk(popularity - noise.log_(), top_k, dim=1).indices
    ids[tokens - pad:] = -1
    return ids


def _padded_rows(case):
    pairs = case["tokens"] * case["top_k"]
    if case.get("max_rows"):
        return case["experts"] * case["max_rows"]
    return -(-pairs // ALIGN) * ALIGN + case["experts"] * ALIGN


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        # trained routers: logits of unit scale with popular experts among them, balance biases that are small beside the scores
        state = dict(case, logits=(normal(t, e) * 1.3 + normal(e) * 0.5).to(FLOATS[case["dtype"]]),
                     balance=normal(e) * 0.05 if case["bias"] else None,
                     used=torch.full((1,), t - case["pad"], dtype=torch.int32, device="cuda") if case["pad"] else None)
        if case["grad"]:
            state["dweights"] = normal(t, case["top_k"])
        return state
    if case["op"] == "layout":
        return dict(case, ids=_routing(case["tokens"], case["experts"], case["top_k"], case["pad"], gen))
    if case["op"] == "combine_grad":
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        dtype = FLOATS[case["dtype"]]
        ids = _routing(t, case["experts"], k, case["pad"], gen)
        return dict(case, dy=normal(t, h).to(torch.bfloat16), rows=normal(_padded_rows(case), h).to(dtype),
                    pos=_plain_layout(ids, case["experts"], 0, _padded_rows(case))[0],
                    weights=torch.softmax(normal(t, k), dim=1))
    m, n, k = case["m"], case["n"], case["k"]
    dtype, out = FLOATS[case["dtype"]], FLOATS[case["out"]]
    state = dict(case, x=normal(m, k).to(dtype), weight=(normal(n, k) / math.sqrt(k)).to(dtype),
                 b=(normal(n) * 0.2).to(dtype) if case["bias"] else None, r=normal(m, n).to(out) if case["residual"] else None)
    if case["grad"]:
        state["dy"] = normal(m, n).to(out)
    return state


# ------------------------------------------------------------------------------------------------------- plain forms
def _plain_route(s):
    """Scores and order in 64 bits: experts near the border of the chosen set differ by less than 32 bits resolve."""
    t, e, k, g = s["tokens"], s["experts"], s["top_k"], s["groups"]
    logits = s["logits"].double()
    if s["scoring"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    choice = score if s["balance"] is None else score + s["balance"].double()
    order = logits if s["balance"] is None else choice        # without a bias the scores rise with the logits
    if g > 1:
        best = torch.sort(choice.view(t, g, e // g), dim=2, descending=True).values[:, :, :2].sum(2)
        chosen = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        allowed = torch.zeros((t, g), dtype=torch.bool, device=logits.device).scatter_(1, chosen, True)
        order = torch.where(allowed.repeat_interleave(e // g, 1), order, -math.inf)
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    weights = score.gather(1, ids)
    if s["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * s["scale"]
    live = (torch.arange(t, device=logits.device) < t - s["pad"]).unsqueeze(1)
    out = [torch.where(live, ids, -1), torch.where(live, weights, 0).float()]
    if s["grad"]:
        dw = torch.where(live, s["dweights"].double(), 0) * s["scale"]
        p = score.gather(1, ids)
        if s["renormalize"]:
            q = p / p.sum(1, keepdim=True)
            dp = dw - (dw * q).sum(1, keepdim=True)           # with respect to p, times the sum of the chosen p
            dl = q * dp * (1 - p if s["scoring"] == "sigmoid" else 1)
            dlogits = torch.zeros_like(logits).scatter_(1, ids, dl)
        elif s["scoring"] == "sigmoid":
            dlogits = torch.zeros_like(logits).scatter_(1, ids, dw * p * (1 - p))
        else:
            dlogits = torch.zeros_like(logits).scatter_(1, ids, dw * p) - score * (dw * p).sum(1, keepdim=True)
        out.append(dlogits.to(s["logits"].dtype))
    return out


def _plain_layout(ids, experts, max_rows, rows):
    """(pair_row, row_token, rows of every expert, start and size of its segment): pairs sorted by expert in their own
    order, each expert's segment padded to ALIGN rows, or every expert given `max_rows` rows."""
    flat = ids.reshape(-1)
    key = torch.where(flat < 0, experts, flat)
    sorted_key, order = torch.sort(key, stable=True)
    count = torch.bincount(key, minlength=experts + 1)[:experts + 1]
    within = torch.arange(flat.numel(), device=ids.device) - (torch.cumsum(count, 0) - count)[sorted_key]
    size = torch.full_like(count, max_rows) if max_rows else (count + ALIGN - 1) // ALIGN * ALIGN
    start = torch.cumsum(size, 0) - size
    fits = sorted_key < experts
    if max_rows:                                       # a pair that finds its expert's rows all taken is dropped
        fits &= within < max_rows
        count = count.clamp(max=max_rows)
    row = torch.where(fits, start[sorted_key] + within, -1)
    pair_row = torch.empty_like(row)
    pair_row[order] = row
    row_token = torch.full((rows + 1,), -1, dtype=torch.int64, device=ids.device)
    row_token[torch.where(row < 0, rows, row)] = torch.where(row < 0, -1, order // ids.shape[1])
    return pair_row, row_token[:rows], count[:experts], start[:experts], size[:experts]


def _plain_combine_grad(s):
    t, k, h = s["tokens"], s["top_k"], s["hidden"]
    r = s["rows"].shape[0]
    pos = s["pos"]
    live = (pos >= 0).view(t, k)
    dy = s["dy"].float()
    picked = s["rows"][pos.clamp(min=0)].view(t, k, h).float()
    dweights = torch.where(live, (picked * dy.unsqueeze(1)).sum(2), 0)
    if not s["rows_grad"]:
        return [dweights]
    drows = torch.zeros((r + 1, h), dtype=s["rows"].dtype, device=dy.device)
    drows[torch.where(pos < 0, r, pos)] = (s["weights"].unsqueeze(2) * dy.unsqueeze(1)).view(t * k, h).to(drows.dtype)
    return [dweights, drows[:r]]


def _plain_linear(s):
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    a = s["activation"]
    if a == "relu":
        y, slope = z.clamp(min=0), (z > 0).float()
    elif a == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    elif a == "silu":
        gate = 1 / (1 + torch.exp(-z))
        y, slope = z * gate, gate * (1 + z * (1 - gate))
    else:
        y, slope = z, None
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(FLOATS[s["out"]])
    if not s["grad"]:
        return [y]
    dz = s["dy"].float() if slope is None else s["dy"].float() * slope
    out = [y, (dz @ w).to(s["x"].dtype), (dz.t() @ x).to(s["weight"].dtype)]
    if s["b"] is not None:
        out.append(dz.sum(0).to(s["b"].dtype))
    return out


# --------------------------------------------------------------------------------------------------------------- run
def run(state):
    s = state
    if own:
        from asymgemm_b200 import dense_ops, moe_ops
    if s["op"] == "route":
        if not own:
            return _plain_route(s)
        ids, weights = moe_ops.route_topk(s["logits"], s["top_k"], scoring=s["scoring"], bias=s["balance"], num_groups=s["groups"],
                                          top_groups=s["top_groups"], renormalize=s["renormalize"], scale=s["scale"], rows_used=s["used"])
        if not s["grad"]:
            return [ids, weights]
        return [ids, weights, moe_ops.route_topk_backward(s["dweights"], ids, s["logits"], scoring=s["scoring"],
                                                          renormalize=s["renormalize"], scale=s["scale"])]
    if s["op"] == "layout":
        if own:
            if s["max_rows"]:
                return list(moe_ops.route_layout_masked(s["ids"], s["experts"], s["max_rows"]))
            return list(moe_ops.route_layout(s["ids"], s["experts"]))
        pair_row, row_token, count, start, size = _plain_layout(s["ids"], s["experts"], s["max_rows"], _padded_rows(s))
        if s["max_rows"]:
            return [pair_row, row_token, count.int()]
        offsets = torch.stack([start, start + size], 1).reshape(-1).int()
        experts = torch.arange(s["experts"] + 1, device=count.device, dtype=torch.int32)
        return [pair_row, row_token, count, offsets, torch.where(experts < s["experts"], experts, -1)]
    if s["op"] == "combine_grad":
        if not own:
            return _plain_combine_grad(s)
        drows, dweights = moe_ops.combine_topk_backward(s["dy"], s["rows"], s["pos"], s["weights"], need_rows=s["rows_grad"])
        return [dweights, drows] if s["rows_grad"] else [dweights]
    if not own:
        return _plain_linear(s)
    if not s["grad"]:
        return [dense_ops.linear(s["x"], s["weight"], bias=s["b"], activation=s["activation"], residual=s["r"], out_dtype=FLOATS[s["out"]])]
    y, pre = dense_ops.linear(s["x"], s["weight"], bias=s["b"], activation=s["activation"], residual=s["r"],
                              out_dtype=FLOATS[s["out"]], return_pre=True)
    grads = dense_ops.linear_backward(s["dy"], s["x"], s["weight"], activation=s["activation"], pre=pre, need_bias=s["b"] is not None)
    return [y] + [g for g in grads if g is not None]


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["dtype"] == "fp32" else 2
        # the backward pass of renormalised weights reads the chosen logits only, and writes whole rows
        b = t * e * size + t * k * 12
        if case["grad"]:
            b += t * e * size + t * k * 4
        return {"bytes": float(b), "flops": 4.0 * t * e}
    if case["op"] == "layout":
        b = case["tokens"] * case["top_k"] * 16 + _padded_rows(case) * 8 + case["experts"] * 20
        return {"bytes": float(b), "flops": 0.0}
    if case["op"] == "combine_grad":
        t, k, h = case["tokens"], case["top_k"], case["hidden"]
        size = 4 if case["dtype"] == "fp32" else 2
        pairs = (t - case["pad"]) * k
        b = t * h * 2 + pairs * h * size + t * k * 16
        if case["rows_grad"]:
            b += _padded_rows(case) * h * size
        return {"bytes": float(b), "flops": 2.0 * pairs * h * (2 if case["rows_grad"] else 1)}
    m, n, k = case["m"], case["n"], case["k"]
    out = 4 if case["out"] == "fp32" else 2
    b = 2 * (m * k + n * k) + m * n * out * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
    f = 2.0 * m * n * k
    if case["grad"]:
        b += m * n * out + 2 * (m * k + n * k) + (2 * n if case["bias"] else 0)
        f *= 3
    return {"bytes": float(b), "flops": f}


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The floating outputs from their definitions in 64 bits (the layout's are whole numbers)."""
    if case["op"] == "layout":
        return None
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "combine_grad":
        dweights = torch.zeros((s["tokens"], s["top_k"]), dtype=torch.float64, device="cuda")
        drows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda") if s["rows_grad"] else None
        pos = s["pos"].view(s["tokens"], s["top_k"])
        for j in range(s["top_k"]):
            token = (pos[:, j] >= 0).nonzero().view(-1)
            row = pos[token, j]
            dy = s["dy"][token].double()
            dweights[token, j] = torch.einsum("th,th->t", dy, s["rows"][row].double())
            if drows is not None:
                drows[row] = dy * s["weights"][token, j].double().unsqueeze(1)
        return [dweights, drows] if drows is not None else [dweights]
    x, w = s["x"].double(), s["weight"].double()
    z = torch.einsum("mk,nk->mn", x, w)
    if s["b"] is not None:
        z += s["b"].double()
    z.requires_grad_(s["grad"])
    act = {"none": lambda v: v * 1.0, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}
    y = act[s["activation"]](z)
    outs = [(y + s["r"].double() if s["r"] is not None else y).detach()]
    if s["grad"]:
        dz, = torch.autograd.grad(y, z, s["dy"].double())
        outs += [torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)]
        if s["b"] is not None:
            outs.append(dz.sum(0))
    return outs


def _exact_route(s):
    """Expert by expert in order of preference, with autograd for the gradient."""
    t, e, g = s["tokens"], s["experts"], s["groups"]
    logits = s["logits"].double().requires_grad_(s["grad"])
    score = torch.softmax(logits, 1) if s["scoring"] == "softmax" else torch.sigmoid(logits)
    with torch.no_grad():
        value = score + s["balance"].double() if s["balance"] is not None else score.clone()
        if g > 1:
            two = value.view(t, g, e // g).topk(min(2, e // g), dim=2).values.sum(2)
            best = two.topk(s["top_groups"], dim=1).indices
            outside = torch.ones((t, g), dtype=torch.bool, device=value.device).scatter_(1, best, False)
            value.view(t, g, e // g)[outside] = -math.inf
        if s["balance"] is None:
            value = torch.where(value == -math.inf, value, logits.detach())
        taken = []
        for _ in range(s["top_k"]):
            top = value.amax(1, keepdim=True)
            first = (value == top).to(torch.uint8).argmax(1, keepdim=True)
            taken.append(first)
            value.scatter_(1, first, -math.inf)
        ids = torch.cat(taken, 1)
    weights = score.gather(1, ids)
    if s["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * s["scale"]
    live = (torch.arange(t, device=logits.device) < t - s["pad"]).unsqueeze(1)
    outs = [None, torch.where(live, weights, 0).detach()]
    if s["grad"]:
        outs.append(torch.autograd.grad(weights, logits, torch.where(live, s["dweights"].double(), 0))[0])
    return outs
