"""Performance cases: a router and its experts' products, through the public Python entry points.

Between `expert_dispatch` and `expert_combine`: which experts a token goes to and with what weights (`expert_route` and its gradient), the product
of every expert's rows with its own matrix, with bias, activation and residual (`expert_product`, its gradient, and the gradient of its
activation).  A case is one call on device-resident data.  Sizes go from the rows of one decoding step, where a call is launches and the
experts' weights read once, up to the products of a training step.

    listed()            the cases by name
    draw(rng)           one more case of the same ranges
    prepare(case, seed) device inputs and the buffers that a program keeps
    run(state)          one call, and everything it produced; by the framework's operators if `own`, else in plain torch
    work(case)          bytes and operations that any implementation needs
    exact(case, seed)   the same outputs from the definition in 64 bits
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
IDS = {"i32": torch.int32, "i64": torch.int64}

#: the most bytes and operations (by work()) of a drawn case; of operations on 32-bit rows a tenth
MOST_BYTES, MOST_FLOPS = 2.0e9, 400e9


def listed():
    return [
        # the tokens of one decoding step choose their experts
        {"name": "route_decode", "op": "expert_route", "n": 48, "experts": 128, "choices": 8, "type": "bf16", "scores": "softmax", "biased": False, "groups": 1,
         "group_choices": 1, "group_best": 1, "renormalize": True, "scale": 1.0, "closed": 0.0},
        # a training batch: sigmoid scores, a bias that keeps the load even, half of the groups taking part
        {"name": "route_batch", "op": "expert_route", "n": 16384, "experts": 256, "choices": 8, "type": "f32", "scores": "sigmoid", "biased": True, "groups": 8,
         "group_choices": 4, "group_best": 2, "renormalize": True, "scale": 2.5, "closed": 0.0},
        # its backward pass where every score matters: the softmax over all experts, weights as they are
        {"name": "route_grad_batch", "op": "expert_route_grad", "n": 16384, "experts": 64, "choices": 6, "type": "bf16", "scores": "softmax", "biased": False,
         "renormalize": False, "scale": 1.0, "closed": 0.0},
        # a micro-batch with padding tokens, of which the chosen scores alone matter
        {"name": "route_grad_microbatch", "op": "expert_route_grad", "n": 1037, "experts": 60, "choices": 4, "type": "f32", "scores": "sigmoid", "biased": True,
         "renormalize": True, "scale": 1.0, "closed": 0.02},
        # the first product of one decoding step: two rows an expert, all of the weights
        {"name": "product_decode", "op": "expert_product", "rows": 33 * 4, "experts": 64, "in": 2048, "out": 2048, "type": "bf16", "ids": "i32", "lies": "out_in",
         "bias": False, "activation": "gated_silu", "residual": False, "keep": False, "dropped": 0.0},
        # the first product of a training batch, with what its backward pass needs
        {"name": "product_batch", "op": "expert_product", "rows": 16384 * 8, "experts": 128, "in": 2048, "out": 1536, "type": "bf16", "ids": "i32",
         "lies": "in_out", "bias": False, "activation": "gated_silu", "residual": False, "keep": True, "dropped": 0.03},
        # a prefill through one of a few large experts, added to what the rows have already
        {"name": "product_prefill", "op": "expert_product", "rows": 8191 * 2, "experts": 8, "in": 4096, "out": 2048, "type": "f16", "ids": "i64", "lies": "out_in",
         "bias": True, "activation": None, "residual": True, "keep": False, "dropped": 0.0},
        # a small model in 32 bits, of odd width
        {"name": "product_odd", "op": "expert_product", "rows": 2 * 1024, "experts": 6, "in": 1000, "out": 1501, "type": "f32", "ids": "i32", "lies": "in_out",
         "bias": True, "activation": "gelu", "residual": False, "keep": True, "dropped": 0.0},
        # between a training batch's two products on the way back
        {"name": "activation_grad_batch", "op": "expert_activation_grad", "rows": 16384 * 6, "out": 1024, "type": "bf16", "activation": "gated_silu"},
        # the same of a micro-batch of few and odd rows
        {"name": "activation_grad_microbatch", "op": "expert_activation_grad", "rows": 1037, "out": 1001, "type": "f16", "activation": "gelu"},
        # the backward pass of a training batch's second product
        {"name": "product_grad_batch", "op": "expert_product_grad", "rows": 16384 * 6, "experts": 64, "in": 1024, "out": 2048, "type": "bf16", "grad": "bf16",
         "ids": "i32", "lies": "out_in", "bias": False, "accumulate": False, "dropped": 0.02},
        # a micro-batch added to 32-bit main gradients
        {"name": "product_grad_microbatch", "op": "expert_product_grad", "rows": 4099 * 2, "experts": 16, "in": 1000, "out": 1280, "type": "bf16", "grad": "f32",
         "ids": "i32", "lies": "in_out", "bias": True, "accumulate": True, "dropped": 0.0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, high):
    # most widths are a power of two or 5/4 or 7/4 of one, some are odd
    return _log_uniform(rng, 33, high) | 1 if rng.random() < 0.2 else rng.choice([w for w in (f << k for f in (4, 5, 7) for k in range(4, 10)) if w <= high])


def draw(rng):
    while True:
        op = rng.choice(["expert_route", "expert_route_grad", "expert_product", "expert_product", "expert_product_grad", "expert_product_grad", "expert_activation_grad"])
        case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
        if op in ("expert_route", "expert_route_grad"):
            groups = rng.choice([1, 1, 1, 2, 4, 8])
            experts = groups * _log_uniform(rng, 4, 512 // groups)
            kept = rng.randint(1, groups)
            case.update(n=_log_uniform(rng, 1, 65536), experts=experts, choices=rng.randint(1, min(8, kept * experts // groups)), scores=rng.choice(["softmax", "sigmoid"]),
                        biased=rng.random() < 0.5, renormalize=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), closed=rng.choice([0.0, 0.0, 0.02, 0.5]))
            if op == "expert_route":
                case.update(groups=groups, group_choices=kept, group_best=rng.choice([1, 2]))
        elif op == "expert_activation_grad":
            case.update(rows=_log_uniform(rng, 1, 131072), out=_width(rng, 3584), activation=rng.choice(["silu", "gelu", "gated_silu", "gated_gelu"]))
        else:
            case.update(rows=_log_uniform(rng, 1, 131072), experts=_log_uniform(rng, 1, 256), ids=rng.choice(["i32", "i64"]), lies=rng.choice(["in_out", "out_in"]),
                        bias=rng.random() < 0.4, dropped=rng.choice([0.0, 0.0, 0.05, 0.5]))
            case["in"], case["out"] = _width(rng, 3584), _width(rng, 3584)
            if op == "expert_product":
                case.update(activation=rng.choice([None, None, "silu", "gelu", "gated_silu", "gated_gelu"]), residual=rng.random() < 0.25)
                case["keep"] = case["activation"] is not None and rng.random() < 0.5
                if case["activation"] in ("gated_silu", "gated_gelu"):
                    case["out"] *= 2
            else:
                case.update(grad=rng.choice([case["type"], "f32"]), accumulate=rng.random() < 0.4)
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS / (10 if case["type"] == "f32" else 1):
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _normal(g, shape, dtype, scale=1.0):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g)


def _offsets(case, seed):
    """Where each expert's rows begin and how many rows there are: some experts are liked better, dropped assignments leave rows behind the last."""
    rng = np.random.default_rng(seed)
    liked = np.exp(0.5 * rng.standard_normal(case["experts"]))
    kept = int(round(case["rows"] * (1.0 - case["dropped"])))
    return np.concatenate([[0], np.cumsum(rng.multinomial(kept, liked / liked.sum()))])


def _weight(g, case, t, scale):
    """[experts, in, out], the outputs of an input or the inputs of an output next to one another"""
    e, i, o = case["experts"], case["in"], case["out"]
    return _normal(g, (e, i, o), t, scale) if case["lies"] == "in_out" else _normal(g, (e, o, i), t, scale).transpose(1, 2)


def _gated(activation):
    return activation in ("gated_silu", "gated_gelu")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, t = case["op"], DTYPES[case["type"]]
    s = {k: case[k] for k in ("op", "choices", "scores", "groups", "group_choices", "group_best", "renormalize", "scale", "activation", "keep", "accumulate") if k in case}
    if op in ("expert_route", "expert_route_grad"):
        n, e = case["n"], case["experts"]
        logits = _normal(g, (n, e), torch.float32) + 0.7 * _normal(g, (e,), torch.float32)
        if case["closed"]:      # experts that may not be chosen, and padding tokens, which choose none
            gone = torch.rand(n, e, generator=g, device="cuda") < case["closed"]
            gone |= torch.rand(n, 1, generator=g, device="cuda") < 0.02
            logits = torch.where(gone, -math.inf, logits)
        s["logits"] = logits.to(t)
        s["bias"] = _normal(g, (e,), torch.float32, 0.05) if case["biased"] else None
        if op == "expert_route_grad":
            s["experts"] = _plain_route(s["logits"], case["choices"], case["scores"], s["bias"], 1, 1, 1, True, 1.0)[0]
            s["dweights"] = _normal(g, (n, case["choices"]), torch.float32, 0.01)
    elif op == "expert_activation_grad":
        s["before"] = _normal(g, (case["rows"], case["out"] * (2 if _gated(case["activation"]) else 1)), t)
        s["dout"] = _normal(g, (case["rows"], case["out"]), t, 0.01)
    else:
        at = _offsets(case, seed)
        s["ends"] = at.tolist()
        s["offsets"] = torch.from_numpy(at).cuda().to(IDS[case["ids"]])
        s["x"] = _normal(g, (case["rows"], case["in"]), t)
        s["weight"] = _weight(g, case, t, 1.0 / math.sqrt(case["in"]))
        if op == "expert_product":
            s["bias"] = _normal(g, (case["experts"], case["out"]), t, 0.1) if case["bias"] else None
            width = case["out"] // (2 if _gated(case["activation"]) else 1)
            s["residual"] = _normal(g, (case["rows"], width), t) if case["residual"] else None
        else:
            s["dout"] = _normal(g, (case["rows"], case["out"]), t, 0.01)
            s["dtype"], s["bias"] = DTYPES[case["grad"]], case["bias"]
            s["into"] = _weight(g, case, s["dtype"], 0.1) if case["accumulate"] else None
    return s


# --------------------------------------------------------------------------------------------------------- plain forms
def _scores(logits, scores):
    """In 64 bits, of the experts that are open (their logit is a number above -inf), and which are."""
    x = logits.double()
    is_open = x > -math.inf
    if scores == "sigmoid":
        return torch.where(is_open, 1.0 / (1.0 + torch.exp(-x)), 0.0), is_open
    e = torch.where(is_open, torch.exp(x - torch.where(is_open, x, -math.inf).amax(1, keepdim=True)), 0.0)
    return e / e.sum(1, keepdim=True).clamp(min=1.0), is_open


def _plain_route(logits, choices, scores, bias, groups, group_choices, group_best, renormalize, scale):
    """Values next to a border decide which expert it is: scores are compared in 64 bits."""
    n, e = logits.shape
    score, is_open = _scores(logits, scores)
    value = score if bias is None else score + bias.double()
    order = torch.where(is_open, logits.double() if bias is None else value, -math.inf)
    if groups > 1:
        best = torch.sort(torch.where(is_open, value if group_best == 2 else order, -math.inf).view(n, groups, e // groups), dim=2, descending=True).values[:, :, :group_best]
        some = best[:, :, 0] > -math.inf
        rank = torch.where(some, torch.where(best > -math.inf, best, 0.0).sum(2), -math.inf)
        kept = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :group_choices]
        stays = torch.zeros(n, groups, dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        order = torch.where(stays[:, :, None].expand(n, groups, e // groups).reshape(n, e), order, -math.inf)
    top, ids = torch.sort(order, dim=1, descending=True, stable=True)
    top, ids = top[:, :choices], ids[:, :choices]
    chosen = top > -math.inf
    w = torch.where(chosen, torch.gather(score, 1, ids), 0.0)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(chosen, ids, -1).int(), (scale * w).float()


def _plain_route_grad(dweights, experts, logits, scores, renormalize, scale):
    score, is_open = _scores(logits, scores)
    score = score.float()
    chosen = experts >= 0
    at = experts.clamp(min=0).long()
    g = torch.where(chosen, scale * dweights, 0.0)
    w = torch.where(chosen, torch.gather(score, 1, at), 0.0)
    spread = lambda v: torch.zeros_like(score).scatter_add_(1, at, torch.where(chosen, v, 0.0))  # noqa: E731
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
        d = w * (g - (g * w).sum(1, keepdim=True))
        d = spread(d) if scores == "softmax" else spread(d) * (1.0 - score)
    elif scores == "softmax":
        d = score * (spread(g) - (g * w).sum(1, keepdim=True))
    else:
        d = spread(g) * score * (1.0 - score)
    return torch.where(is_open, d, 0.0).to(logits.dtype)


def _activated(x, activation):
    if activation is None:
        return x
    if _gated(activation):
        half = x.shape[-1] // 2
        return _activated(x[..., :half], activation[6:]) * x[..., half:]
    if activation == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * torch.erfc(-x * math.sqrt(0.5))


def _slope(x, activation):
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return s * (1.0 + x * (1.0 - s))
    return 0.5 * torch.erfc(-x * math.sqrt(0.5)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)


def _plain_activation_grad(dout, before, activation):
    d, x = dout.float(), before.float()
    if not _gated(activation):
        return (d * _slope(x, activation)).to(before.dtype)
    half = x.shape[1] // 2
    a, b = x[:, :half], x[:, half:]
    return torch.cat([d * b * _slope(a, activation[6:]), d * _activated(a, activation[6:])], dim=1).to(before.dtype)


def _plain_product(x, ends, weight, bias, activation, residual, keep):
    width = weight.shape[2]
    out = torch.zeros(x.shape[0], width // (2 if _gated(activation) else 1), dtype=x.dtype, device=x.device)
    before = torch.zeros(x.shape[0], width, dtype=x.dtype, device=x.device) if keep else None
    for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        if a == b:
            continue
        h = x[a:b].float() @ weight[e].float()
        if bias is not None:
            h = h + bias[e].float()
        if keep:
            before[a:b] = h
        h = _activated(h, activation)
        out[a:b] = h if residual is None else h + residual[a:b].float()
    return (out, before) if keep else out


def _plain_product_grad(dout, x, ends, weight, bias, dtype, into):
    dx = torch.zeros_like(x)
    dweight = torch.zeros_like(weight, dtype=dtype) if into is None else into      # of weight's layout
    dbias = torch.zeros(weight.shape[0], weight.shape[2], device=x.device) if bias else None
    for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
        if a == b:
            continue
        d = dout[a:b].float()
        dx[a:b] = d @ weight[e].float().t()
        dw = x[a:b].float().t() @ d
        dweight[e] = dw if into is None else dweight[e].float() + dw
        if bias:
            dbias[e] = d.sum(0)
    return (dx, dweight, dbias) if bias else (dx, dweight)


def run(s):
    op = s["op"]
    if own:
        import thrust_b200 as tb
        if op == "expert_route":
            return tb.expert_route(s["logits"], s["choices"], s["scores"], s["bias"], s["groups"], s["group_choices"], s["group_best"], s["renormalize"], s["scale"])
        if op == "expert_route_grad":
            return tb.expert_route_grad(s["dweights"], s["experts"], s["logits"], s["scores"], s["renormalize"], s["scale"])
        if op == "expert_product":
            return tb.expert_product(s["x"], s["offsets"], s["weight"], s["bias"], s["activation"], s["residual"], s["keep"])
        if op == "expert_activation_grad":
            return tb.expert_activation_grad(s["dout"], s["before"], s["activation"])
        dx, dweight, dbias = tb.expert_product_grad(s["dout"], s["x"], s["offsets"], s["weight"], bias=s["bias"], dtype=s["dtype"], out=s["into"],
                                                    accumulate=s["into"] is not None)
        return (dx, dweight, dbias) if s["bias"] else (dx, dweight)
    if op == "expert_route":
        return _plain_route(s["logits"], s["choices"], s["scores"], s["bias"], s["groups"], s["group_choices"], s["group_best"], s["renormalize"], s["scale"])
    if op == "expert_route_grad":
        return _plain_route_grad(s["dweights"], s["experts"], s["logits"], s["scores"], s["renormalize"], s["scale"])
    if op == "expert_product":
        return _plain_product(s["x"], s["ends"], s["weight"], s["bias"], s["activation"], s["residual"], s["keep"])
    if op == "expert_activation_grad":
        return _plain_activation_grad(s["dout"], s["before"], s["activation"])
    return _plain_product_grad(s["dout"], s["x"], s["ends"], s["weight"], s["bias"], s["dtype"], s["into"])


# ------------------------------------------------------------------------------------------------------ what it costs
def work(case):
    op, b = case["op"], SIZE[case["type"]]
    if op in ("expert_route", "expert_route_grad"):
        n, e, k = case["n"], case["experts"], case["choices"]
        if op == "expert_route":
            return {"bytes": n * e * b + (4 * e if case["biased"] else 0) + 8 * n * k, "flops": 4 * n * e}
        # without the whole softmax the logits of the chosen experts are all that is read
        read = e if case["scores"] == "softmax" and not case["renormalize"] else k
        return {"bytes": n * (read + e) * b + 8 * n * k, "flops": 4 * n * read}
    m, o = case["rows"], case["out"]
    if op == "expert_activation_grad":
        width = o * (2 if _gated(case["activation"]) else 1)
        return {"bytes": m * (o + 2 * width) * b, "flops": 8 * m * width}
    i, e = case["in"], case["experts"]
    kept = m * (1.0 - case["dropped"])
    used = e * (1.0 - (1.0 - 1.0 / e) ** kept) if e > 1 else 1.0      # experts that have rows, on average
    ids = (e + 1) * (4 if case["ids"] == "i32" else 8)
    if op == "expert_product":
        width = o // (2 if _gated(case["activation"]) else 1)
        out = m * width + (m * o if case["keep"] else 0) + (kept * width if case["residual"] else 0)
        return {"bytes": ids + (kept * i + used * i * o + out + (used * o if case["bias"] else 0)) * b, "flops": 2 * kept * i * o}
    grad = SIZE[case["grad"]]
    return {"bytes": ids + (kept * (i + o) + used * i * o + m * i) * b + (2 * used if case["accumulate"] else e) * i * o * grad + (4 * e * o if case["bias"] else 0),
            "flops": 4 * kept * i * o}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_scores(x, scores):
    x = x.double().cpu().numpy()
    with np.errstate(all="ignore"):
        if scores == "sigmoid":
            return x, np.exp(-np.logaddexp(0.0, -x))
        top = np.where(np.isneginf(x.max(1)), 0.0, x.max(1))
        p = np.exp(x - top[:, None])
        return x, p / np.maximum(p.sum(1), 1e-300)[:, None]


def _exact_route(s):
    """Row after row what the definition says of weights; which experts they belong to are whole numbers, which the two sides compare."""
    ids = _plain_route(s["logits"], s["choices"], s["scores"], s["bias"], s["groups"], s["group_choices"], s["group_best"], False, 1.0)[0].cpu().numpy()
    _, score = _exact_scores(s["logits"], s["scores"])
    w = np.where(ids >= 0, np.take_along_axis(score, np.maximum(ids, 0).astype(np.int64), axis=1), 0.0)
    if s["renormalize"]:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return [None, torch.from_numpy(s["scale"] * w).cuda()]


def _exact_route_grad(s):
    """The Jacobian of each row's weights, chosen expert by chosen expert."""
    _, score = _exact_scores(s["logits"], s["scores"])
    ids, g = s["experts"].cpu().numpy(), s["scale"] * s["dweights"].double().cpu().numpy()
    n, k = ids.shape
    rows = np.arange(n)
    slope = score * (1.0 - score)
    total = np.zeros(n)
    mean = np.zeros(n)      # of the choices' gradients, weighted by their scores
    for j in range(k):
        p = np.where(ids[:, j] >= 0, score[rows, ids[:, j]], 0.0)
        total += p
        mean += p * g[:, j]
    d = np.zeros_like(score)
    for j in range(k):
        r = rows[ids[:, j] >= 0]
        c = ids[r, j]
        if s["renormalize"]:
            inner = (g[r, j] - mean[r] / total[r]) / total[r]
            d[r, c] += inner * (slope[r, c] if s["scores"] == "sigmoid" else score[r, c])
        elif s["scores"] == "sigmoid":
            d[r, c] += g[r, j] * slope[r, c]
        else:
            d[r, c] += g[r, j] * score[r, c]
    if s["scores"] == "softmax" and not s["renormalize"]:
        d -= score * mean[:, None]
    return torch.from_numpy(d).cuda()


def _exact_act(x, name):
    return x * torch.sigmoid(x) if name == "silu" else x * torch.special.ndtr(x)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "expert_route":
        return _exact_route(s)
    if op == "expert_route_grad":
        return _exact_route_grad(s)
    if op == "expert_activation_grad":
        name, x = case["activation"], s["before"].double()
        gate, up = x.chunk(2, dim=1) if _gated(name) else (x, None)
        kind = name[-4:]
        phi = torch.sigmoid(gate) if kind == "silu" else torch.special.ndtr(gate)
        slope = phi + gate * (phi * (1.0 - phi) if kind == "silu" else torch.exp(-gate ** 2 / 2.0) / math.sqrt(2.0 * math.pi))
        d = s["dout"].double()
        return d * slope if up is None else torch.cat([d * up * slope, d * gate * phi], dim=1)
    spans = [(e, slice(a, b)) for e, (a, b) in enumerate(zip(s["ends"][:-1], s["ends"][1:])) if b > a]
    x, w = s["x"], s["weight"]
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    if op == "expert_product":
        before = new(case["rows"], case["out"])
        for e, span in spans:
            torch.matmul(x[span].double(), w[e].double(), out=before[span])
            if s["bias"] is not None:
                before[span] += s["bias"][e].double()
        name = case["activation"]
        if name is None:
            out = before.clone()
        elif _gated(name):
            gate, up = before.chunk(2, dim=1)
            out = _exact_act(gate, name[-4:]) * up
        else:
            out = _exact_act(before, name)
        if s["residual"] is not None:
            end = s["ends"][-1]
            out[:end] += s["residual"][:end].double()
        return [out, before] if case["keep"] else out
    dx, dw = new(case["rows"], case["in"]), s["into"].double() if case["accumulate"] else new(*w.shape)
    db = new(case["experts"], case["out"])
    for e, span in spans:
        d = s["dout"][span].double()
        torch.matmul(d, w[e].double().t(), out=dx[span])
        dw[e] += torch.matmul(x[span].double().t(), d)
        db[e] = d.sum(0)
    return [dx, dw, db] if case["bias"] else [dx, dw]
