"""Plain 64-bit forms of the router and the experts' products, expert after expert, each with a bound on how far a 32-bit computation of it may be off.

The bounds, with u = 2^-24 (one rounding to 32 bits), before `layers_util.near` doubles them once for terms of second order.  A sum of k products whose
additions may cut off instead of rounding is off by at most (k + 1) 2u times the sum of their absolute values; a bias adds one rounding more.  An activation
hands an error on with its slope, which is at most 1.13 (silu 1.1, gelu 1.13), and adds its own: silu's sigmoid is good to (8 + 1.2 |x|) 2u of itself as a
gate is; gelu's normal distribution comes from erfc of an argument rounded twice, whose relative error is multiplied by at most x^2 + 1.  Slopes have the
same errors on each of their terms."""
import torch

from layers_util import U
from layers_util import near as near_finite

SLOPE = 1.13


def near(got, want, error):
    """layers_util.near; what lies past the middle between the type's largest number and the next power of two is rounded to infinity."""
    top = torch.finfo(got.dtype).max
    beyond = want.abs() - error > top * (1 + torch.finfo(got.dtype).eps / 4)
    assert (got[beyond].double() == want[beyond].sign() * torch.inf).all()
    near_finite(torch.where(beyond, 0.0, got).to(got.dtype), torch.where(beyond, 0.0, want), torch.where(beyond, 0.0, error))


def act(x, name):
    """(act(x), its slope, what a computation of either may be off by, for an exact x)"""
    if name is None:
        return x, torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x)
    if name == "silu":
        s, off = torch.sigmoid(x), (8 + 1.2 * x.abs().clamp(max=200)) * 2 * U
        return x * s, s * (1 + x * (1 - s)), off * (x * s).abs(), 4 * off * (s + (x * s).abs())
    p, off = 0.5 * torch.erfc(-x * 0.5 ** 0.5), (8 + 4 * (x * x).clamp(max=400)) * U
    bell = torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5
    return x * p, p + x * bell, off * (x * p).abs(), 4 * off * (p + (x * bell).abs())


def halves(name):
    return (name[6:], True) if name is not None and name.startswith("gated_") else (name, False)


def spans(offsets, n):
    at = [min(max(int(o), 0), n) for o in offsets.tolist()]
    return [(e, a, b) for e, (a, b) in enumerate(zip(at[:-1], at[1:])) if b > a]


def product(x, offsets, weight, bias=None, activation=None, residual=None):
    """(out, before, the errors of both)"""
    n, width = x.shape[0], weight.shape[2]
    before = torch.zeros(n, width, dtype=torch.float64, device=x.device)
    error = torch.zeros_like(before)
    for e, a, b in spans(offsets, n):
        r, w = x[a:b].double(), weight[e].double()
        before[a:b] = r @ w
        error[a:b] = (x.shape[1] + 1) * 2 * U * (r.abs() @ w.abs())
        if bias is not None:
            before[a:b] += bias[e].double()
            error[a:b] += U * before[a:b].abs()
    name, gated = halves(activation)
    half = width // 2 if gated else width
    y, _, off, _ = act(before[:, :half], name)
    eout = SLOPE * error[:, :half] + off if name else error
    if gated:
        up = before[:, half:]
        eout = eout * up.abs() + error[:, half:] * y.abs() + U * (y * up).abs()
        y = y * up
    out = torch.zeros_like(y)
    for e, a, b in spans(offsets, n):
        out[a:b] = y[a:b] if residual is None else y[a:b] + residual[a:b].double()
    if residual is not None:
        eout = eout + U * out.abs()
    return out, before, eout, error


def activation_grad(dout, before, activation):
    """(dbefore, its error)"""
    name, gated = halves(activation)
    d, x = dout.double(), before.double()
    if not gated:
        _, s, _, off = act(x, name)
        return d * s, d.abs() * (off + 2 * U * s.abs())
    half = x.shape[1] // 2
    y, s, oy, os = act(x[:, :half], name)
    up = x[:, half:]
    return (torch.cat([d * up * s, d * y], 1),
            torch.cat([(d * up).abs() * (os + 4 * U * s.abs()), d.abs() * (oy + 2 * U * y.abs())], 1))


def product_grad(dout, x, offsets, weight, into=None):
    """(drows, dweight, dbias, the errors of the three)"""
    n = x.shape[0]
    experts, i, o = weight.shape
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=x.device)  # noqa: E731
    dx, edx, dw, edw, db, edb = new(n, i), new(n, i), new(experts, i, o), new(experts, i, o), new(experts, o), new(experts, o)
    for e, a, b in spans(offsets, n):
        r, d, w = x[a:b].double(), dout[a:b].double(), weight[e].double()
        dx[a:b], edx[a:b] = d @ w.t(), (o + 1) * 2 * U * (d.abs() @ w.abs().t())
        dw[e], edw[e] = r.t() @ d, (b - a + 1) * 2 * U * (r.abs().t() @ d.abs())
        db[e], edb[e] = d.sum(0), (b - a + 1) * U * d.abs().sum(0)
    if into is not None:
        edw = edw + U * (dw.abs() + into.double().abs())
        dw = dw + into.double()
    return dx, dw, db, edx, edw, edb


# ------------------------------------------------------------------------------------------------ routing
def scores(logits, kind):
    """In 64 bits, and which experts are open"""
    x = logits.double()
    is_open = x > -torch.inf
    if kind == "sigmoid":
        return torch.where(is_open, torch.sigmoid(x), 0.0), is_open
    top = torch.where(is_open, x, -torch.inf).amax(1, keepdim=True)
    e = torch.where(is_open, torch.where(x == top, 1.0, torch.exp(x - top)), 0.0)
    return e / e.sum(1, keepdim=True).clamp(min=1.0), is_open


def route(logits, choices, kind="softmax", bias=None, groups=1, group_choices=None, group_best=2, renormalize=True, scale=1.0):
    """(experts, weights) on the host, row after row and choice after choice"""
    score, is_open = scores(logits, kind)
    n, e = logits.shape
    size, group_choices = e // groups, groups if group_choices is None else group_choices
    score, is_open, x = score.cpu().tolist(), is_open.cpu().tolist(), logits.double().cpu().tolist()
    bias = None if bias is None else bias.double().cpu().tolist()
    ids, weights = [], []
    for r in range(n):
        value = [(score[r][c] if bias is None else score[r][c] + bias[c]) if is_open[r][c] else float("-inf") for c in range(e)]
        value = [v if v > float("-inf") else float("-inf") for v in value]
        order = [x[r][c] if value[c] > float("-inf") else value[c] for c in range(e)] if bias is None else list(value)
        if groups > 1:
            rank = []
            for g in range(groups):
                by = sorted((value if group_best == 2 else order)[g * size:(g + 1) * size], reverse=True)[:group_best]
                rank.append(sum(v for v in by if v > float("-inf")) if by[0] > float("-inf") else float("-inf"))
            kept = sorted(range(groups), key=lambda g: (-rank[g], g))[:group_choices]
            order = [v if c // size in kept else float("-inf") for c, v in enumerate(order)]
        best = [c for c in sorted(range(e), key=lambda c: (-order[c], c))[:choices] if order[c] > float("-inf")]
        w = [score[r][c] for c in best]
        if renormalize:
            total = sum(w)
            w = [v / total if total else 0.0 for v in w]
        ids.append(best + [-1] * (choices - len(best)))
        weights.append([scale * v for v in w] + [0.0] * (choices - len(best)))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(weights, dtype=torch.float64)


def route_grad(dweights, experts, logits, kind="softmax", renormalize=True, scale=1.0):
    """By autograd, in 64 bits"""
    x = logits.double().detach().clone()
    is_open = x > -torch.inf
    x = torch.where(is_open, x, 0.0).requires_grad_()
    if kind == "sigmoid":
        score = torch.where(is_open, torch.sigmoid(x), 0.0)
    else:
        shifted = torch.where(is_open, x, -torch.inf)
        top = shifted.amax(1, keepdim=True).detach()
        e = torch.where(is_open, torch.exp(x - torch.where(top > -torch.inf, top, 0.0)), 0.0)
        score = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    at = experts.long()
    valid = (at >= 0) & (at < logits.shape[1])
    valid &= torch.gather(is_open, 1, at.clamp(0, logits.shape[1] - 1))
    w = torch.where(valid, torch.gather(score, 1, at.clamp(0, logits.shape[1] - 1)), 0.0)
    if renormalize:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    (scale * w * torch.where(valid, dweights.double(), 0.0)).sum().backward()
    return torch.where(is_open, x.grad, 0.0)
