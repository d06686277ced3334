"""Plain 64-bit forms of the operators on rows, token after token and id after id, each with a bound on how far a 32-bit
computation of it may be off.

The bounds.  u = 2^-24 is what one rounding to 32 bits costs, STORE[t] what the rounding of a stored result costs.  A sum of m products in
any order is off by at most (m + 1) u times the sum of their absolute values.  keep and give of a gate g come from an exponential that is good to
2 + 1.2 |g| units in its last place (2 u each), a reciprocal and a product: GATE(g) = (8 + 1.2 |g|) 2u each, relatively.  The recurrence hands its
error on multiplied by keep, and a step adds at most GATE + 4u of what it adds up; that holds for any grouping of the steps, in which a
product of m gates is off by m GATE at most, just as the m steps are.  Everything is doubled once at the end for terms of second order."""
import torch

U = 2.0 ** -24
STORE = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}     # below the smallest normal number steps are even


def gate_error(g):
    return (8 + 1.2 * g.abs().clamp(max=100)) * 2 * U      # past 100 the exponential is zero


def near(got, want, error):
    """got within `error` (of 32-bit arithmetic) of want, after one rounding to got's type."""
    assert got.shape == want.shape
    g = got.double()
    bound = 2 * error + STORE[got.dtype] * (want.abs() + 2 * error) + 2 * U * want.abs() + TINY[got.dtype]
    ok = (g - want).abs() <= bound
    if not bool(ok.all()):
        at = torch.nonzero(~ok)[0].tolist()
        raise AssertionError("at %s: got %r, want %r, bound %r; %d of %d off" % (at, g[tuple(at)].item(), want[tuple(at)].item(), bound[tuple(at)].item(),
                                                                              int((~ok).sum()), ok.numel()))


# ------------------------------------------------------------------------------------------------ embedding
def embedding(weight, tokens, scale):
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < weight.shape[0])
    out = torch.zeros(flat.numel(), weight.shape[1], dtype=torch.float64, device=weight.device)
    out[ok] = weight[flat[ok]].double() * scale
    return out.view(tuple(tokens.shape) + (weight.shape[1],))


def embedding_grad(dout, tokens, rows, scale, into=None):
    """(the gradient, the bound of its error)"""
    flat, d = tokens.reshape(-1).long(), dout.reshape(-1, dout.shape[-1])
    ok = (flat >= 0) & (flat < rows)
    sums = torch.zeros(rows, d.shape[1], dtype=torch.float64, device=d.device)
    size, count = torch.zeros_like(sums), torch.zeros(rows, 1, dtype=torch.float64, device=d.device)
    sums.index_add_(0, flat[ok], d[ok].double())
    size.index_add_(0, flat[ok], d[ok].double().abs())
    count.index_add_(0, flat[ok], torch.ones(int(ok.sum()), 1, dtype=torch.float64, device=d.device))
    sums, error = sums * scale, (count + 3) * U * size * abs(scale)
    if into is not None:
        error = error + U * (sums.abs() + into.double().abs())
        sums = sums + into.double()
    return sums, error


# ------------------------------------------------------------------------------------------------ gated scan
def _spans(x, offsets):
    if offsets is not None:
        o = offsets.tolist()
        return list(zip(o[:-1], o[1:]))
    if x.dim() == 2:
        return [(0, x.shape[0])]
    return [(b * x.shape[1], (b + 1) * x.shape[1]) for b in range(x.shape[0])]


def _flat(t):
    return t.reshape(-1, t.shape[-1]).double()


def gated_scan(x, gate, h0=None, offsets=None):
    """(h, last, their errors); sequences of equal length are walked together"""
    spans = _spans(x, offsets)
    xf, gf = _flat(x), _flat(gate)
    keep, give, wrong = torch.sigmoid(gf), torch.sigmoid(-gf), gate_error(gf) + 4 * U
    h, eh = torch.zeros_like(xf), torch.zeros_like(xf)
    last = torch.zeros(len(spans), xf.shape[1], dtype=torch.float64, device=x.device) if h0 is None else h0.double().clone()
    elast = torch.zeros_like(last)
    for group in _groups(spans):
        seqs = torch.tensor(group, device=x.device)
        first = torch.tensor([spans[s][0] for s in group], device=x.device)
        state, e = last[seqs], elast[seqs]
        for t in range(spans[group[0]][1] - spans[group[0]][0]):
            r = first + t
            e = keep[r] * e + wrong[r] * ((keep[r] * state).abs() + (give[r] * xf[r]).abs())
            state = keep[r] * state + give[r] * xf[r]
            h[r], eh[r] = state, e
        last[seqs], elast[seqs] = state, e
    return h.view(x.shape), last, eh.view(x.shape), elast


def gated_scan_grad(dh, x, gate, h, h0=None, dlast=None, offsets=None):
    """(dx, dgate, dh0, their errors)"""
    spans = _spans(x, offsets)
    xf, gf, hf, df = _flat(x), _flat(gate), _flat(h), _flat(dh)
    keep, give, wrong = torch.sigmoid(gf), torch.sigmoid(-gf), gate_error(gf) + 4 * U
    dx, dgate, edx, edgate = (torch.zeros_like(xf) for _ in range(4))
    zero = torch.zeros(len(spans), xf.shape[1], dtype=torch.float64, device=x.device)
    start = zero if h0 is None else h0.double()
    dh0 = zero.clone() if dlast is None else dlast.double().clone()
    edh0 = zero.clone()
    for group in _groups(spans):
        seqs = torch.tensor(group, device=x.device)
        first = torch.tensor([spans[s][0] for s in group], device=x.device)
        carry, e = dh0[seqs], edh0[seqs]
        for t in range(spans[group[0]][1] - spans[group[0]][0] - 1, -1, -1):
            r = first + t
            before = hf[r - 1] if t else start[seqs]
            e = e + U * (df[r].abs() + carry.abs())
            total = df[r] + carry
            slope = keep[r] * give[r]
            dx[r], edx[r] = give[r] * total, give[r] * (e + wrong[r] * total.abs())
            dgate[r] = slope * (before - xf[r]) * total
            edgate[r] = slope * ((before - xf[r]).abs() * (e + 2 * wrong[r] * total.abs()) + U * (before.abs() + xf[r].abs()) * total.abs())
            carry, e = keep[r] * total, keep[r] * (e + wrong[r] * total.abs())
        dh0[seqs], edh0[seqs] = carry, e
    return dx.view(x.shape), dgate.view(x.shape), dh0, edx.view(x.shape), edgate.view(x.shape), edh0


def _groups(spans):
    by_length = {}
    for s, (a, b) in enumerate(spans):
        by_length.setdefault(b - a, []).append(s)
    return by_length.values()


# ------------------------------------------------------------------------------------------------ experts
def plan(experts, num_experts):
    """(slots, sources, offsets) as lists, expert after expert and assignment after assignment"""
    flat = experts.reshape(-1).tolist()
    places = [[] for _ in range(num_experts)]
    for i, e in enumerate(flat):
        if 0 <= e < num_experts:
            places[e].append(i)
    slots, sources, offsets = [-1] * len(flat), [], [0]
    for p in places:
        for i in p:
            slots[i] = len(sources)
            sources.append(i)
        offsets.append(len(sources))
    return slots, sources + [-1] * (len(flat) - len(sources)), offsets


def combine(rows, slots, weights=None):
    """(out, its error)"""
    n, k = slots.shape
    ok = slots >= 0
    part = torch.zeros(n, k, rows.shape[1], dtype=torch.float64, device=rows.device)
    part[ok] = rows[slots[ok].long()].double()
    if weights is not None:
        part[ok] = part[ok] * weights[ok].double()[:, None]
    return part.sum(1), (k + 1) * U * part.abs().sum(1)


def combine_grad(dout, rows, slots, weights):
    """(drows, dweights, the errors of both)"""
    ok = slots >= 0
    drows = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device)
    dweights = torch.zeros(slots.shape, dtype=torch.float64, device=rows.device)
    size = torch.zeros_like(dweights)
    token = torch.nonzero(ok)[:, 0]
    at = slots[ok].long()
    drows[at] = dout[token].double() * weights[ok].double()[:, None]
    products = dout[token].double() * rows[at].double()
    dweights[ok] = products.sum(1)
    size[ok] = products.abs().sum(1)
    return drows, dweights, U * drows.abs(), (rows.shape[1] + 1) * U * size
