"""Performance cases: operators of a language model's layers on rows of channels, through the public Python entry points.

Three operators and their gradients: rows looked up by token (`embedding`), a gated linear recurrence along a sequence
(`gated_scan`, and `gated_step` for one token of each sequence), and rows sorted by expert and back (`expert_dispatch`,
`expert_combine`).  A case is one call on device-resident data.  Sizes go from the rows of one decoding step, where a call is
launches and latency, up to the batches of a training step.

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

#: the most bytes (by work()) that a drawn case moves
MOST_BYTES = 700e6


def listed():
    return [
        # the tokens of one decoding step of a batch of requests
        {"name": "embedding_decode", "op": "embedding", "n": 48, "rows": 50000, "dim": 2048, "type": "bf16", "ids": "i64", "padding": 0.0},
        # a prefill of packed prompts with padding between them
        {"name": "embedding_prefill", "op": "embedding", "n": 16391, "rows": 100003, "dim": 4096, "type": "bf16", "ids": "i32", "padding": 0.04},
        # a micro-batch added to a 32-bit main gradient
        {"name": "embedding_grad_microbatch", "op": "embedding_grad", "n": 4099, "rows": 32000, "dim": 1000, "type": "bf16", "out": "f32",
         "ids": "i64", "padding": 0.0, "accumulate": True},
        # the whole gradient of a large training batch
        {"name": "embedding_grad_batch", "op": "embedding_grad", "n": 65536, "rows": 128000, "dim": 2048, "type": "bf16", "out": "bf16",
         "ids": "i64", "padding": 0.02, "accumulate": False},
        # one token of each request in flight, states kept in a pool, some places of the batch unused
        {"name": "gated_step_decode", "op": "gated_step", "n": 96, "pool": 128, "dim": 4096, "type": "bf16", "ids": "i32", "unused": 0.1},
        # a prefill of packed prompts of unequal lengths, each with the state it continues from
        {"name": "gated_scan_packed", "op": "gated_scan", "batch": 37, "rows": 20011, "dim": 2560, "type": "bf16", "packed": True, "ids": "i32",
         "initial": True, "fused": True, "tail": 0},
        # one long document, few channels, 32 bits
        {"name": "gated_scan_long", "op": "gated_scan", "batch": 1, "rows": 65537, "dim": 1024, "type": "f32", "packed": False, "ids": "i32",
         "initial": False, "fused": False, "tail": 0},
        # the backward pass of a training batch
        {"name": "gated_scan_grad_batch", "op": "gated_scan_grad", "batch": 8, "rows": 8 * 4096, "dim": 2048, "type": "bf16", "packed": False,
         "ids": "i32", "initial": False, "fused": False, "tail": 0},
        # one decoding step sent to its experts
        {"name": "expert_dispatch_decode", "op": "expert_dispatch", "n": 33, "choices": 4, "experts": 64, "dim": 2048, "type": "bf16", "ids": "i64",
         "dropped": 0.0},
        # a training batch sent to its experts, some assignments over capacity
        {"name": "expert_dispatch_batch", "op": "expert_dispatch", "n": 16384, "choices": 8, "experts": 128, "dim": 2048, "type": "bf16", "ids": "i64",
         "dropped": 0.03},
        # what two of a few large experts made of a prefill, added up
        {"name": "expert_combine_prefill", "op": "expert_combine", "n": 8191, "choices": 2, "experts": 8, "dim": 4096, "type": "f16", "ids": "i32",
         "dropped": 0.0, "weighted": True},
        # the backward pass of a training batch
        {"name": "expert_combine_grad_batch", "op": "expert_combine_grad", "n": 16384, "choices": 6, "experts": 64, "dim": 2048, "type": "bf16",
         "ids": "i64", "dropped": 0.02},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    ops = ["embedding", "embedding_grad", "gated_scan", "gated_scan_grad", "gated_step", "expert_dispatch", "expert_combine", "expert_combine_grad",
           "expert_dispatch_grad"]
    while True:
        case = {"op": rng.choice(ops), "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "ids": rng.choice(["i32", "i64"])}
        op = case["op"]
        # most widths are a power of two or 5/4 or 7/4 of one, some are odd
        case["dim"] = _log_uniform(rng, 32, 8192) | 1 if rng.random() < 0.25 else rng.choice([4, 5, 7]) << rng.randint(4, 10)
        if op in ("embedding", "embedding_grad"):
            case.update(n=_log_uniform(rng, 1, 65536), rows=_log_uniform(rng, 100, 200000), padding=rng.choice([0.0, 0.0, 0.05, 0.5]))
            if op == "embedding_grad":
                case.update(out=rng.choice([case["type"], "f32"]), accumulate=rng.random() < 0.4)
        elif op == "gated_step":
            n = _log_uniform(rng, 1, 2048)
            case.update(n=n, pool=n + rng.randrange(0, n + 1), unused=rng.choice([0.0, 0.1, 0.5]))
        elif op in ("gated_scan", "gated_scan_grad"):
            batch, length = _log_uniform(rng, 1, 256), _log_uniform(rng, 1, 65536)
            packed = rng.random() < 0.5
            rows = batch * length + (rng.randrange(0, batch) if packed else 0)
            case.update(batch=batch, packed=packed, rows=rows, initial=rng.random() < 0.5, fused=rng.random() < 0.5,
                        tail=rows // 20 if packed and rng.random() < 0.3 else 0)
        else:
            experts = _log_uniform(rng, 2, 512)
            case.update(n=_log_uniform(rng, 1, 65536), experts=experts, choices=rng.randint(1, min(8, experts)), dropped=rng.choice([0.0, 0.0, 0.05, 0.5]))
            if op == "expert_combine":
                case["weighted"] = rng.random() < 0.8
        if work(case)["bytes"] <= MOST_BYTES:
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _tokens(g, n, rows, padding, ids):
    """Token ids as frequent as words are (the share of the r-th most frequent falls as 1/r), in no order; -1 for padding."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    tok = (rank * 7919 + 17) % rows          # 7919 is prime and divides no `rows` that matters: a permutation, or nearly one
    if padding:
        tok = torch.where(torch.rand(n, generator=g, device="cuda") < padding, -1, tok)
    return tok.to(IDS[ids])


def _expected_distinct(n, rows):
    """How many different ids _tokens draws on average."""
    r = np.arange(1, rows + 1, dtype=np.float64)
    p = np.log1p(1.0 / r) / math.log(rows + 1.0)
    return float(np.sum(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def _normal(g, shape, dtype, scale=1.0):
    out = torch.empty(shape, device="cuda", dtype=dtype)
    return out.normal_(0.0, scale, generator=g)


def _assignments(g, case):
    """The best `choices` of each token's router scores (some experts are liked better), their weights, dropped ones with id -1; of the
    tokens one in fifty is padding and goes to no expert."""
    n, e, k = case["n"], case["experts"], case["choices"]
    score = torch.randn(n, e, generator=g, device="cuda") + 0.7 * torch.randn(e, generator=g, device="cuda")
    top, ids = torch.topk(score, k, dim=1)
    weights = torch.softmax(top, dim=1).contiguous()
    if case["dropped"]:
        gone = torch.rand(n, k, generator=g, device="cuda") < case["dropped"]
        gone |= torch.rand(n, 1, generator=g, device="cuda") < 0.02
        ids = torch.where(gone, -1, ids)
    return ids.to(IDS[case["ids"]]).contiguous(), weights


def _offsets(g, case):
    """Where the packed sequences begin: unequal lengths (a length of zero may be among them), and an end, behind which there may
    be a tail of rows that are no sequence's."""
    end = case["rows"] - case["tail"]
    cut = torch.rand(case["batch"] - 1, generator=g, device="cuda", dtype=torch.float64)
    cut = (cut * (end + 1)).long().sort().values
    first, last = torch.zeros(1, device="cuda", dtype=torch.long), torch.full((1,), end, device="cuda", dtype=torch.long)
    return torch.cat([first, cut, last]).to(IDS[case["ids"]])


def _sequence_inputs(g, case):
    n, d, b, t = case["rows"], case["dim"], case["batch"], DTYPES[case["type"]]
    shape = (n, d) if case["packed"] else (b, n // b, d)
    # most channels keep a state for tens of tokens, some for thousands
    keep = 1.0 + 5.0 * torch.rand(d, generator=g, device="cuda")
    if case["fused"]:      # x and gate are the halves of one projection's output
        both = _normal(g, shape[:-1] + (2 * d,), t)
        x, gate = both[..., :d], both[..., d:]
    else:
        x, gate = _normal(g, shape, t), _normal(g, shape, t)
    gate.add_(keep.to(t))
    s = {"x": x, "gate": gate, "offsets": _offsets(g, case) if case["packed"] else None,
         "h0": _normal(g, (b, d), torch.float32) if case["initial"] else None}
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, t = case["op"], DTYPES[case["type"]]
    s = {"op": op}
    if op in ("embedding", "embedding_grad"):
        s["tokens"] = _tokens(g, case["n"], case["rows"], case["padding"], case["ids"])
        s["scale"] = math.sqrt(case["dim"])
        if op == "embedding":
            s["weight"] = _normal(g, (case["rows"], case["dim"]), t, 0.02)
        else:
            s["dout"] = _normal(g, (case["n"], case["dim"]), t, 0.01)
            s["rows"], s["dtype"] = case["rows"], DTYPES[case["out"]]
            s["into"] = _normal(g, (case["rows"], case["dim"]), s["dtype"], 0.1) if case["accumulate"] else None
    elif op == "gated_step":
        n, d = case["n"], case["dim"]
        s["x"], s["gate"] = _normal(g, (n, d), t), _normal(g, (n, d), t).add_(2.0)
        s["state"] = _normal(g, (case["pool"], d), torch.float32)
        slots = torch.randperm(case["pool"], generator=g, device="cuda")[:n]
        s["slots"] = torch.where(torch.rand(n, generator=g, device="cuda") < case["unused"], -1, slots).to(IDS[case["ids"]])
    elif op in ("gated_scan", "gated_scan_grad"):
        s.update(_sequence_inputs(g, case))
        if op == "gated_scan_grad":
            s["h"] = _plain_gated_scan(s["x"], s["gate"], s["h0"], s["offsets"])[0]
            s["dh"] = _normal(g, tuple(s["x"].shape), t, 0.01)
            s["dlast"] = _normal(g, (case["batch"], case["dim"]), torch.float32, 0.01) if case["initial"] else None
    else:
        ids, weights = _assignments(g, case)
        s["experts"], s["ids"], s["weights"] = case["experts"], ids, weights
        if op == "expert_dispatch":
            s["x"] = _normal(g, (case["n"], case["dim"]), t)
        else:
            slots, sources, offsets = _plain_plan(ids, case["experts"])
            s["plan"] = (slots, sources, offsets)
            s["rows"] = _normal(g, (ids.numel(), case["dim"]), t)
            if op == "expert_combine_grad":
                s["dout"] = _normal(g, (case["n"], case["dim"]), t, 0.01)
            if op == "expert_dispatch_grad" or not case.get("weighted", True):
                s["weights"] = None
    return s


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_embedding(weight, tokens, scale):
    there = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight[torch.where(there, tokens, 0).long()].float() * scale
    return torch.where(there[:, None], rows, 0.0).to(weight.dtype)


def _plain_embedding_grad(dout, tokens, rows, scale, dtype, into):
    there = (tokens >= 0) & (tokens < rows)
    total = torch.zeros(rows, dout.shape[1], device=dout.device)
    total.index_add_(0, torch.where(there, tokens, 0).long(), torch.where(there[:, None], dout.float() * scale, 0.0))
    if into is None:
        return total.to(dtype)
    return into.copy_(into.float() + total)


def _linear_scan(a, b):
    """h[i] = a[i] h[i-1] + b[i] along the first axis: neighbours joined, half as many solved, the others put in between."""
    n = a.shape[0]
    if n == 1:
        return b
    m = n // 2
    odd = _linear_scan(a[1::2] * a[0:2 * m:2], a[1::2] * b[0:2 * m:2] + b[1::2])
    h = torch.empty_like(b)
    h[1::2] = odd
    h[0] = b[0]
    h[2::2] = a[2::2] * odd[:(n - 1) // 2] + b[2::2]
    return h


def _places(n, batch, offsets):
    """Of each row: its sequence, whether it is in one at all, whether it is the first or the last of it."""
    if offsets is None:
        offsets = torch.arange(batch + 1, device="cuda") * (n // batch)
    offsets = offsets.long()
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(offsets, row, right=True) - 1
    inside = (seq >= 0) & (seq < offsets.numel() - 1)
    seq = seq.clamp(0, offsets.numel() - 2)
    return offsets, seq, inside[:, None], (row == offsets[seq])[:, None], (row + 1 == offsets[seq + 1])[:, None]


def _plain_gated_scan(x, gate, h0, offsets):
    d = x.shape[-1]
    batch = offsets.numel() - 1 if offsets is not None else x.shape[0] if x.dim() == 3 else 1
    xf, gf = x.reshape(-1, d).float(), gate.reshape(-1, d).float()
    offsets, seq, inside, first, _ = _places(xf.shape[0], batch, offsets)
    start = torch.zeros(batch, d, device="cuda") if h0 is None else h0
    a, b = torch.sigmoid(gf), torch.sigmoid(-gf) * xf
    b = torch.where(inside, torch.where(first, b + a * start[seq], b), 0.0)
    a = torch.where(inside & ~first, a, 0.0)
    h = _linear_scan(a, b)
    empty = offsets[1:] == offsets[:-1]
    last = torch.where(empty[:, None], start, h[(offsets[1:] - 1).clamp(min=0)])
    return h.to(x.dtype).view(x.shape), last


def _plain_gated_scan_grad(dh, x, gate, h, h0, dlast, offsets):
    d = x.shape[-1]
    batch = offsets.numel() - 1 if offsets is not None else x.shape[0] if x.dim() == 3 else 1
    xf, gf, hf, df = (v.reshape(-1, d).float() for v in (x, gate, h, dh))
    offsets, seq, inside, first, final = _places(xf.shape[0], batch, offsets)
    zero = torch.zeros(batch, d, device="cuda")
    start, end = zero if h0 is None else h0, zero if dlast is None else dlast
    a, c = torch.sigmoid(gf), torch.sigmoid(-gf)
    b = torch.where(inside, torch.where(final, df + end[seq], df), 0.0)
    after = torch.where(inside & ~final, torch.cat([a[1:], torch.zeros_like(a[:1])]), 0.0)
    s = _linear_scan(after.flip(0), b.flip(0)).flip(0)
    before = torch.where(first, start[seq], torch.cat([torch.zeros_like(hf[:1]), hf[:-1]]))
    dx = torch.where(inside, c * s, 0.0)
    dgate = torch.where(inside, a * c * (before - xf) * s, 0.0)
    at = offsets[:-1].clamp(max=xf.shape[0] - 1)
    empty = offsets[1:] == offsets[:-1]
    dh0 = torch.where(empty[:, None], end, a[at] * s[at])
    return dx.to(x.dtype).view(x.shape), dgate.to(x.dtype).view(x.shape), dh0


def _plain_gated_step(x, gate, state, slots):
    there = (slots >= 0) & (slots < state.shape[0])
    at = torch.where(there, slots, 0).long()
    h = torch.sigmoid(gate.float()) * state[at] + torch.sigmoid(-gate.float()) * x.float()
    h = torch.where(there[:, None], h, 0.0)
    # unused places add nothing to row 0
    state.index_add_(0, at, torch.where(there[:, None], h - state[at], 0.0))
    return h.to(x.dtype)


def _plain_plan(ids, experts):
    flat = ids.reshape(-1).long()
    m = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(m, device="cuda")
    kept = key < experts
    slots = torch.where(kept, place, -1).int().view(ids.shape)
    sources = torch.where(kept[order], order, -1).int()
    offsets = torch.searchsorted(key[order], torch.arange(experts + 1, device="cuda")).int()
    return slots, sources, offsets


def _plain_dispatch(x, ids, experts):
    plan = _plain_plan(ids, experts)
    sources = plan[1].long()
    rows = torch.where((sources >= 0)[:, None], x[sources.clamp(min=0) // ids.shape[1]], 0.0)
    return rows, plan


def _plain_combine(rows, slots, weights):
    kept = slots >= 0
    part = torch.where(kept[..., None], rows[slots.clamp(min=0).long()].float(), 0.0)
    if weights is not None:
        part = part * torch.where(kept, weights, 0.0)[..., None]
    return part.sum(1).to(rows.dtype)


def _plain_combine_grad(dout, rows, slots, sources, weights):
    kept, d = slots >= 0, dout.float()
    dweights = torch.where(kept, (rows[slots.clamp(min=0).long()].float() * d[:, None]).sum(2), 0.0)
    i = sources.long().clamp(min=0)
    drows = d[i // slots.shape[1]] * weights.reshape(-1)[i][:, None]
    return torch.where((sources >= 0)[:, None], drows, 0.0).to(rows.dtype), dweights


def run(s):
    op = s["op"]
    if own:
        import thrust_b200 as tb
        if op == "embedding":
            return tb.embedding(s["weight"], s["tokens"], s["scale"])
        if op == "embedding_grad":
            return tb.embedding_grad(s["dout"], s["tokens"], s["rows"], s["scale"], dtype=s["dtype"], out=s["into"], accumulate=s["into"] is not None)
        if op == "gated_scan":
            return tb.gated_scan(s["x"], s["gate"], s["h0"], s["offsets"])
        if op == "gated_scan_grad":
            return tb.gated_scan_grad(s["dh"], s["x"], s["gate"], s["h"], s["h0"], s["dlast"], s["offsets"])
        if op == "gated_step":
            return tb.gated_step(s["x"], s["gate"], s["state"], s["slots"]), s["state"]
        if op == "expert_dispatch":
            rows, plan = tb.expert_dispatch(s["x"], s["ids"], s["experts"])
            return rows, tuple(plan)
        if op == "expert_combine":
            return tb.expert_combine(s["rows"], tb.ExpertPlan(*s["plan"]), s["weights"])
        if op == "expert_combine_grad":
            return tb.expert_combine_grad(s["dout"], s["rows"], tb.ExpertPlan(*s["plan"]), s["weights"])
        return tb.expert_dispatch_grad(s["rows"], tb.ExpertPlan(*s["plan"]))
    if op == "embedding":
        return _plain_embedding(s["weight"], s["tokens"], s["scale"])
    if op == "embedding_grad":
        return _plain_embedding_grad(s["dout"], s["tokens"], s["rows"], s["scale"], s["dtype"], s["into"])
    if op == "gated_scan":
        return _plain_gated_scan(s["x"], s["gate"], s["h0"], s["offsets"])
    if op == "gated_scan_grad":
        return _plain_gated_scan_grad(s["dh"], s["x"], s["gate"], s["h"], s["h0"], s["dlast"], s["offsets"])
    if op == "gated_step":
        return _plain_gated_step(s["x"], s["gate"], s["state"], s["slots"]), s["state"]
    if op == "expert_dispatch":
        return _plain_dispatch(s["x"], s["ids"], s["experts"])
    if op == "expert_combine":
        return _plain_combine(s["rows"], s["plan"][0], s["weights"])
    if op == "expert_combine_grad":
        return _plain_combine_grad(s["dout"], s["rows"], s["plan"][0], s["plan"][1], s["weights"])
    return _plain_combine(s["rows"], s["plan"][0], None)


# ------------------------------------------------------------------------------------------------------ what it costs
def work(case):
    op, d, e = case["op"], case["dim"], SIZE[case["type"]]
    i = 4 if case["ids"] == "i32" else 8
    if op in ("embedding", "embedding_grad"):
        n = case["n"]
        used = n * (1.0 - case["padding"])
        distinct = _expected_distinct(used, case["rows"])
        if op == "embedding":
            return {"bytes": n * i + distinct * d * e + n * d * e, "flops": used * d}
        o = SIZE[case["out"]]
        return {"bytes": n * i + used * d * e + (2 * distinct if case["accumulate"] else case["rows"]) * d * o, "flops": 2 * used * d}
    if op == "gated_step":
        used = case["n"] * (1.0 - case["unused"])
        return {"bytes": case["n"] * i + used * d * (2 * e + 8) + case["n"] * d * e, "flops": 10 * used * d}
    if op in ("gated_scan", "gated_scan_grad"):
        n, states = case["rows"] * d, case["batch"] * d * 4
        places = (case["batch"] + 1) * i if case["packed"] else 0
        if op == "gated_scan":
            return {"bytes": 3 * n * e + states * (2 if case["initial"] else 1) + places, "flops": 10 * n}
        return {"bytes": 6 * n * e + states * (3 if case["initial"] else 1) + places, "flops": 16 * n}
    n, m = case["n"], case["n"] * case["choices"]
    gone = 1.0 - (1.0 - case["dropped"]) * 0.98 if case["dropped"] else 0.0
    kept = m * (1.0 - gone)
    if op == "expert_dispatch":
        return {"bytes": m * i + n * d * e + m * d * e + 8 * m + 4 * (case["experts"] + 1), "flops": m}
    if op == "expert_combine_grad":
        return {"bytes": 12 * m + (n + kept + m) * d * e, "flops": 3 * kept * d}
    weighted = op == "expert_combine" and case["weighted"]
    return {"bytes": (8 if weighted else 4) * m + (kept + n) * d * e, "flops": (2 if weighted else 1) * kept * d}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_sequences(s):
    """Each sequence's first row and length, on the host."""
    x = s["x"]
    if s["offsets"] is not None:
        o = s["offsets"].cpu().numpy().astype(np.int64)
        return o[:-1], np.diff(o)
    b, t = x.shape[:2]
    return np.arange(b) * t, np.full(b, t)


def _exact_gated_scan(s):
    """Token after token of all sequences at once, the longer ones first, so that those which have ended are left off."""
    x, gate = s["x"].flatten(0, -2).double(), s["gate"].flatten(0, -2).double()
    first, length = _exact_sequences(s)
    order = np.argsort(-length, kind="stable")
    b, d = len(first), x.shape[1]
    state = torch.zeros(b, d, device="cuda", dtype=torch.float64) if s["h0"] is None else s["h0"].double()
    state = state[torch.from_numpy(order).cuda()].clone()
    at = torch.from_numpy(first[order]).cuda()
    h = torch.zeros_like(x)
    for t in range(int(length.max(initial=0))):
        live = int((length > t).sum())
        r = at[:live] + t
        keep = 1.0 / (1.0 + torch.exp(-gate[r]))
        state[:live] = x[r] + keep * (state[:live] - x[r])
        h[r] = state[:live]
    last = torch.empty_like(state)
    last[torch.from_numpy(order).cuda()] = state
    return [h.view(s["x"].shape), last]


def _exact_gated_scan_grad(s):
    shape, d = s["x"].shape, s["x"].shape[-1]
    x, gate, h, dh = (s[k].flatten(0, -2).double() for k in ("x", "gate", "h", "dh"))
    first, length = _exact_sequences(s)
    order = np.argsort(-length, kind="stable")
    b = len(first)
    back = torch.from_numpy(order).cuda()
    zero = torch.zeros(b, d, device="cuda", dtype=torch.float64)
    start = (zero if s["h0"] is None else s["h0"].double())[back]
    carry = (zero if s["dlast"] is None else s["dlast"].double())[back].clone()
    at = torch.from_numpy(first[order]).cuda()
    dx, dgate = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(int(length.max(initial=0)) - 1, -1, -1):
        live = int((length > t).sum())
        r = at[:live] + t
        keep = 1.0 / (1.0 + torch.exp(-gate[r]))
        before = start[:live] if t == 0 else h[r - 1]
        total = dh[r] + carry[:live]
        dx[r] = total * (1.0 - keep)
        dgate[r] = total * (before - x[r]) * keep * (1.0 - keep)
        carry[:live] = total * keep
    dh0 = torch.empty_like(carry)
    dh0[back] = carry
    return [dx.view(shape), dgate.view(shape), dh0]


def exact(case, seed):
    op = case["op"]
    if op in ("gated_scan", "gated_scan_grad"):
        s = prepare(case, seed)
        return _exact_gated_scan(s) if op == "gated_scan" else _exact_gated_scan_grad(s)
    s = prepare(case, seed)
    if op == "embedding":
        keep = (s["tokens"] >= 0) & (s["tokens"] < case["rows"])
        out = torch.zeros(case["n"], case["dim"], device="cuda", dtype=torch.float64)
        out[keep] = s["weight"][s["tokens"][keep].long()].double() * s["scale"]
        return out
    if op == "embedding_grad":
        out = torch.zeros(case["rows"], case["dim"], device="cuda", dtype=torch.float64)
        if s["into"] is not None:
            out += s["into"].double()
        keep = (s["tokens"] >= 0) & (s["tokens"] < case["rows"])
        out.index_put_((s["tokens"][keep].long(),), s["dout"][keep].double() * s["scale"], accumulate=True)
        return out
    if op == "gated_step":
        h, state = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float64), s["state"].double()
        used = torch.nonzero(s["slots"] >= 0)[:, 0]
        slot, keep = s["slots"][used].long(), 1.0 / (1.0 + torch.exp(-s["gate"][used].double()))
        state[slot] = keep * state[slot] + (1.0 - keep) * s["x"][used].double()
        h[used] = state[slot]
        return [h, state]
    if op == "expert_dispatch":
        flat = s["ids"].reshape(-1).cpu().numpy()
        order = np.concatenate([np.nonzero(flat == e)[0] for e in range(case["experts"])]).astype(np.int64)
        rows = torch.zeros(flat.size, case["dim"], device="cuda", dtype=torch.float64)
        rows[:order.size] = s["x"].double()[torch.from_numpy(order // case["choices"]).cuda()]
        return [rows, None]
    slots, weights = s["plan"][0], s["weights"]
    token, choice = torch.nonzero(slots >= 0, as_tuple=True)
    at = slots[token, choice].long()
    w = torch.ones(at.numel(), device="cuda", dtype=torch.float64) if weights is None else weights[token, choice].double()
    if op == "expert_combine_grad":
        drows = torch.zeros(s["rows"].shape, device="cuda", dtype=torch.float64)
        dweights = torch.zeros(slots.shape, device="cuda", dtype=torch.float64)
        d = s["dout"].double()[token]
        drows[at] = d * w[:, None]
        dweights[token, choice] = torch.einsum("id,id->i", d, s["rows"][at].double())
        return [drows, dweights]
    out = torch.zeros(case["n"], case["dim"], device="cuda", dtype=torch.float64)
    out.index_add_(0, token, s["rows"][at].double() * w[:, None])
    return out
