"""Operators on rows of channels, over the C ABI: what a language model's layers ask of gather, scan, sort and reduce_by_key.

Rows looked up by token and the gradient of the table (embedding, embedding_grad); a gated linear recurrence along
sequences, its gradient, and its form for one token of each sequence (gated_scan, gated_scan_grad, gated_step); rows sorted by
expert and back, with both gradients (expert_dispatch, expert_combine, expert_combine_grad, expert_dispatch_grad); which experts a token
goes to (expert_route, expert_route_grad) and what they make of its row (expert_product, expert_activation_grad, expert_product_grad).

Tensors live on the current CUDA device.  Rows are float32, float16 or bfloat16, their channels next to one another; the rows of an
input may lie further apart than they are long, evenly (one half of a fused projection, say), everything else is contiguous.
Arithmetic is in 32 bits and rounded once where a result is stored.  Ids are int32 or int64; an id outside its range names
nothing: its result is zero, and what belongs to it, NaNs included, reaches no result.  Outputs must not overlap inputs.

Every call only enqueues work on the current stream, like reduce_to_device.  There is no fallback path.
"""
import ctypes
from collections import namedtuple

import torch

from . import _lib, api
from .api import _call_and_wait, _check, _raw_stream, _stream_captures

__all__ = ["ExpertPlan", "embedding", "embedding_grad", "gated_scan", "gated_scan_grad", "gated_step", "expert_dispatch", "expert_combine",
           "expert_combine_grad", "expert_dispatch_grad", "expert_route", "expert_route_grad", "expert_product", "expert_activation_grad", "expert_product_grad"]

_ROW_CODE = {torch.float32: 8, torch.float16: 10, torch.bfloat16: 11}
_ID_CODE = {torch.int32: 4, torch.int64: 6}
_F32, _I32 = torch.float32, torch.int32
_SCORES = {"softmax": 0, "sigmoid": 1}
_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gated_silu": 5, "gated_gelu": 6}

#: What expert_dispatch found out: slots [tokens, choices], the place of each assignment among the rows (-1: none); sources
#: [tokens * choices], the assignment (token * choices + choice) at each place (-1 behind the last); offsets [experts + 1],
#: where each expert's rows begin, and last how many rows there are.  All int32.
ExpertPlan = namedtuple("ExpertPlan", "slots sources offsets")

# the current device without torch.cuda's checks, where torch offers that; asked only once a CUDA tensor has been seen
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _device_of(what, t):
    """The current device, which t must be on."""
    dev = t.get_device()
    if dev < 0 or dev != _current_device():
        raise ValueError("%s: a tensor on the current CUDA device is needed" % what)
    return dev


def _row_step(what, t, dev):
    """How many elements lie between the beginnings of neighbouring rows."""
    if t.get_device() != dev:
        raise ValueError("%s: a tensor on the current CUDA device is needed" % what)
    if t.dtype not in _ROW_CODE or t.dim() < 1:
        raise ValueError("%s: rows of float32, float16 or bfloat16 are needed" % what)
    if t.is_contiguous():
        return t.shape[-1]
    dim = t.shape[-1]
    step = expected = None
    for size, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
        if size == 1:
            continue
        if step is None:
            step = expected = stride
        elif stride != expected:
            raise ValueError("%s: rows that are not evenly spaced: make it contiguous" % what)
        expected *= size
    step = dim if step is None else step
    if (dim > 1 and t.stride(-1) != 1) or step < dim:
        raise ValueError("%s: channels of a row must be neighbours, and rows must not overlap: make it contiguous" % what)
    return step


def _packed(what, t, dtype, shape, dev):
    if t.get_device() != dev or t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s: a contiguous tensor of type %s and shape %s on the current CUDA device is needed" % (what, dtype, tuple(shape)))
    return t.data_ptr()


def _maybe(what, t, dtype, shape, dev):
    return None if t is None else _packed(what, t, dtype, shape, dev)


def _ids(what, t, dev):
    if t.get_device() != dev:
        raise ValueError("%s: a tensor on the current CUDA device is needed" % what)
    if t.dtype not in _ID_CODE or not t.is_contiguous():
        raise ValueError("%s: contiguous int32 or int64 ids are needed" % what)
    return _ID_CODE[t.dtype]


def _same(what, t, like, dev):
    """A second input like the first one: its row step."""
    if t.shape != like.shape or t.dtype != like.dtype:
        raise ValueError("%s: shape %s and type %s are needed" % (what, tuple(like.shape), like.dtype))
    return _row_step(what, t, dev)


def _enqueue(tag, what, fn, dev, *args):
    """A call with a workspace.  What is there is used as it is if it is large enough."""
    key = (dev, _raw_stream(dev), tag)
    kept = api.workspaces.at(key)
    with kept.lock:
        if kept.ptr is not None:
            rc = getattr(_lib.load(), fn)(*args, kept.ptr, kept.size_ref, key[1])
            if rc != 1:      # cudaErrorInvalidValue: too small, perhaps
                if kept.no_graph and _stream_captures():      # _Kept.used
                    kept.no_graph = False
                return _check(rc, what)
        _call_and_wait(tag, what, fn, *args, sync=False, key=key)      # made, or made larger, or the error raised


# ---------------------------------------------------------------------------------- rows by token
def embedding(weight, tokens, scale=1.0, out=None):
    """scale * weight[tokens]: weight [rows, dim], tokens of any shape; a token outside [0, rows) (padding) has a row of zeros.
    Returns tokens.shape + (dim,), of weight's type."""
    dev = _device_of("weight", weight)
    step, code = _row_step("weight", weight, dev), _ids("tokens", tokens, dev)
    if weight.dim() != 2:
        raise ValueError("weight: [rows, dim] is needed")
    rows, dim = weight.shape
    dtype = weight.dtype
    if out is None:
        out = torch.empty(*tokens.shape, dim, dtype=dtype, device=weight.device)
        to = out.data_ptr()
    else:
        to = _packed("out", out, dtype, tokens.shape + (dim,), dev)
    _check(_lib.load().tb200_embedding(weight.data_ptr(), rows, step, tokens.data_ptr(), code, tokens.numel(), dim, _ROW_CODE[dtype], scale, to, _raw_stream(dev)), "embedding")
    return out


def embedding_grad(dout, tokens, num_rows, scale=1.0, dtype=None, out=None, accumulate=False, sync=False):
    """The gradient of embedding's weight: [num_rows, dim] of type dtype (dout's by default), row v = scale * the sum of dout over the
    places of token v.  accumulate: added to `out` (a gradient that several micro-batches share; float32 as a rule).  The order of the
    sums is fixed, so the same inputs give the same bits.  sync: waits for the result and raises if the sort's waits ran out; without
    it such a failure shows as NaNs.  A result without elements is not waited for."""
    dev = _device_of("dout", dout)
    step, code = _row_step("dout", dout, dev), _ids("tokens", tokens, dev)
    dim = dout.shape[-1]
    if dout.shape[:-1] != tokens.shape:
        raise ValueError("dout: shape %s is needed" % (tuple(tokens.shape) + (dim,),))
    if num_rows < 0 or num_rows >= 1 << 31 or tokens.numel() >= 1 << 31:
        raise ValueError("rows and tokens are counted in 31 bits")
    if accumulate and out is None:
        raise ValueError("accumulate adds to `out`")
    dtype = out.dtype if out is not None and dtype is None else dtype or dout.dtype
    if dtype not in _ROW_CODE:
        raise ValueError("dtype: float32, float16 or bfloat16")
    out = torch.empty(num_rows, dim, dtype=dtype, device=dout.device) if out is None else out
    args = (dout.data_ptr(), step, tokens.data_ptr(), code, tokens.numel(), num_rows, dim, _ROW_CODE[dout.dtype], _ROW_CODE[dtype], scale, int(accumulate),
            _packed("out", out, dtype, (num_rows, dim), dev))
    if out.numel() == 0:      # nothing to write: no kernel runs, and the workspace says nothing of this call
        return out
    if sync:
        _call_and_wait("embedding_grad", "embedding_grad", "tb200_embedding_grad", *args)
    else:
        _enqueue("embedding_grad", "embedding_grad", "tb200_embedding_grad", dev, *args)
    return out


# ---------------------------------------------------------------------------------- gated recurrence
def _sequences(x, offsets, dev):
    """(batch, rows, dim, offsets' address, their code) of [batch, length, dim] or of [rows, dim] cut at offsets."""
    if x.dim() not in (2, 3) or (x.dim() == 3 and offsets is not None):
        raise ValueError("x: [batch, length, dim], or [rows, dim] with or without offsets")
    dim = x.shape[-1]
    if offsets is None:
        batch = x.shape[0] if x.dim() == 3 else 1
        return batch, x.shape[0] * x.shape[1] if x.dim() == 3 else x.shape[0], dim, None, 0
    code = _ids("offsets", offsets, dev)
    if offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("offsets: one more than there are sequences")
    return offsets.numel() - 1, x.shape[0], dim, offsets.data_ptr(), code


def gated_scan(x, gate, h0=None, offsets=None, out=None):
    """h[t] = a[t] h[t-1] + (1 - a[t]) x[t] with a = sigmoid(gate), in every channel of every sequence, from h0 (zeros by default).

    x, gate: [batch, length, dim], or [rows, dim]: one sequence, or those that `offsets` (ids [sequences + 1], not decreasing) cut the rows
    into, empty ones among them; rows outside [offsets[0], offsets[-1]) belong to none and have h = 0.  h0: float32 [sequences, dim].  A state that is
    not finite leaves no later one of its sequence finite.
    Returns (h, last): h as x, last float32 [sequences, dim], the unrounded state behind each sequence (h0's where that is empty)."""
    dev = _device_of("x", x)
    xs, gs = _row_step("x", x, dev), _same("gate", gate, x, dev)
    batch, n, dim, offs, code = _sequences(x, offsets, dev)
    dtype = x.dtype
    if out is None:
        h = torch.empty(x.shape, dtype=dtype, device=x.device)
        to = h.data_ptr()
    else:
        h, to = out, _packed("out", out, dtype, x.shape, dev)
    last = torch.empty(batch, dim, dtype=_F32, device=x.device)
    _enqueue("gated", "gated_scan", "tb200_gated_scan", dev, x.data_ptr(), xs, gate.data_ptr(), gs, _maybe("h0", h0, _F32, (batch, dim), dev), offs, code, batch, n, dim,
             _ROW_CODE[dtype], to, last.data_ptr())
    return h, last


def gated_scan_grad(dh, x, gate, h, h0=None, dlast=None, offsets=None):
    """The gradients of gated_scan's x, gate and h0, from those of h and of last (zeros by default); h is what gated_scan returned.
    Returns (dx, dgate, dh0): as x, as x, and float32 [sequences, dim]."""
    dev = _device_of("x", x)
    xs, ds, gs, hs = _row_step("x", x, dev), _same("dh", dh, x, dev), _same("gate", gate, x, dev), _same("h", h, x, dev)
    batch, n, dim, offs, code = _sequences(x, offsets, dev)
    dx, dgate = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dh0 = torch.empty(batch, dim, dtype=_F32, device=x.device)
    _enqueue("gated", "gated_scan_grad", "tb200_gated_scan_grad", dev, dh.data_ptr(), ds, x.data_ptr(), xs, gate.data_ptr(), gs, h.data_ptr(), hs,
             _maybe("h0", h0, _F32, (batch, dim), dev), _maybe("dlast", dlast, _F32, (batch, dim), dev), offs, code, batch, n, dim, _ROW_CODE[x.dtype], dx.data_ptr(),
             dgate.data_ptr(), dh0.data_ptr())
    return dx, dgate, dh0


def gated_step(x, gate, state, slots=None, out=None):
    """One token of each sequence: x, gate [n, dim]; state float32 [pool, dim] holds the sequences' states and is changed in place, row i uses
    state[slots[i]] (state[i] without slots).  A slot may occur once; one outside [0, pool) is an unused place of the batch.  Returns h [n, dim]."""
    dev = _device_of("x", x)
    xs, gs = _row_step("x", x, dev), _same("gate", gate, x, dev)
    if x.dim() != 2 or state.dim() != 2 or (slots is not None and slots.shape != x.shape[:1]):
        raise ValueError("x: [n, dim], state: [pool, dim], slots: [n]")
    n, dim = x.shape
    pool = state.shape[0]
    if slots is None and pool < n:
        raise ValueError("state: a row for each of x's is needed")
    at, code = (None, 0) if slots is None else (slots.data_ptr(), _ids("slots", slots, dev))
    if out is None:
        h = torch.empty(n, dim, dtype=x.dtype, device=x.device)
        to = h.data_ptr()
    else:
        h, to = out, _packed("out", out, x.dtype, x.shape, dev)
    _check(_lib.load().tb200_gated_step(x.data_ptr(), xs, gate.data_ptr(), gs, _packed("state", state, _F32, (pool, dim), dev), pool, at, code, n, dim, _ROW_CODE[x.dtype], to,
                                        _raw_stream(dev)), "gated_step")
    return h


# ---------------------------------------------------------------------------------- rows by expert
def _assignments(what, t):
    if t.dim() != 2 or not 1 <= t.shape[1] <= 32 or t.numel() >= 1 << 30:
        raise ValueError("%s: [tokens, choices] with 1 to 32 choices and less than 2^30 in all is needed" % what)
    return t.shape


def expert_dispatch(x, experts, num_experts):
    """Tokens' rows sorted by expert: x [tokens, dim], experts [tokens, choices] ids; those outside [0, num_experts) are dropped.
    Returns (rows, plan): rows [tokens * choices, dim], expert e's at plan.offsets[e] to plan.offsets[e + 1] in the order of their
    assignments, zeros behind the last; plan (an ExpertPlan) is what the way back needs."""
    dev = _device_of("x", x)
    step, code = _row_step("x", x, dev), _ids("experts", experts, dev)
    n, choices = _assignments("experts", experts)
    if x.dim() != 2 or x.shape[0] != n:
        raise ValueError("x: [%d, dim] is needed" % n)
    if not 1 <= num_experts <= 1024:
        raise ValueError("1 to 1024 experts")
    dim, m, device = x.shape[1], n * choices, x.device
    rows = torch.empty(m, dim, dtype=x.dtype, device=device)
    slots = torch.empty(n, choices, dtype=_I32, device=device)
    sources = torch.empty(m, dtype=_I32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=_I32, device=device)
    _enqueue("experts", "expert_dispatch", "tb200_expert_dispatch", dev, x.data_ptr(), step, experts.data_ptr(), code, n, choices, num_experts, dim, _ROW_CODE[x.dtype],
             rows.data_ptr(), slots.data_ptr(), sources.data_ptr(), offsets.data_ptr())
    return rows, ExpertPlan(slots, sources, offsets)


def _planned(rows, plan):
    dev = _device_of("rows", rows)
    slots = plan.slots
    n, choices = _assignments("plan.slots", slots)
    step = _row_step("rows", rows, dev)
    if rows.dim() != 2 or rows.shape[0] != n * choices:
        raise ValueError("rows: [%d, dim] is needed" % (n * choices))
    return dev, n, choices, rows.shape[1], step, _packed("plan.slots", slots, _I32, slots.shape, dev)


def expert_combine(rows, plan, weights=None):
    """The experts' rows brought back to their tokens and added up, in the order of the choices: out[t] = sum over k of weights[t, k] *
    rows[plan.slots[t, k]], dropped ones left out.  weights: float32 [tokens, choices]; None: all one.  Returns [tokens, dim]."""
    dev, n, choices, dim, step, slots = _planned(rows, plan)
    out = torch.empty(n, dim, dtype=rows.dtype, device=rows.device)
    _check(_lib.load().tb200_expert_combine(rows.data_ptr(), step, slots, _maybe("weights", weights, _F32, (n, choices), dev), n, choices, dim, _ROW_CODE[rows.dtype],
                                            out.data_ptr(), _raw_stream(dev)), "expert_combine")
    return out


def expert_combine_grad(dout, rows, plan, weights):
    """The gradients of expert_combine's rows and weights: drows as rows (zeros behind the last row in use), dweights as weights (zero
    where nothing was sent)."""
    dev, n, choices, dim, step, slots = _planned(rows, plan)
    if dout.shape != (n, dim) or dout.dtype != rows.dtype:
        raise ValueError("dout: shape %s and type %s are needed" % ((n, dim), rows.dtype))
    if weights is None:
        raise ValueError("weights: expert_combine's are needed (ones, if it was called without)")
    offsets = plan.offsets
    if offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("plan.offsets: one more than there are experts")
    drows = torch.empty(n * choices, dim, dtype=rows.dtype, device=rows.device)
    dweights = torch.empty(n, choices, dtype=_F32, device=rows.device)
    _check(_lib.load().tb200_expert_combine_grad(dout.data_ptr(), _row_step("dout", dout, dev), rows.data_ptr(), step, slots,
                                                 _packed("weights", weights, _F32, (n, choices), dev),
                                                 _packed("plan.offsets", offsets, _I32, offsets.shape, dev) + 4 * (offsets.numel() - 1), n, choices, dim,
                                                 _ROW_CODE[rows.dtype], drows.data_ptr(), dweights.data_ptr(), _raw_stream(dev)), "expert_combine_grad")
    return drows, dweights


def expert_dispatch_grad(drows, plan):
    """The gradient of expert_dispatch's x: each token's rows added up."""
    return expert_combine(drows, plan)


# ---------------------------------------------------------------------------------- routing
def _logits(logits, choices, scores):
    dev = _device_of("logits", logits)
    step = _row_step("logits", logits, dev)
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 1024:
        raise ValueError("logits: [tokens, experts] of 1 to 1024 experts is needed")
    if not 1 <= choices <= min(32, logits.shape[1]) or logits.shape[0] * choices >= 1 << 30:
        raise ValueError("choices: 1 to 32, no more than there are experts, and less than 2^30 in all")
    if scores not in _SCORES:
        raise ValueError('scores: "softmax" or "sigmoid"')
    return dev, step


def expert_route(logits, choices, scores="softmax", bias=None, groups=1, group_choices=None, group_best=2, renormalize=True, scale=1.0):
    """Which experts each token goes to: of logits [tokens, experts] the `choices` best by score + bias, the best first, the lower index
    before an equal one.  scores: "softmax" over the token's experts whose logit is neither NaN nor -infinity, or "sigmoid"; bias: float32 [experts], which takes
    part in the choice alone (an expert that it closes keeps its share of the softmax).  An expert whose logit, or score + bias, is NaN or -infinity is not open and never chosen.  groups: only the group_choices (all by
    default) best of so many equal groups of neighbouring experts take part, by the sum of their group_best (1 or 2) best score + bias.
    Returns (experts, weights): int32 [tokens, choices], -1 where no open expert is left (expert_dispatch drops it); float32, scale times the
    score, divided by the sum of the chosen ones' scores if renormalize, 0 where no expert is.  Scores are compared as 64-bit numbers."""
    dev, step = _logits(logits, choices, scores)
    n, e = logits.shape
    group_choices = groups if group_choices is None else group_choices
    if not 1 <= groups <= 32 or e % groups or not 1 <= group_choices <= groups or group_best not in (1, 2):
        raise ValueError("groups: 1 to 32 that divide the experts, group_choices: 1 to groups, group_best: 1 or 2")
    experts = torch.empty(n, choices, dtype=_I32, device=logits.device)
    weights = torch.empty(n, choices, dtype=_F32, device=logits.device)
    _check(_lib.load().tb200_expert_route(logits.data_ptr(), step, n, e, _ROW_CODE[logits.dtype], _maybe("bias", bias, _F32, (e,), dev), choices, _SCORES[scores], groups,
                                          group_choices, group_best, int(renormalize), scale, experts.data_ptr(), weights.data_ptr(), _raw_stream(dev)), "expert_route")
    return experts, weights


def expert_route_grad(dweights, experts, logits, scores="softmax", renormalize=True, scale=1.0):
    """The gradient of expert_route's logits, of their type, from that of its weights; experts is what it returned.  The choice has none, nor has
    the bias.  A choice that is no expert, or one whose logit is NaN or -infinity, has no part; choices of the same expert add up."""
    if experts.dim() != 2:
        raise ValueError("experts: [tokens, choices] is needed")
    choices = experts.shape[1]
    dev, step = _logits(logits, choices, scores)
    n, e = logits.shape
    dlogits = torch.empty(n, e, dtype=logits.dtype, device=logits.device)
    _check(_lib.load().tb200_expert_route_grad(_packed("dweights", dweights, _F32, (n, choices), dev), _packed("experts", experts, _I32, (n, choices), dev), logits.data_ptr(), step, n, e,
                                               choices, _ROW_CODE[logits.dtype], _SCORES[scores], int(renormalize), scale, dlogits.data_ptr(), _raw_stream(dev)), "expert_route_grad")
    return dlogits


# ---------------------------------------------------------------------------------- experts' products
def _enqueue_product(what, fn, dev, *args):
    """_enqueue, but a captured call has a workspace of its own, which belongs to the graph: operands are laid out anew there, and graphs that were captured
    on one stream may be replayed side by side."""
    if not _stream_captures():
        return _enqueue(what, what, fn, dev, *args)
    call, stream, need = getattr(_lib.load(), fn), _raw_stream(dev), ctypes.c_size_t(0)
    _check(call(*args, None, ctypes.byref(need), stream), what)
    room = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    _check(call(*args, room.data_ptr(), ctypes.byref(need), stream), what)


def _matrices(what, t, dev):
    """How [experts, in, out] lies: (experts' distance, rows' distance, whether inputs are neighbours instead of outputs)."""
    if t.get_device() != dev:
        raise ValueError("%s: a tensor on the current CUDA device is needed" % what)
    if t.dim() != 3 or not 1 <= t.shape[0] <= 1024 or max(t.shape[1:]) >= 1 << 24:
        raise ValueError("%s: [experts, in, out] of 1 to 1024 experts and less than 2^24 channels is needed" % what)
    experts, inputs, outputs = t.shape
    if t.is_contiguous():
        return inputs * outputs, outputs, 0
    each, i, o = t.stride()
    for inside, size, step, near, rows in ((0, outputs, i, o, inputs), (1, inputs, o, i, outputs)):
        if size == 1:
            near = 1
        if rows == 1:
            step = size
        if near == 1 and step >= size and (experts == 1 or each >= (rows - 1) * step + size):
            return each if experts > 1 else rows * step, step, inside
    raise ValueError("%s: inputs or outputs must be neighbours, and nothing may overlap: make it contiguous" % what)


def _rows_and_experts(rows, offsets, weight):
    dev = _device_of("rows", rows)
    step, code = _row_step("rows", rows, dev), _ids("offsets", offsets, dev)
    lies = _matrices("weight", weight, dev)
    if weight.dtype != rows.dtype or rows.dim() != 2 or rows.shape[1] != weight.shape[1]:
        raise ValueError("rows: [rows, in] and weight: [experts, in, out] of one type are needed")
    if offsets.dim() != 1 or offsets.numel() != weight.shape[0] + 1:
        raise ValueError("offsets: one more than there are experts")
    return dev, step, code, lies


def expert_product(rows, offsets, weight, bias=None, activation=None, residual=None, keep=False):
    """Each expert's rows times its matrix: before[i] = rows[i] @ weight[e] + bias[e] for the rows from offsets[e] to offsets[e + 1] (ids [experts + 1],
    not decreasing: expert_dispatch's plan.offsets), out = act(before) + residual; rows that are no expert's are zero.

    rows [n, in], weight [experts, in, out], contiguous or the transpose of such (out, in) matrices, bias [experts, out], residual as out, all of one
    type.  activation: None, "silu", "gelu" (by the error function), or "gated_silu", "gated_gelu": the outputs are halves [a | b], and act(a) * b comes
    of them.  Sums are 32 bits, rounded once; an infinite float32 operand may leave NaNs where the definition says infinity.  Returns out [n, out] (gated: [n, out / 2]); with keep (out, before), before [n, out] for expert_activation_grad."""
    dev, step, code, lies = _rows_and_experts(rows, offsets, weight)
    if activation not in _ACTIVATIONS:
        raise ValueError("activation: None, or one of %s" % ", ".join(k for k in _ACTIVATIONS if k))
    (experts, inputs, outputs), n, dtype, act = weight.shape, rows.shape[0], rows.dtype, _ACTIVATIONS[activation]
    if act & 4 and outputs % 2:
        raise ValueError("weight: a gated activation needs two halves of outputs")
    width = outputs // 2 if act & 4 else outputs
    to, extra = None, 0
    if residual is not None:
        if residual.shape != (n, width) or residual.dtype != dtype:
            raise ValueError("residual: shape %s and type %s are needed" % ((n, width), dtype))
        to, extra = residual.data_ptr(), _row_step("residual", residual, dev)
    out = torch.empty(n, width, dtype=dtype, device=rows.device)
    before = torch.empty(n, outputs, dtype=dtype, device=rows.device) if keep else None
    _enqueue_product("expert_product", "tb200_expert_product", dev, rows.data_ptr(), step, offsets.data_ptr(), code, weight.data_ptr(), *lies,
             _maybe("bias", bias, dtype, (experts, outputs), dev), to, extra, act, n, experts, inputs, outputs, _ROW_CODE[dtype], out.data_ptr(),
             before.data_ptr() if keep else None)
    return (out, before) if keep else out


def expert_activation_grad(dout, before, activation):
    """The gradient of what expert_product kept, from that of act(before): dout [n, width], before [n, width], or [n, 2 width] of a gated activation."""
    dev = _device_of("before", before)
    act = _ACTIVATIONS.get(activation, 0)
    if not act:
        raise ValueError("activation: one of %s" % ", ".join(k for k in _ACTIVATIONS if k))
    if before.dim() != 2 or dout.dim() != 2 or before.shape != (dout.shape[0], dout.shape[1] * (2 if act & 4 else 1)) or dout.dtype != before.dtype or before.dtype not in _ROW_CODE:
        raise ValueError("dout: [n, width] and before: [n, width], gated [n, 2 width], of one type are needed")
    n, width = dout.shape
    dbefore = torch.empty(before.shape, dtype=before.dtype, device=before.device)
    _check(_lib.load().tb200_expert_activation_grad(dout.data_ptr(), _row_step("dout", dout, dev), _packed("before", before, before.dtype, before.shape, dev), act, n, width,
                                                    _ROW_CODE[before.dtype], dbefore.data_ptr(), _raw_stream(dev)), "expert_activation_grad")
    return dbefore


def expert_product_grad(dout, rows, offsets, weight, bias=False, dtype=None, out=None, accumulate=False):
    """The gradients of expert_product's rows, weight and (with bias) bias, from dout, that of `before` (expert_activation_grad's result; without an
    activation out's; the residual's gradient is out's itself).  The gradient of weight is of type dtype (weight's by default, or float32) and lies as weight
    does; accumulate: added to `out` (a gradient that several micro-batches share).  Returns (drows, dweight, dbias): as rows, as weight or `out`, and
    float32 [experts, out] or None.  The order of the sums is fixed: the same inputs give the same bits."""
    dev, step, code, lies = _rows_and_experts(rows, offsets, weight)
    (experts, inputs, outputs), n = weight.shape, rows.shape[0]
    if dout.shape != (n, outputs) or dout.dtype != rows.dtype:
        raise ValueError("dout: shape %s and type %s are needed" % ((n, outputs), rows.dtype))
    dstep = _row_step("dout", dout, dev)
    if accumulate and out is None:
        raise ValueError("accumulate adds to `out`")
    dtype = out.dtype if out is not None and dtype is None else dtype or weight.dtype
    if dtype not in (weight.dtype, _F32):
        raise ValueError("dtype: weight's, or float32")
    inside = lies[2]
    if out is None:
        out = torch.empty((experts, outputs, inputs) if inside else weight.shape, dtype=dtype, device=rows.device)
        out = out.transpose(1, 2) if inside else out
    if out.shape != weight.shape:
        raise ValueError("out: shape %s is needed" % (tuple(weight.shape),))
    to = _packed("out", out.transpose(1, 2) if inside else out, dtype, (experts, outputs, inputs) if inside else (experts, inputs, outputs), dev)
    drows = torch.empty(n, inputs, dtype=rows.dtype, device=rows.device)
    dbias = torch.empty(experts, outputs, dtype=_F32, device=rows.device) if bias else None
    _enqueue_product("expert_product_grad", "tb200_expert_product_grad", dev, dout.data_ptr(), dstep, rows.data_ptr(), step, offsets.data_ptr(), code, weight.data_ptr(), *lies, n, experts, inputs, outputs,
                     _ROW_CODE[rows.dtype], _ROW_CODE[dtype], int(accumulate), drows.data_ptr(), to, dbias.data_ptr() if bias else None)
    return drows, out, dbias
