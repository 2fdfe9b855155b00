"""The layers of a mixture of update rules on the MI355X (HIP) path, forward and adjoint, in float32, bfloat16 and
float16: rows that each use a few of many experts' weights.

The reference has no counterpart. ``route`` chooses each row's experts and their weights, and a ``Plan`` sorts the
choices by expert; ``linear`` is each expert's linear layer over its slots of the plan; ``combine`` adds a row's slots
up again:

    r = route(logits, top_k=2)
    h = linear(x, w1, r.plan, b1, "gelu", gather=True)             # [slots, hidden], rows taken through the plan
    y = combine(linear(h.out, w2, r.plan, b2).out, r.plan, r.weights, residual=x)

Tensors, contexts and streams are those of ``layers``: CUDA tensors whose last axis runs through memory, results
freshly allocated except where an argument is added to, the current stream's context unless one is given. No autograd
graph is recorded; gradients are the ``*_adjoint`` functions'. Nothing here waits for the GPU, so calls can be captured.
"""
from __future__ import annotations

from dataclasses import dataclass
from enum import IntEnum

import torch

from . import _abi
from ._lib import lib
from .layers import (_TYPES, _activation, _address, _call, _context, _gradient, _matrix, _vector, Activation,
                     LinearAdjoint, LinearOutput)


class Scores(IntEnum):
    """NPA_SCORE_*: of a row's logits."""

    softmax = _abi.SCORE_SOFTMAX
    sigmoid = _abi.SCORE_SIGMOID


_SCORES = {s.name: s.value for s in Scores} | {s: s.value for s in Scores}
MOST_EXPERTS, MOST_CHOICES, MOST_SLOTS = 1024, 32, 1 << 30


@dataclass(frozen=True)
class Plan:
    """The entries (row r's j-th choice is entry r * top_k + j) sorted by expert, int32: expert e's slots are
    offsets[e] .. offsets[e + 1] - 1 (``offsets`` [experts + 1]), ``order`` [slots] is the entry of each slot and
    ``slots`` [rows, top_k] the slot of each entry. Entries without an expert have the slots from offsets[-1] on."""

    offsets: object
    order: object
    slots: object

    def __post_init__(self):
        for t, what in ((self.offsets, "offsets"), (self.order, "order"), (self.slots, "slots")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not torch.int32 or not t.is_contiguous() \
                    or t.get_device() != self.offsets.get_device():
                raise _abi.InvalidArgument(f"invalid argument: a plan's {what} has to be contiguous int32 on one GPU")
        if self.offsets.dim() != 1 or self.slots.dim() != 2 or self.order.dim() != 1:
            raise _abi.InvalidArgument("invalid argument: a plan's offsets and order have one dim, its slots two")
        if self.offsets.numel() < 2 or self.order.numel() != self.slots.numel():
            raise _abi.OutputShape(f"a plan of {self.offsets.numel()} offsets, order of {self.order.numel()} and slots of "
                                   f"shape {tuple(self.slots.shape)}")

    @classmethod
    def _of(cls, offsets, order, slots):
        """One of arrays that were made here: without its checks (1 us of a call of 18)."""
        made = cls.__new__(cls)
        made.__dict__.update(offsets=offsets, order=order, slots=slots)
        return made

    @property
    def experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def rows(self) -> int:
        return self.slots.shape[0]

    @property
    def top_k(self) -> int:
        return self.slots.shape[1]


@dataclass
class RouteOutput:
    """Each row's experts [.., top_k] (int32, -1: none) and their weights (float32), and the plan of all of them."""

    experts: object
    weights: object
    plan: Plan


@dataclass
class CombineAdjoint:
    """The gradients of y [slots, width] and of the weights [rows, top_k] (None where there are none)."""

    y: object
    weights: object


def _choices(rows: int, top_k: int, experts: int):
    if not 1 <= experts <= MOST_EXPERTS:
        raise _abi.InvalidArgument(f"invalid argument: 1 to {MOST_EXPERTS} experts are served, got {experts}")
    if not 1 <= top_k <= min(experts, MOST_CHOICES):
        raise _abi.InvalidArgument(f"invalid argument: top_k is 1 to {MOST_CHOICES} and at most the experts' number "
                                   f"{experts}, got {top_k}")
    if rows * top_k > MOST_SLOTS:
        raise _abi.InvalidArgument(f"invalid argument: {rows} rows of {top_k} choices; at most 2^30 in all")


def _scores(scores) -> int:
    code = _SCORES.get(scores)
    if code is None:
        raise _abi.InvalidArgument(f"invalid argument: unknown scores {scores!r}")
    return code


def _words(t, what: str, dtype, rows: int, top_k: int, like):
    """An int32 or float32 array [.., top_k] (or flat) of each choice."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != like.get_device():
        raise _abi.InvalidArgument(f"invalid argument: {what} has to be {dtype} on {like.device}")
    if t.numel() != rows * top_k or (t.dim() > 1 and t.shape[-1] != top_k):
        raise _abi.OutputShape(f"{what} of shape {tuple(t.shape)} does not match expected {rows} rows of {top_k}")
    return t if t.is_contiguous() else t.contiguous()


def _plan(plan, like) -> Plan:
    if not isinstance(plan, Plan):
        raise _abi.InvalidArgument(f"invalid argument: a Plan is needed, got {type(plan).__name__}")
    if plan.offsets.get_device() != like.get_device():
        raise _abi.InvalidArgument(f"invalid argument: a plan on {plan.offsets.device}, expected {like.device}")
    return plan


def _empty_plan(rows: int, top_k: int, experts: int, like):
    offsets = like.new_empty(experts + 1, dtype=torch.int32)
    return offsets, offsets.new_empty(rows * top_k), offsets.new_empty((rows, top_k))


def route(logits, top_k: int, scores=Scores.softmax, bias=None, groups: int = 1, top_groups: int = 1,
          renormalise: bool = True, scale: float = 1.0, ctx=None) -> RouteOutput:
    """The ``top_k`` best experts of each row of ``logits`` [.., experts], their weights and the plan
    (npa_expert_route). Experts are ordered by score + ``bias`` (without a bias by logit), equal ones by index, and
    only those of the ``top_groups`` best groups are chosen (a group's value: the sum of its two largest). A logit or
    bias of -inf closes an expert; choices that no open expert is left for are -1, of weight 0. The weights are the
    scores, without the bias, over their sum (+ 1e-20) if ``renormalise``, times ``scale``."""
    logits, rows, experts, stride = _matrix(logits, "logits")
    _choices(rows, top_k, experts)
    bias = _vector(bias, "bias", experts, logits)
    ctx = _context(logits, ctx)
    shape = logits.shape[:-1] + (top_k,)
    chosen = logits.new_empty(shape, dtype=torch.int32)
    weights = logits.new_empty(shape, dtype=torch.float32)
    offsets, order, slots = _empty_plan(rows, top_k, experts, logits)
    kind = _TYPES[logits.dtype]
    cfg = _abi.NpaRouteCfg(rows, stride, 0, experts, top_k, groups, top_groups, kind,
                           kind if bias is None else _TYPES[bias.dtype], _scores(scores), int(bool(renormalise)),
                           float(scale))
    _call("npa_expert_route", ctx, cfg, logits.data_ptr(), _address(bias), chosen.data_ptr(), weights.data_ptr(),
          offsets.data_ptr(), order.data_ptr(), slots.data_ptr())
    return RouteOutput(chosen, weights, Plan._of(offsets, order, slots))


def route_adjoint(weights_adjoint, logits, experts, scores=Scores.softmax, renormalise: bool = True,
                  scale: float = 1.0, ctx=None):
    """The gradient of route's logits from that of its weights, for the experts it chose
    (npa_expert_route_adjoint); the choice itself has none."""
    logits, rows, count, stride = _matrix(logits, "logits")
    top_k = experts.shape[-1] if isinstance(experts, torch.Tensor) and experts.dim() else 0
    _choices(rows, top_k, count)
    experts = _words(experts, "experts", torch.int32, rows, top_k, logits)
    weights_adjoint = _words(weights_adjoint, "weights_adjoint", torch.float32, rows, top_k, logits)
    ctx = _context(logits, ctx)
    out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    kind = _TYPES[logits.dtype]
    cfg = _abi.NpaRouteCfg(rows, stride, 0, count, top_k, 1, 1, kind, kind, _scores(scores), int(bool(renormalise)),
                           float(scale))
    _call("npa_expert_route_adjoint", ctx, cfg, logits.data_ptr(), experts.data_ptr(), weights_adjoint.data_ptr(),
          out.data_ptr())
    return out


def plan(chosen, experts: int, ctx=None) -> Plan:
    """The plan of choices [.., top_k] (int32) that a program has made itself (npa_expert_plan). An index that is none
    of 0 .. experts - 1 is an entry without an expert."""
    if not isinstance(chosen, torch.Tensor) or not chosen.is_cuda or chosen.dtype is not torch.int32 or not chosen.dim():
        raise _abi.InvalidArgument("invalid argument: chosen has to be an int32 CUDA tensor [.., top_k]")
    top_k = chosen.shape[-1]
    rows = chosen.shape[:-1].numel()
    _choices(rows, top_k, experts)
    chosen = chosen.contiguous()
    ctx = _context(chosen, ctx)
    offsets, order, slots = _empty_plan(rows, top_k, experts, chosen)
    ctx.check(lib().npa_expert_plan(ctx.handle, rows, top_k, experts, chosen.data_ptr(), offsets.data_ptr(),
                                    order.data_ptr(), slots.data_ptr()))
    return Plan._of(offsets, order, slots)


def _weight(weight, plan: Plan, inputs: int, like):
    """(tensor, outputs, row distance) of the experts' weights [experts, outputs, inputs]."""
    if not isinstance(weight, torch.Tensor) or weight.dtype is not like.dtype or weight.get_device() != like.get_device():
        raise _abi.InvalidArgument(f"invalid argument: weight has to be {like.dtype} on {like.device}")
    if weight.dim() != 3 or weight.shape[0] != plan.experts or weight.shape[2] != inputs:
        raise _abi.OutputShape(f"weight of shape {tuple(weight.shape)} does not match expected ({plan.experts}, outputs, "
                               f"{inputs})")
    outputs = weight.shape[1]
    if not weight.is_contiguous():
        e, r, c = weight.stride()
        if c == 1 and r >= inputs and e == outputs * r:
            return weight, outputs, r
        weight = weight.contiguous()
    return weight, outputs, inputs


def linear(x, weight, plan, bias=None, activation=Activation.identity, gather: bool = False,
           keep_preactivation: bool = False, ctx=None) -> LinearOutput:
    """activation(x weight[e]^T + bias[e]) for each slot of each expert e (npa_expert_linear): ``weight`` [experts, out,
    in], ``bias`` [experts, out], ``x`` [slots, in], or [.., in] rows, each slot's taken through the plan, where
    ``gather``. Results are [slots, out]; slots without an expert are rows of zeros."""
    x, rows, inputs, stride = _matrix(x, "x")
    plan = _plan(plan, x)
    slots = plan.order.shape[0]
    if rows != (plan.rows if gather else slots):
        raise _abi.OutputShape(f"x of {rows} rows does not match the plan's {plan.rows} rows and {slots} slots")
    w, outputs, w_stride = _weight(weight, plan, inputs, x)
    if isinstance(bias, torch.Tensor) and bias.dim() > 1 and bias.shape[-1] != outputs:
        raise _abi.OutputShape(f"bias of shape {tuple(bias.shape)} does not match expected ({plan.experts}, {outputs})")
    bias = _vector(bias, "bias", plan.experts * outputs, x)
    ctx = _context(x, ctx)
    out = x.new_empty((slots, outputs))
    z = torch.empty_like(out) if keep_preactivation else None
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaExpertLinearCfg(plan.rows, stride, w_stride, 0, 0, 0, 0, plan.experts, plan.top_k, inputs, outputs, kind,
                                  _activation(activation), kind if bias is None else _TYPES[bias.dtype], kind, 0,
                                  int(bool(gather)))
    _call("npa_expert_linear", ctx, cfg, x.data_ptr(), w.data_ptr(), _address(bias), plan.offsets.data_ptr(),
          plan.order.data_ptr(), out.data_ptr(), _address(z))
    return LinearOutput(out, z)


def linear_adjoint(out_adjoint, x, weight, plan, preactivation=None, activation=Activation.identity,
                   gather: bool = False, bias: bool = True, weight_adjoint=None, bias_adjoint=None, inputs: bool = True,
                   parameters: bool = True, ctx=None) -> LinearAdjoint:
    """The reverse mode of linear (npa_expert_linear_adjoint). ``preactivation`` is the one that linear kept (none for the
    identity). ``inputs``, ``parameters`` and ``bias`` say which gradients are wanted; with ``gather`` x's is summed over
    each row's slots. Gradients of parameters are of the weight's type and zeros for an expert without slots;
    ``weight_adjoint`` (and ``bias_adjoint``, where ``bias``), of that type or float32, are added to instead."""
    x, rows, k, stride = _matrix(x, "x")
    plan = _plan(plan, x)
    slots = plan.order.shape[0]
    if rows != (plan.rows if gather else slots):
        raise _abi.OutputShape(f"x of {rows} rows does not match the plan's {plan.rows} rows and {slots} slots")
    w, n, w_stride = _weight(weight, plan, k, x)
    dy, _, _, dy_stride = _matrix(out_adjoint, "out_adjoint", n, slots, x)
    z, _, _, z_stride = (None, 0, 0, 0) if preactivation is None else \
        _matrix(preactivation, "preactivation", n, slots, x)
    bias = bias and parameters
    added = weight_adjoint is not None
    if (bias_adjoint is not None) != (added and bias) or (added and not parameters):
        raise _abi.InvalidArgument("invalid argument: weight_adjoint and, with a bias, bias_adjoint are given together")
    if added:
        _gradient(weight_adjoint, "weight_adjoint", (plan.experts, n, k), x)
        if bias:
            _gradient(bias_adjoint, "bias_adjoint", (plan.experts, n), x)
            if bias_adjoint.dtype != weight_adjoint.dtype:
                raise _abi.InvalidArgument("invalid argument: weight_adjoint and bias_adjoint differ in type")
    elif parameters:
        weight_adjoint = x.new_empty((plan.experts, n, k))
        if bias:
            bias_adjoint = x.new_empty((plan.experts, n))
    ctx = _context(x, ctx)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if inputs else None
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaExpertLinearCfg(plan.rows, stride, w_stride, 0, z_stride, dy_stride, 0, plan.experts, plan.top_k, k, n,
                                  kind, _activation(activation), kind,
                                  kind if weight_adjoint is None else _TYPES[weight_adjoint.dtype], int(added),
                                  int(bool(gather)))
    _call("npa_expert_linear_adjoint", ctx, cfg, x.data_ptr(), w.data_ptr(), _address(z), plan.offsets.data_ptr(),
          plan.order.data_ptr(), plan.slots.data_ptr(), dy.data_ptr(), _address(dx), _address(weight_adjoint),
          _address(bias_adjoint))
    return LinearAdjoint(dx, weight_adjoint, bias_adjoint)


def combine(y, plan, weights=None, residual=None, ctx=None):
    """residual + the sum over a row's choices j of weights[row, j] * y[slot of j] (npa_expert_combine): ``y`` [slots,
    width], ``weights`` [.., top_k] float32 (none: 1), ``residual`` [.., width], whose shape the result has (else
    [rows, width])."""
    y, slots, width, stride = _matrix(y, "y")
    plan = _plan(plan, y)
    if slots != plan.order.shape[0]:
        raise _abi.OutputShape(f"y of {slots} rows does not match the plan's {plan.order.shape[0]} slots")
    weights = None if weights is None else _words(weights, "weights", torch.float32, plan.rows, plan.top_k, y)
    residual, _, _, r_stride = (None, 0, 0, 0) if residual is None else \
        _matrix(residual, "residual", width, plan.rows, y)
    ctx = _context(y, ctx)
    out = y.new_empty((plan.rows, width) if residual is None else residual.shape)
    cfg = _abi.NpaCombineCfg(plan.rows, stride, r_stride, 0, 0, 0, plan.experts, plan.top_k, width, _TYPES[y.dtype])
    _call("npa_expert_combine", ctx, cfg, y.data_ptr(), plan.offsets.data_ptr(), plan.slots.data_ptr(),
          _address(weights), _address(residual), out.data_ptr())
    return out


def combine_adjoint(out_adjoint, y, plan, weights=None, ctx=None) -> CombineAdjoint:
    """The reverse mode of combine (npa_expert_combine_adjoint); a residual's gradient is out_adjoint itself. Slots
    without an expert have gradients of zero."""
    y, slots, width, stride = _matrix(y, "y")
    plan = _plan(plan, y)
    if slots != plan.order.shape[0]:
        raise _abi.OutputShape(f"y of {slots} rows does not match the plan's {plan.order.shape[0]} slots")
    dout, _, _, d_stride = _matrix(out_adjoint, "out_adjoint", width, plan.rows, y)
    weights = None if weights is None else _words(weights, "weights", torch.float32, plan.rows, plan.top_k, y)
    weights_adjoint = None if weights is None else torch.empty_like(weights)
    ctx = _context(y, ctx)
    dy = torch.empty_like(y, memory_format=torch.contiguous_format)
    cfg = _abi.NpaCombineCfg(plan.rows, stride, 0, 0, d_stride, 0, plan.experts, plan.top_k, width, _TYPES[y.dtype])
    _call("npa_expert_combine_adjoint", ctx, cfg, y.data_ptr(), plan.offsets.data_ptr(), plan.slots.data_ptr(),
          _address(weights), dout.data_ptr(), dy.data_ptr(), _address(weights_adjoint))
    return CombineAdjoint(dy, weights_adjoint)
