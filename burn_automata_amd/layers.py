"""The dense layers of a trained update rule on the MI355X (HIP) path: layer norm and linear layer,
forward and adjoint, in float32, bfloat16 and float16.

The reference's kernel crate has no counterpart (its update MLP is ``NpaModel.forward_from_features_with_eps``):
these are the layers a program needs to train an update rule, or to run one of another depth or width, next
to ``kernels.perceive_with_options`` and ``kernels.perceive_adjoint_with_options``.

Matrices are CUDA tensors of two or more dims whose last one runs through memory; leading dims are rows, which
may lie apart at one distance (a column slice of a wider tensor is taken in place, anything else is copied).
Results are freshly allocated, except where an argument says that gradients are added to it. Without ``ctx``, a
call runs on torch's current stream of the tensors' device, on a context of that stream and thread. A ``ctx`` on
another stream is refused, as results are allocated and copies made on the current one.

No autograd graph is recorded: results do not require gradients whatever the inputs do, and ``backward`` does not pass
through these calls. Their gradients are the ``*_adjoint`` functions.
"""
from __future__ import annotations

import ctypes as C
import threading
from dataclasses import dataclass
from enum import IntEnum

import torch

from . import _abi
from ._lib import lib
from .runtime import Context


class Activation(IntEnum):
    """NPA_ACT_*: gelu is the tanh form."""

    identity = _abi.ACT_IDENTITY
    relu = _abi.ACT_RELU
    gelu = _abi.ACT_GELU
    silu = _abi.ACT_SILU


@dataclass
class LayerNormOutput:
    """The normed rows, and each row's mean and 1 / sqrt(variance + eps) in float32."""

    out: object
    mean: object
    rstd: object


@dataclass
class LayerNormAdjoint:
    """The gradients of x, gamma and beta (None where there is no gamma)."""

    x: object
    gamma: object
    beta: object


@dataclass
class LinearOutput:
    """The layer's rows, and what its activation was applied to (None unless it was asked for)."""

    out: object
    preactivation: object


@dataclass
class LinearAdjoint:
    """The gradients of x, weight and bias (None where one was not asked for)."""

    x: object
    weight: object
    bias: object


class _Own(dict):
    """One thread's contexts by (device, stream). They outlive the thread, as a graph may have captured their
    workspaces, and serve the next thread that works on their stream."""

    free: dict = {}

    def take(self, device: int, stream: int) -> Context:
        try:
            ctx = _Own.free[device, stream].pop()
        except (KeyError, IndexError):
            ctx = Context(device, stream)
        self[device, stream] = ctx
        return ctx

    def __del__(self):
        for key, ctx in self.items():
            self.free.setdefault(key, []).append(ctx)


class _Contexts(threading.local):
    """The contexts of this thread: a context serves one thread at a time."""

    def __init__(self):
        self.of = _Own()


_CONTEXTS = _Contexts()
_FUNCTIONS: dict = {}
_TYPES = {torch.float32: _abi.TYPE_F32, torch.bfloat16: _abi.TYPE_BF16, torch.float16: _abi.TYPE_F16}
_ACTIVATIONS = {a.name: a.value for a in Activation} | {a: a.value for a in Activation}

# The current stream's handle without a Stream object around it (1 us of a call of 8).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def current_context(device: int = 0) -> Context:
    """The context that calls on ``device`` use without one of their own: of torch's current stream and this
    thread, so that neither two streams nor two threads share workspaces. It is kept until the process ends."""
    stream = _raw_stream(device)
    ctx = _CONTEXTS.of.get((device, stream))
    return _CONTEXTS.of.take(device, stream) if ctx is None else ctx


def _context(x, ctx):
    """The caller's context, or the current one of the tensor's device."""
    device = x.get_device()
    if ctx is not None:
        if device != ctx.device:
            raise _abi.InvalidArgument(f"invalid argument: a tensor on {x.device} and a context on device "
                                       f"{ctx.device}")
        stream = _raw_stream(device)
        if stream != ctx.stream:
            raise _abi.InvalidArgument(f"invalid argument: a context on stream {ctx.stream:#x} and a current stream "
                                       f"{stream:#x}")
        return ctx
    return current_context(device)


def _matrix(t, what: str, cols=None, rows=None, like=None):
    """(tensor, rows, cols, row distance) of a matrix argument."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise _abi.InvalidArgument(f"invalid argument: {what} is not a CUDA tensor")
    if like is None:
        if t.dtype not in _TYPES:
            raise _abi.InvalidArgument(f"invalid argument: {what} is {t.dtype}; float32, bfloat16 and float16 are "
                                       f"served")
    elif t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise _abi.InvalidArgument(f"invalid argument: {what} is {t.dtype} on {t.device}, expected {like.dtype} "
                                   f"on {like.device}")
    shape = t.shape
    if len(shape) == 2:
        r, c = shape
    elif len(shape) > 2:
        r, c = shape[:-1].numel(), shape[-1]
    else:
        raise _abi.InvalidArgument(f"invalid argument: {what} has {t.dim()} dims; rows and columns are needed")
    if (cols is not None and c != cols) or (rows is not None and r != rows):
        raise _abi.OutputShape(f"{what} of {r} rows by {c} does not match expected "
                               f"{r if rows is None else rows} by {c if cols is None else cols}")
    if t.is_contiguous():
        return t, r, c, c
    if len(shape) == 2 and t.stride(1) == 1 and t.stride(0) >= c:
        return t, r, c, t.stride(0)
    return t.contiguous(), r, c, c


def _vector(t, what: str, length: int, like):
    """A parameter: of the layer's type or float32, contiguous."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.get_device() != like.get_device() or \
            (t.dtype is not like.dtype and t.dtype is not torch.float32):
        raise _abi.InvalidArgument(f"invalid argument: {what} has to be float32 or {like.dtype} on {like.device}")
    if t.numel() != length:
        raise _abi.OutputShape(f"{what} of {t.numel()} elements does not match expected {length}")
    return t if t.is_contiguous() else t.contiguous()


def _call(name: str, ctx, cfg, *arrays):
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(lib(), name)
    code = fn(ctx.handle, C.byref(cfg), *arrays)
    if code:
        ctx.check(code)


def _address(t):
    return None if t is None else t.data_ptr()


def _gradient(t, what: str, shape, like):
    """A gradient that is added to: used in place."""
    if tuple(t.shape) != tuple(shape):
        raise _abi.OutputShape(f"{what} of shape {tuple(t.shape)} does not match expected {tuple(shape)}")
    if t.device != like.device or t.dtype not in (like.dtype, torch.float32) or not t.is_contiguous():
        raise _abi.InvalidArgument(f"invalid argument: {what} has to be contiguous, float32 or {like.dtype} on "
                                   f"{like.device}")
    return t


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5, ctx=None) -> LayerNormOutput:
    """(x - mean) / sqrt(variance + eps) * gamma + beta over the last axis (npa_layer_norm)."""
    x, rows, width, stride = _matrix(x, "x")
    gamma, beta = _vector(gamma, "gamma", width, x), _vector(beta, "beta", width, x)
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        raise _abi.InvalidArgument(f"invalid argument: gamma is {gamma.dtype} and beta {beta.dtype}")
    ctx = _context(x, ctx)
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    param = gamma if gamma is not None else beta
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaNormCfg(rows, stride, 0, 0, 0, width, kind, kind if param is None else _TYPES[param.dtype], 0,
                          float(eps))
    _call("npa_layer_norm", ctx, cfg, x.data_ptr(), _address(gamma), _address(beta), out.data_ptr(), mean.data_ptr(),
          rstd.data_ptr())
    return LayerNormOutput(out, mean, rstd)


def layer_norm_adjoint(out_adjoint, x, mean, rstd, gamma=None, gamma_adjoint=None, beta_adjoint=None,
                       ctx=None) -> LayerNormAdjoint:
    """The reverse mode of layer_norm for the statistics it returned (npa_layer_norm_adjoint). With gamma its
    gradient and beta's are computed, in gamma's type; ``gamma_adjoint`` and ``beta_adjoint``, given together,
    are added to instead."""
    x, rows, width, stride = _matrix(x, "x")
    dy, _, _, dy_stride = _matrix(out_adjoint, "out_adjoint", width, rows, x)
    gamma = _vector(gamma, "gamma", width, x)
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if t.numel() != rows:
            raise _abi.OutputShape(f"{what} of {t.numel()} elements does not match expected {rows}")
        if t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
            raise _abi.InvalidArgument(f"invalid argument: {what} has to be contiguous float32 on {x.device}")
    added = gamma_adjoint is not None
    if added != (beta_adjoint is not None):
        raise _abi.InvalidArgument("invalid argument: gamma_adjoint and beta_adjoint are given together")
    if added:
        _gradient(gamma_adjoint, "gamma_adjoint", (width,), x)
        _gradient(beta_adjoint, "beta_adjoint", (width,), x)
        if gamma_adjoint.dtype != beta_adjoint.dtype or (gamma is not None and gamma.dtype != gamma_adjoint.dtype):
            raise _abi.InvalidArgument("invalid argument: gamma, gamma_adjoint and beta_adjoint differ in type")
    elif gamma is not None:
        gamma_adjoint, beta_adjoint = torch.empty_like(gamma), torch.empty_like(gamma)
    ctx = _context(x, ctx)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaNormCfg(rows, stride, 0, dy_stride, 0, width, kind,
                          kind if gamma_adjoint is None else _TYPES[gamma_adjoint.dtype], int(added), 0.0)
    _call("npa_layer_norm_adjoint", ctx, cfg, x.data_ptr(), _address(gamma), mean.data_ptr(), rstd.data_ptr(),
          dy.data_ptr(), dx.data_ptr(), _address(gamma_adjoint), _address(beta_adjoint))
    return LayerNormAdjoint(dx, gamma_adjoint, beta_adjoint)


def _activation(a) -> int:
    code = _ACTIVATIONS.get(a)
    if code is None:
        raise _abi.InvalidArgument(f"invalid argument: unknown activation {a!r}")
    return code


def linear(x, weight, bias=None, activation=Activation.identity, residual=None, keep_preactivation: bool = False,
           ctx=None) -> LinearOutput:
    """activation(x weight^T + bias) + residual (npa_linear): x [rows, in], weight [out, in]. The preactivation
    is kept for linear_adjoint where it is asked for."""
    x, rows, inputs, stride = _matrix(x, "x")
    w, outputs, _, w_stride = _matrix(weight, "weight", inputs, None, x)
    bias = _vector(bias, "bias", outputs, x)
    residual, _, _, r_stride = (None, 0, 0, 0) if residual is None else \
        _matrix(residual, "residual", outputs, rows, x)
    ctx = _context(x, ctx)
    out = x.new_empty(x.shape[:-1] + (outputs,))
    z = torch.empty_like(out) if keep_preactivation else None
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaLinearCfg(rows, stride, w_stride, r_stride, 0, 0, 0, 0, inputs, outputs, kind,
                            _activation(activation), kind if bias is None else _TYPES[bias.dtype], kind, 0)
    _call("npa_linear", ctx, cfg, x.data_ptr(), w.data_ptr(), _address(bias), _address(residual), out.data_ptr(),
          _address(z))
    return LinearOutput(out, z)


def linear_adjoint(out_adjoint, x, weight, preactivation=None, activation=Activation.identity, bias: bool = True,
                   weight_adjoint=None, bias_adjoint=None, inputs: bool = True, parameters: bool = True,
                   ctx=None) -> LinearAdjoint:
    """The reverse mode of linear (npa_linear_adjoint); a residual's gradient is out_adjoint itself.
    ``preactivation`` is the one that linear kept (none for the identity). ``inputs``, ``parameters`` and
    ``bias`` say which gradients are wanted. Gradients of parameters are of the weight's type;
    ``weight_adjoint`` (and ``bias_adjoint``, where ``bias``), of that type or float32, are added to instead."""
    x, rows, k, stride = _matrix(x, "x")
    w, n, _, w_stride = _matrix(weight, "weight", k, None, x)
    dy, _, _, dy_stride = _matrix(out_adjoint, "out_adjoint", n, rows, x)
    z, _, _, z_stride = (None, 0, 0, 0) if preactivation is None else \
        _matrix(preactivation, "preactivation", n, rows, x)
    bias = bias and parameters
    added = weight_adjoint is not None
    if (bias_adjoint is not None) != (added and bias) or (added and not parameters):
        raise _abi.InvalidArgument("invalid argument: weight_adjoint and, with a bias, bias_adjoint are given together")
    if added:
        _gradient(weight_adjoint, "weight_adjoint", (n, k), x)
        if bias:
            _gradient(bias_adjoint, "bias_adjoint", (n,), x)
            if bias_adjoint.dtype != weight_adjoint.dtype:
                raise _abi.InvalidArgument("invalid argument: weight_adjoint and bias_adjoint differ in type")
    elif parameters:
        weight_adjoint = x.new_empty((n, k))
        if bias:
            bias_adjoint = x.new_empty(n)
    ctx = _context(x, ctx)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if inputs else None
    kind = _TYPES[x.dtype]
    cfg = _abi.NpaLinearCfg(rows, stride, w_stride, 0, 0, z_stride, dy_stride, 0, k, n, kind, _activation(activation),
                            kind, kind if weight_adjoint is None else _TYPES[weight_adjoint.dtype], int(added))
    _call("npa_linear_adjoint", ctx, cfg, x.data_ptr(), w.data_ptr(), _address(z), dy.data_ptr(), _address(dx),
          _address(weight_adjoint), _address(bias_adjoint))
    return LinearAdjoint(dx, weight_adjoint, bias_adjoint)
