"""Position-wise layers with gradients: `linear` (matrix product with bias, activation and residual in its epilogue), `gated_linear` (both
projections of a gated feed-forward block, activation and product in one kernel) and the modules built from them.

They stand beside InpaintNet's Conv1d + activation layers (reference model.py:76-87) and the 1x1 head (model.py:45), for rows of any width in
fp32, bf16 or fp16.  `x` is (..., k) with any leading shape, one position per row: InpaintNet's (N, L, C) sequences go in as they are.

    from tracknetv3_amd.feedforward import GatedFeedForward
    block = GatedFeedForward(256, 704).to("cuda", torch.bfloat16)
    y = block(x)                                  # x + W_out (silu(W_gate x) * W_up x)

The pre-activation is kept for the backward pass -- linear's in the tensors' type, gated_linear's in fp32 -- and sums are fp32.  All tensors of a call have
one type: under torch.autocast nothing is cast, a 16-bit input with fp32 weights is refused.  A backward pass with create_graph=True is refused.
A captured backward pass needs that no eager graph from the default stream, of these layers or of any other operation, is alive over the tensors whose
gradients it computes: drop the outputs of earlier steps, or run them on a side stream.  For the tensors that these layers are called with it is refused
otherwise; a tensor that only other operations see is theirs to check.
"""
import math

import torch
from torch import nn
from torch.autograd import forward_ad

from . import ops

ACTIVATIONS = {"none": ops.ACT_NONE, "leaky_relu": ops.ACT_LEAKY_RELU, "sigmoid": ops.ACT_SIGMOID, "relu": ops.ACT_RELU, "silu": ops.ACT_SILU,
               "gelu": ops.ACT_GELU, "gelu_tanh": ops.ACT_GELU_TANH}


def _act(act):
    if isinstance(act, str) and act in ACTIVATIONS:
        return ACTIVATIONS[act]
    if not isinstance(act, int) or not ops.ACT_NONE <= act <= ops.ACT_GELU_TANH:
        raise ValueError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
    return act


# There is no forward-mode derivative.  autograd says so where an input requires a gradient; otherwise the call would return an output without a tangent.
def _no_tangents(what, *tensors):
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: an input carries a forward-mode tangent, and the position-wise layers have no forward-mode derivative")


# (The backward passes call the ops' unchecked form: every tensor is the forward's own or has the shape and type that autograd guarantees, on the
# device that autograd made current.  Their results would be constants to a second derivative: a graph of the backward pass is refused.)
def _no_second_derivative():
    if torch.is_grad_enabled():
        raise RuntimeError("linear / gated_linear have no second derivative: backward with create_graph=True is refused")


# A leaf's gradient accumulator belongs to the stream on which the first graph over the leaf was recorded, by whatever operation, and lives as long as any
# graph over it.  If that is the default stream, a backward pass captured on another would have to make the default stream wait inside the capture, which
# the runtime answers by ending the process: such a call is refused, before anything of the backward pass is launched.
def _capturable(ctx, x):
    if x.is_cuda and torch._C._cuda_isCurrentStreamCapturing():
        _refuse_default_stream(ops._lib.gradient_streams(ctx))


def _refuse_default_stream(streams):
    if 0 in streams:
        raise RuntimeError("linear / gated_linear: this backward pass is being captured while an eager graph of the same tensors, recorded on the "
                           "default stream, is alive: drop its outputs first, or run it on a side stream")


def _linear_grads(ctx, dy):
    _no_second_derivative()
    x, weight, pre = ctx.saved_tensors
    _capturable(ctx, x)
    need = ctx.needs_input_grad
    dx = dw = db = None
    if need[0] or need[1] or need[2]:
        n, k = weight.shape
        dx, dw, db = ops._linear_backward_call(False, dy if dy.is_contiguous() else dy.contiguous(), x, weight, pre, ctx.act, need, x.numel() // k, k, n,
                                               ops._LINEAR_DTYPES[x.dtype])
    return dx, dw, db, (dy if need[3] else None), None


def _gated_linear_grads(ctx, dh):
    _no_second_derivative()
    x, weight, pre = ctx.saved_tensors
    _capturable(ctx, x)
    n2, k = weight.shape
    return ops._linear_backward_call(True, dh if dh.is_contiguous() else dh.contiguous(), x, weight, pre, ctx.act, ctx.needs_input_grad, x.numel() // k, k,
                                     n2 // 2, ops._LINEAR_DTYPES[x.dtype]) + (None,)


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


# (Copies of tensors that are not contiguous are made inside: the Function's edges lead to the caller's own nodes, which _capturable has to see.)
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x, weight = _contiguous(x), _contiguous(weight)
        y, pre = ops.linear(x, weight, _contiguous(bias), _contiguous(residual), act, want_pre=True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = act
        return y

    backward = staticmethod(_linear_grads)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act):
        x, weight = _contiguous(x), _contiguous(weight)
        h, pre = ops.gated_linear(x, weight, _contiguous(bias), act, want_pre=True)
        ctx.save_for_backward(x, weight, pre)
        ctx.act = act
        return h

    backward = staticmethod(_gated_linear_grads)


def linear(x, weight, bias=None, residual=None, act="none"):
    """act(x weight^T + bias) + residual; x (..., k), weight (n, k), bias (n,), residual (..., n), all of one type.  act: a name of ACTIVATIONS
    or an ops.ACT_* constant.  Differentiable once in every tensor, by a backward pass (a forward-mode tangent is refused)."""
    act = _act(act)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act)
    if forward_ad._current_level >= 0:
        _no_tangents("linear", x, weight, bias, residual)
    return ops.linear(_contiguous(x), _contiguous(weight), _contiguous(bias), _contiguous(residual), act)


def gated_linear(x, weight, bias=None, act="silu"):
    """act(g) * u with [g | u] = x weight^T + bias; x (..., k), weight (2 n, k) with the gate's n rows first, bias (2 n,).  Differentiable as
    `linear` is."""
    act = _act(act)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GatedLinear.apply(x, weight, bias, act)
    if forward_ad._current_level >= 0:
        _no_tangents("gated_linear", x, weight, bias)
    return ops.gated_linear(_contiguous(x), _contiguous(weight), _contiguous(bias), act)


class Linear(nn.Linear):
    """nn.Linear (same parameters and state_dict) with an activation and a residual in the product's epilogue."""

    def __init__(self, in_features, out_features, bias=True, act="none", device=None, dtype=None):
        if in_features < 1 or out_features < 1:
            raise ValueError(f"Linear: widths must be positive, got {in_features} -> {out_features}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        _act(act)
        self.act = act

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual, self.act)


class GatedFeedForward(nn.Module):
    """y = W_out (act(W_gate x + b_gate) * (W_up x + b_up)) + b_out [+ x].  weight (2 hidden, dim) holds W_gate's rows, then W_up's."""

    def __init__(self, dim, hidden, act="silu", bias=False, residual=True, device=None, dtype=None):
        super().__init__()
        _act(act)
        if int(dim) < 1 or int(hidden) < 1:
            raise ValueError(f"GatedFeedForward: widths must be positive, got dim {dim}, hidden {hidden}")
        kw = {"device": device, "dtype": dtype}
        self.dim, self.hidden, self.act, self.residual = int(dim), int(hidden), act, bool(residual)
        self.weight = nn.Parameter(torch.empty(2 * self.hidden, self.dim, **kw))
        self.weight_out = nn.Parameter(torch.empty(self.dim, self.hidden, **kw))
        self.bias = nn.Parameter(torch.empty(2 * self.hidden, **kw)) if bias else None
        self.bias_out = nn.Parameter(torch.empty(self.dim, **kw)) if bias else None
        for p, fan_in in ((self.weight, self.dim), (self.bias, self.dim), (self.weight_out, self.hidden), (self.bias_out, self.hidden)):
            if p is not None:
                nn.init.uniform_(p, -1 / math.sqrt(fan_in), 1 / math.sqrt(fan_in))      # nn.Linear's range

    def forward(self, x):
        if x.dim() < 1 or x.shape[-1] != self.dim:
            raise ValueError(f"GatedFeedForward expects (..., {self.dim}), got {tuple(x.shape)}")
        h = gated_linear(x, self.weight, self.bias, self.act)
        return linear(h, self.weight_out, self.bias_out, x if self.residual else None)
