"""What stands between the aggregations of a deep model: the norm of its rows and dense layers, each with what follows it in the same pass, and with
8 bits a value of their inputs kept for the backward pass where memory is what limits a batch.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from . import _lib as L
from . import ops


def _norm_by_operators(x, weight, bias, eps, relu):
    """The same in torch's operators, for who has to see those; what the backward pass needs is kept in full."""
    if torch.is_autocast_enabled():
        x, weight, bias = (None if t is None else t.float() for t in (x, weight, bias))
    if x.dtype not in ops._FEAT or x.dim() < 1 or not (torch.jit.is_tracing() or 1 <= x.size(-1) <= L.NORM_MAX_DIM):
        raise RuntimeError("x must have dtype in %s and rows of 1 to %d columns" % ([str(t) for t in ops._FEAT], L.NORM_MAX_DIM))
    if any(t is not None and (t.dim() != 1 or t.dtype != x.dtype or not (torch.jit.is_tracing() or t.size(0) == x.size(-1))) for t in (weight, bias)):
        raise RuntimeError("weight and bias must hold a value of x's type for each column")
    if not eps >= 0.0:
        raise RuntimeError("eps (%g) must not be negative" % eps)
    with torch.autocast("cuda", enabled=False):
        h = x.double()
        h = h - h.mean(-1, keepdim=True)
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
        y = h if weight is None else h * weight.double()
        y = y if bias is None else y + bias.double()
        return (torch.where(y <= 0, 0.0, y) if relu else y).to(x.dtype)


def layer_norm(x, weight=None, bias=None, eps=1e-5, relu=False, keep8=False):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (at most 2048 columns), ``relu``: ``max(.., 0)`` of it, with gradients
    for all three.  ``x``: float32 or bfloat16 on the GPU, any leading dimensions; rows that lie apart are taken as they are, other orders copied.
    ``weight``, ``bias``: of x's type, or ``None`` for ones and zeros.  Mean, variance and the normed values are formed in 64 bits, so that rows far from
    zero keep what they differ in.
    For the backward pass ``x`` is kept with 12 bytes a row, and with ``relu`` a bit a value.  ``keep8=True``: in ``x``'s place the normed values, 8 bits each: 32
    neighbouring columns share a step, ``2**(floor(log2(largest magnitude)) - 6)``, and the nearest of -127 .. 127 steps is held; gradients are those of
    the values so held (32 columns with one that is not finite are held as not a number).
    Under autocast in float32, as torch's.  No gradients of gradients.  Under tracing, forward-mode differentiation, transforms of
    ``torch.func`` and modes that follow the operators: by torch's operators, with nothing kept in 8 bits."""
    if not all(t is None or (isinstance(t, torch.Tensor) and t.is_cuda) for t in (weight, bias)) or not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise RuntimeError("x, weight and bias must be CUDA tensors")
    if ops._unseen(x, weight, bias):
        return _norm_by_operators(x, weight, bias, eps, relu)
    return L.host().layer_norm(x, weight, bias, eps, bool(relu), bool(keep8), L.NORM_MAX_DIM)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension whose ``forward`` is ``layer_norm``; a state of either is one of the other's.  ``relu``: the activation
    behind it goes with it (``forward(x, relu)``: in its place, if given).  ``keep8``: 8 bits a value are kept for the backward pass."""

    def __init__(self, features, eps=1e-5, elementwise_affine=True, bias=True, relu=False, keep8=False):
        super().__init__(features, eps=eps, elementwise_affine=elementwise_affine, bias=bias)
        if len(self.normalized_shape) != 1:
            raise ValueError("the norm is over one dimension, not %s" % (self.normalized_shape,))
        self.relu, self.keep8 = bool(relu), bool(keep8)

    def forward(self, x, relu=None):
        if isinstance(x, torch.Tensor) and x.dim() > 0 and x.size(-1) != self.normalized_shape[0]:
            raise RuntimeError("x has rows of %d columns, not of %d" % (x.size(-1), self.normalized_shape[0]))
        return layer_norm(x, self.weight, self.bias, self.eps, self.relu if relu is None else relu, self.keep8)

    def extra_repr(self):
        return super().extra_repr() + (", relu=True" if self.relu else "") + (", keep8=True" if self.keep8 else "")


def _linear_by_operators(x, weight, bias, activation, residual):
    """The same in torch's operators, for who has to see those; what the backward pass needs is kept in full."""
    if torch.is_autocast_enabled():
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias, residual = (None if t is None else t.to(to) for t in (x, weight, bias, residual))
    sized = not torch.jit.is_tracing()  # (a trace is of any sizes, and its operators have their own checks)
    if x.dim() < 1 or weight.dim() != 2 or (sized and not (x.size(-1) == weight.size(1) and all(1 <= d <= L.LINEAR_MAX_DIM for d in weight.shape))):
        raise RuntimeError("x %s and weight %s must be [.., d] and [out, d] with 1 <= d, out <= %d" % (tuple(x.shape), tuple(weight.shape), L.LINEAR_MAX_DIM))
    if x.dtype not in ops._FEAT or any(t is not None and t.dtype != x.dtype for t in (weight, bias, residual)):
        raise RuntimeError("x, weight, bias and residual must all be of one type in %s" % [str(t) for t in ops._FEAT])
    if bias is not None and (bias.dim() != 1 or (sized and bias.size(0) != weight.size(0))):
        raise RuntimeError("bias must hold a value for each row of weight")
    if residual is not None and sized and tuple(residual.shape) != (*x.shape[:-1], weight.size(0)):
        raise RuntimeError("residual must be of the output's sizes")
    with torch.autocast("cuda", enabled=False):
        z = F.linear(x.float(), weight.float(), None if bias is None else bias.float())
        if activation is not None:
            z = {"relu": torch.relu, "gelu": F.gelu, "silu": F.silu}[activation](z)
        return (z if residual is None else z + residual.float()).to(x.dtype)


def linear(x, weight, bias=None, activation=None, residual=None, keep8=False):
    """``activation(x weight^T + bias) + residual`` for ``x`` [.., d] and ``weight`` [out, d], with gradients for all four.  Float32 or bfloat16 on the GPU, all of one
    type, ``d`` and ``out`` up to 4096; rows that lie apart are taken as they are (bfloat16: where they start on four bytes), other orders copied.
    ``activation``: ``None``, ``"relu"``, ``"gelu"`` (by the normal distribution function) or ``"silu"``; ``residual``: of the output's sizes.
    Sums are float32, and the output is rounded once; a row with an infinite value is infinite by its weights' signs.  In the backward pass the gradient behind the activation is rounded to the type once more.
    For the backward pass ``weight`` is kept, ``x`` if ``weight`` has a gradient (no other reads it), and for ``"relu"`` a bit a value, for ``"gelu"`` and ``"silu"`` their derivatives (float32, or beside bfloat16 2**15 times it in float16: eleven bits down to 2**-29).  ``keep8=True``: in ``x``'s place
    8 bits a value of it, as ``layer_norm`` holds them: ``weight``'s gradient is that of the values so held, all others are not touched by it.
    Under autocast, its type is taken, which must be one of the two, for the residual and the output too.  No gradients of gradients.  Under tracing, forward-mode differentiation, transforms of ``torch.func`` and modes
    that follow the operators: by torch's operators, with nothing kept in 8 bits."""
    if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (x, weight)) or not all(t is None or (isinstance(t, torch.Tensor) and t.is_cuda) for t in (bias, residual)):
        raise RuntimeError("x, weight, bias and residual must be CUDA tensors")
    if activation not in L.ACTIVATIONS:
        raise RuntimeError("activation must be one of %s" % ", ".join(map(repr, L.ACTIVATIONS)))
    if ops._unseen(x, weight, bias, residual):
        return _linear_by_operators(x, weight, bias, activation, residual)
    return L.host().linear(x, weight, bias, L.ACTIVATIONS[activation], residual, bool(keep8), L.LINEAR_MAX_DIM)


class Linear(nn.Linear):
    """``nn.Linear`` whose ``forward(x, residual=None)`` is ``linear``, with its ``activation`` and ``keep8``; a state of either is one of the other's."""

    def __init__(self, in_features, out_features, bias=True, activation=None, keep8=False):
        super().__init__(in_features, out_features, bias=bias)
        if activation not in L.ACTIVATIONS:
            raise ValueError("activation must be one of %s" % ", ".join(map(repr, L.ACTIVATIONS)))
        self.activation, self.keep8 = activation, bool(keep8)

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, self.activation, residual, self.keep8)

    def extra_repr(self):
        return super().extra_repr() + (", activation=%s" % self.activation if self.activation else "") + (", keep8=True" if self.keep8 else "")


class FeedForward(nn.Module):
    """``x + down(activation(up(norm(x))))``, the block that a deep model has between its aggregations: a norm and two dense layers, ``features`` to ``hidden`` and
    back, with the activation behind the first and the residual behind the second.  ``keep8``: all three keep 8 bits a value of what their backward passes need of
    their inputs (``x`` itself is kept by nobody: the residual's gradient is the output's).
    Under autocast ``x`` keeps its type, as beside torch's modules: what is added to rows of another type than autocast's is added by an operator of its own."""

    def __init__(self, features, hidden, activation="gelu", eps=1e-5, keep8=False):
        super().__init__()
        self.norm = LayerNorm(features, eps=eps, keep8=keep8)
        self.up = Linear(features, hidden, activation=activation, keep8=keep8)
        self.down = Linear(hidden, features, keep8=keep8)

    def forward(self, x):
        h = self.up(self.norm(x))
        if torch.is_autocast_enabled() and x.dtype != torch.get_autocast_dtype("cuda"):
            return x + self.down(h)
        return self.down(h, residual=x)
