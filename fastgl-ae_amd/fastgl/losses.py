"""A model's last product and its loss as one operator (the reference's last layer and ``nn.CrossEntropyLoss``, train_fastgl.py:328,383):
softmax cross entropy over any number of classes without the logits in memory.  For a handful of classes that saves launches; for as many
classes as a graph has nodes (which entity is it, out of all?) it saves gigabytes.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops
from .conv import _Linear


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, ignore_index, reduction):
        (n, dim), classes = x.shape, int(weight.size(0))
        dev, dtype = x.device, L.F32 if x.dtype == torch.float32 else L.BF16
        want = (L.XENT_ROWS if ctx.needs_input_grad[0] else 0) | (L.XENT_WEIGHTS if any(ctx.needs_input_grad[1:3]) else 0)
        ctx.sizes = n, classes, dim, dtype, reduction, want
        ctx.types = x.dtype, bias is not None
        lib = L.lib()
        with ops._on_device(dev):
            if n == 0:
                ctx.state = torch.empty(0, device=dev)
                return torch.full((0,) if reduction == L.REDUCE["none"] else (), float("nan") if reduction == L.REDUCE["mean"] else 0.0, device=dev)
            loss = torch.empty((n,) if reduction == L.REDUCE["none"] else (), dtype=torch.float32, device=dev)
            state = L.workspace(lib.fgl_linear_cross_entropy_state_bytes(n, classes, dim, dtype, want), dev)
            ws = L.workspace(lib.fgl_linear_cross_entropy_workspace_bytes(n, classes, dim, dtype, want, 0), dev)
            L.check(lib.fgl_linear_cross_entropy(x.data_ptr(), *x.stride(), weight.data_ptr(), *weight.stride(), L.ptr(bias), labels.data_ptr(),
                                                 int(labels.dtype == torch.int64), ignore_index, n, classes, dim, dtype, reduction, want, loss.data_ptr(),
                                                 state.data_ptr(), state.numel(), ws.data_ptr(), ws.numel(), L.stream_handle()))
        ctx.state = state  # (no tensor of the caller's: it cannot be changed in between)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        n, classes, dim, dtype, reduction, want = ctx.sizes
        of_type, with_bias = ctx.types
        dev = d_loss.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        lib = L.lib()
        with ops._on_device(dev):
            make = torch.empty if n else torch.zeros
            d_x = make((n, dim), dtype=of_type, device=dev) if need_x else None
            d_w = make((classes, dim), dtype=of_type, device=dev) if need_w or need_b else None
            d_b = make(classes, dtype=of_type, device=dev) if need_b else None
            if n:
                d_loss = d_loss.contiguous()
                ws = L.workspace(lib.fgl_linear_cross_entropy_workspace_bytes(n, classes, dim, dtype, want, 1), dev)
                L.check(lib.fgl_linear_cross_entropy_backward(d_loss.data_ptr(), n, classes, dim, dtype, reduction, want, ctx.state.data_ptr(),
                                                              ctx.state.numel(), L.ptr(d_x), L.ptr(d_w), L.ptr(d_b), ws.data_ptr(), ws.numel(), L.stream_handle()))
        return d_x, d_w if need_w else None, d_b, None, None, None


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, reduction="mean"):
    """``cross_entropy(x weight^T + bias, labels)`` in float32, with gradients for ``x`` [n, d], ``weight`` [classes, d] (a transposed view of a
    [d, classes] weight will do) and ``bias`` [classes]: float32 or bfloat16, all of one type, ``d`` up to 512.  The logits are formed in pieces
    and never stored; sums, maxima and losses are float32.  ``labels`` [n]: int32 or int64; rows labelled ``ignore_index`` have no loss and no
    gradient; a label outside ``[0, classes)`` makes a loss that is not a number.  A bias of -1e30 or less, ``-inf`` and the type's lowest value among them, leaves its class out; ``x`` and
    ``weight`` are finite, logits below 1e9 in magnitude.  ``reduction``: ``"mean"`` over the rows that have a label (not a number if none has), ``"sum"`` or ``"none"``.
    Under autocast, its type is taken.  No gradients of gradients."""
    if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (x, weight, labels)) or not (bias is None or (isinstance(bias, torch.Tensor) and bias.is_cuda)):
        raise RuntimeError("x, weight, labels and bias must be CUDA tensors")
    if torch.is_autocast_enabled():
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(to), weight.to(to), None if bias is None else bias.to(to)
    if x.dim() != 2 or weight.dim() != 2 or x.size(1) != weight.size(1) or weight.size(0) < 1 or not 1 <= x.size(1) <= L.XENT_MAX_DIM:
        raise RuntimeError("x %s and weight %s must be [n, d] and [classes, d] with 1 <= d <= %d" % (tuple(x.shape), tuple(weight.shape), L.XENT_MAX_DIM))
    if x.dtype not in ops._FEAT or weight.dtype != x.dtype or not (bias is None or bias.dtype == x.dtype):
        raise RuntimeError("x, weight and bias must all be of one type in %s" % [str(d) for d in ops._FEAT])
    if bias is not None and (bias.dim() != 1 or bias.size(0) != weight.size(0) or not bias.is_contiguous()):
        raise RuntimeError("bias must be contiguous and hold a value for each class")
    if labels.dim() != 1 or labels.size(0) != x.size(0) or labels.dtype not in ops._PTR or not labels.is_contiguous():
        raise RuntimeError("labels must be contiguous int32 or int64, one for each row of x")
    if reduction not in L.REDUCE:
        raise RuntimeError("reduction must be one of %s" % ", ".join(L.REDUCE))
    ops._same_device(x, weight, labels, bias)
    return _LinearCrossEntropy.apply(x, weight, bias, labels, int(ignore_index), L.REDUCE[reduction])


class LinearCrossEntropy(_Linear):
    """A last layer that gives the loss: ``nn.Linear(in_features, num_classes)`` whose ``forward(x, labels)`` is ``linear_cross_entropy``;
    ``logits(x)`` are the layer's outputs."""

    def __init__(self, in_features, num_classes, bias=True, ignore_index=-100, reduction="mean"):
        super().__init__(in_features, num_classes, bias=bias)
        self.ignore_index, self.reduction = int(ignore_index), reduction

    def forward(self, x, labels):
        return linear_cross_entropy(x, self.weight, labels, self.bias, self.ignore_index, self.reduction)

    def logits(self, x):
        return super().forward(x)
