"""A model's last product and its loss as one operator (the reference's last layer and ``nn.CrossEntropyLoss``, train_fastgl.py:328,383):
softmax cross entropy over any number of classes without the logits in memory.  For a handful of classes that saves launches; for as many
classes as a graph has nodes (which entity is it, out of all?) it saves gigabytes.
"""
from __future__ import annotations

import torch
from torch.nn import functional as F

from . import _lib as L
from . import ops
from .conv import _Linear


def _by_operators(x, weight, labels, bias, ignore_index, reduction):
    """The same in torch's operators, for who has to see those: with the logits in memory, in float32."""
    if torch.is_autocast_enabled():
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(to), weight.to(to), None if bias is None else bias.to(to)
    sized = not torch.jit.is_tracing()  # (a trace is of any sizes, and its operators have their own checks)
    if x.dim() != 2 or weight.dim() != 2 or (sized and not (x.size(1) == weight.size(1) and weight.size(0) >= 1 and 1 <= x.size(1) <= L.XENT_MAX_DIM)):
        raise RuntimeError("x %s and weight %s must be [n, d] and [classes, d] with 1 <= d <= %d" % (tuple(x.shape), tuple(weight.shape), L.XENT_MAX_DIM))
    if not (x.dtype in ops._FEAT and weight.dtype == x.dtype and (bias is None or bias.dtype == x.dtype)):
        raise RuntimeError("x, weight and bias must all be of one type in %s" % [str(t) for t in ops._FEAT])
    if bias is not None and (bias.dim() != 1 or (sized and bias.size(0) != weight.size(0))):
        raise RuntimeError("bias must hold a value for each class")
    if labels.dim() != 1 or labels.dtype not in (torch.int32, torch.int64) or (sized and labels.size(0) != x.size(0)):
        raise RuntimeError("labels must be int32 or int64, one for each row of x")
    with torch.autocast("cuda", enabled=False):
        valid = labels != ignore_index
        named = (labels >= 0) & (labels < weight.size(0))
        weight = weight.float()
        if bias is not None:
            bias = bias.float()
            left_out = bias <= -1e30
            weight, bias = torch.where(left_out[:, None], 0.0, weight), torch.where(left_out, float("-inf"), bias)
        logits = F.linear(torch.where(valid[:, None], x.float(), 0.0), weight, bias)
        losses = -torch.log_softmax(logits, 1).gather(1, torch.where(named, labels, 0).long()[:, None])[:, 0]
        losses = torch.where(valid, losses * torch.where(valid & ~named, float("nan"), 1.0), 0.0)  # (a bad label's gradients are no numbers either)
        if reduction == "none":
            return losses
        count = valid.sum()
        return losses.sum() if reduction == "sum" else torch.where(count > 0, losses.sum() / count.clamp(min=1), float("nan"))


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, reduction="mean"):
    """``cross_entropy(x weight^T + bias, labels)`` in float32, with gradients for ``x`` [n, d], ``weight`` [classes, d] (a transposed view of a
    [d, classes] weight will do) and ``bias`` [classes]: float32 or bfloat16, all of one type, ``d`` up to 512.  The logits are formed in pieces
    and never stored; sums, maxima and losses are float32.  ``labels`` [n]: int32 or int64; rows labelled ``ignore_index`` have no loss and no
    gradient, whatever they hold; a label outside ``[0, classes)`` makes a loss that is not a number.  A bias of -1e30 or less, ``-inf`` and the type's
    lowest value among them, leaves its class out, whatever its weights hold; the others and the other rows of ``x`` are finite (float32: below 3.38e38), logits
    below 1e9 in magnitude.
    In float32 each term of a logit or gradient has that type's precision for itself, however far columns, rows and classes lie apart; values and
    shares below 2^-110 have fewer bits.  Fewer than 2^29
    rows and classes together, and 2^28 pieces of 32 columns of ``x``.  ``reduction``: ``"mean"`` over the rows that have a label (not a number if
    none has), ``"sum"`` or ``"none"``.
    In the logits' place the graph keeps copies of ``x`` (two) and ``weight`` of 2 bytes a value in bfloat16 and 6 in float32, columns padded to a
    multiple of 32 (more than 256: to 384 or 512, in float32 also 320), and ``x``'s gradient in float32; the forward pass needs a second copy of ``weight`` meanwhile.  A
    gradient of ``bias`` alone costs what ``weight``'s does, and rows without a label, in ``x`` anywhere, what others do.
    Under autocast, its type is taken.  No gradients of gradients.  Under tracing, forward-mode differentiation, transforms of ``torch.func`` and modes
    that follow the operators: by torch's operators, with the logits in memory."""
    if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (x, weight, labels)) or not (bias is None or (isinstance(bias, torch.Tensor) and bias.is_cuda)):
        raise RuntimeError("x, weight, labels and bias must be CUDA tensors")
    if reduction not in L.REDUCE:
        raise RuntimeError("reduction must be one of %s" % ", ".join(L.REDUCE))
    if ops._unseen(x, weight, labels, bias):
        return _by_operators(x, weight, labels, bias, ignore_index, reduction)
    return L.host().linear_cross_entropy(x, weight, labels, bias, ignore_index, L.REDUCE[reduction], L.XENT_MAX_DIM)


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
