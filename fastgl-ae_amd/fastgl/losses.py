"""A model's last product and its loss as one operator (the reference's last layer and ``nn.CrossEntropyLoss``, train_fastgl.py:328,383):
softmax cross entropy over any number of classes without the logits in memory.  For a handful of classes that saves launches; for as many
classes as a graph has nodes (which entity is it, out of all?) it saves gigabytes.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .conv import _Linear


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, reduction="mean"):
    """``cross_entropy(x weight^T + bias, labels)`` in float32, with gradients for ``x`` [n, d], ``weight`` [classes, d] (a transposed view of a
    [d, classes] weight will do) and ``bias`` [classes]: float32 or bfloat16, all of one type, ``d`` up to 512.  The logits are formed in pieces
    and never stored; sums, maxima and losses are float32.  ``labels`` [n]: int32 or int64; rows labelled ``ignore_index`` have no loss and no
    gradient, whatever they hold; a label outside ``[0, classes)`` makes a loss that is not a number.  A bias of -1e30 or less, ``-inf`` and the type's
    lowest value among them, leaves its class out; ``weight`` and the other rows of ``x`` are finite (float32: below 3.38e38), logits below 1e9 in magnitude.
    In float32 each term of a logit or gradient has that type's precision for itself, however far columns, rows and classes lie apart; values and
    shares below 2^-110 have fewer bits.  Fewer than 2^29
    rows and classes together, and 2^28 pieces of 32 columns of ``x``.  ``reduction``: ``"mean"`` over the rows that have a label (not a number if
    none has), ``"sum"`` or ``"none"``.
    Under autocast, its type is taken.  No gradients of gradients."""
    if not all(isinstance(t, torch.Tensor) and t.is_cuda for t in (x, weight, labels)) or not (bias is None or (isinstance(bias, torch.Tensor) and bias.is_cuda)):
        raise RuntimeError("x, weight, labels and bias must be CUDA tensors")
    if reduction not in L.REDUCE:
        raise RuntimeError("reduction must be one of %s" % ", ".join(L.REDUCE))
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
