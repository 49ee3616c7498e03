"""Dropout between layers (the reference's ``nn.Dropout``, GraphConv.py:71,84-85) whose mask is never stored: whether an element is
kept is a function of its position, a seed and a stream number (``fgl_dropout``), formed again in the backward pass.  Runs are
reproducible from the seed alone, whatever else draws random numbers, and a layer's activation goes with it in one pass.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L
from . import ops


def dropout(x, p=0.5, seed=0, stream=0, relu=False, training=True, stream_offset=None):
    """``x`` (``relu``: ``max(x, 0)``) with each element kept with probability ``1 - p`` and divided by it, zero otherwise, whatever it
    holds.  Element ``i`` of ``x`` in row-major order is kept if word ``i % 4`` of ``philox4x32_10(counter=(i // 4 low, i // 4 high, stream,
    0x44524F50), key=seed)`` is at least ``round(p * 2**32)``: calls that share a ``seed`` take a ``stream`` (32 bits) of their own each.
    ``stream_offset``: a one-element int32 device tensor that is added to ``stream`` when the kernels run; a captured call draws
    another mask at every replay before which the caller changes it (after the backward pass, which reads it again).
    ``x``: float32 or bfloat16 on the GPU, contiguous or a matrix whose rows lie apart.  ``training=False``: ``x`` itself, or its ``relu``."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if not 0 <= seed < 1 << 64 or not 0 <= stream < 1 << 32:
        raise RuntimeError("seed (%d) and stream (%d) are unsigned, of 64 and 32 bits" % (seed, stream))
    if stream_offset is not None:
        ops._check_input(stream_offset, "stream_offset", ops._I32)
    if not training:
        if not relu:
            return x
        p, stream_offset = 0.0, None
    return L.host().dropout(x, p, seed, stream, relu, stream_offset)


class Dropout(nn.Module):
    """``dropout`` as a layer: ``seed`` makes the masks of a run, every call in training takes the next stream (``calls`` counts them;
    set it to repeat or resume a run).  Layers of one model take a seed each, or share one instance.  ``relu=True``: the activation before it goes with it, in
    evaluation too.  ``stream_offset``: as for ``dropout``, for calls that are captured in a graph (whose stream numbers are those of the
    capture: advance it by more than the calls that one replay makes).  A layer that is computed anew for its backward pass (activation
    checkpoints) would take another stream there: call ``dropout`` with a ``stream`` of its own in such a layer."""

    def __init__(self, p=0.5, seed=0, relu=False):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("p (%g) is no probability" % p)
        self.p, self.seed, self.relu = float(p), int(seed), bool(relu)
        self.calls = 0
        self.stream_offset = None

    def forward(self, x):
        if not self.training:
            return dropout(x, 0.0, relu=self.relu, training=False)
        stream = self.calls & 0xFFFFFFFF
        self.calls += 1
        return dropout(x, self.p, self.seed, stream, self.relu, True, self.stream_offset)

    def extra_repr(self):
        return "p=%g, seed=%d%s" % (self.p, self.seed, ", relu=True" if self.relu else "")
