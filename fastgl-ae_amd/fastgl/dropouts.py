"""Dropout between layers (the reference's ``nn.Dropout``, GraphConv.py:71,84-85) whose mask is never stored: whether an element is
kept is a function of its position, a seed and a stream number (``fgl_dropout``), formed again in the backward pass.  Runs are
reproducible from the seed alone, whatever else draws random numbers, and a layer's activation goes with it in one pass.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib as L
from . import ops


def _drop(x, p, seed, stream, relu, stream_offset):
    """fgl_dropout on ``x``: rows with unit column stride, or any shape without gaps."""
    rows, cols, stride = (1, x.numel(), x.numel()) if x.is_contiguous() else (int(x.size(0)), int(x.size(1)), int(x.stride(0)))
    with ops._on_device(x.device):
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if out.numel():
            L.check(L.lib().fgl_dropout(x.data_ptr(), stride, rows, cols, L.F32 if x.dtype == torch.float32 else L.BF16, p, seed, stream,
                                        L.ptr(stream_offset), int(relu), out.data_ptr(), L.stream_handle()))
    return out


def _gaps_in_rows_only(x):
    return x.is_contiguous() or (x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= x.size(1))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, stream, relu, stream_offset):
        out = _drop(x, p, seed, stream, relu, stream_offset)
        ctx.args = p, seed, stream
        ctx.relu = relu
        ctx.save_for_backward(out if relu else None, stream_offset)  # (the mask is made again from the same offset: one changed meanwhile is an error)
        return out

    @staticmethod
    def backward(ctx, d_out):
        p, seed, stream = ctx.args
        out, stream_offset = ctx.saved_tensors
        if torch.is_grad_enabled():  # (a graph of the gradients is being built; the gradient is linear in d_out)
            if ctx.relu:
                return torch.where(out <= 0, 0.0, d_out * (1.0 / (1.0 - p) if p < 1.0 else 0.0)), None, None, None, None, None
            return _Dropout.apply(d_out if _gaps_in_rows_only(d_out) else d_out.contiguous(), p, seed, stream, False, stream_offset), None, None, None, None, None
        if not ctx.relu:
            return _drop(d_out if _gaps_in_rows_only(d_out) else d_out.contiguous(), p, seed, stream, False, stream_offset), None, None, None, None, None
        d_out = d_out.contiguous()
        with ops._on_device(d_out.device):
            d_x = torch.empty(out.shape, dtype=out.dtype, device=out.device)
            if d_x.numel():
                L.check(L.lib().fgl_dropout_relu_backward(d_out.data_ptr(), out.data_ptr(), out.numel(), L.F32 if out.dtype == torch.float32 else L.BF16, p,
                                                          d_x.data_ptr(), L.stream_handle()))
        return d_x, None, None, None, None, None


def dropout(x, p=0.5, seed=0, stream=0, relu=False, training=True, stream_offset=None):
    """``x`` (``relu``: ``max(x, 0)``) with each element kept with probability ``1 - p`` and divided by it, zero otherwise, whatever it
    holds.  Element ``i`` of ``x`` in row-major order is kept if word ``i % 4`` of ``philox4x32_10(counter=(i // 4 low, i // 4 high, stream,
    0x44524F50), key=seed)`` is at least ``round(p * 2**32)``: calls that share a ``seed`` take a ``stream`` (32 bits) of their own each.
    ``stream_offset``: a one-element int32 device tensor that is added to ``stream`` when the kernels run; a captured call draws
    another mask at every replay before which the caller changes it (after the backward pass, which reads it again).
    ``x``: float32 or bfloat16 on the GPU, contiguous or a matrix whose rows lie apart.  ``training=False``: ``x`` itself, or its ``relu``."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if x.dtype not in ops._FEAT:
        raise RuntimeError("x must have dtype in %s, got %s" % ([str(d) for d in ops._FEAT], x.dtype))
    if not _gaps_in_rows_only(x):
        raise RuntimeError("x must be contiguous, or a matrix with unit column stride")
    p, seed, stream = float(p), int(seed), int(stream)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError("p (%g) is no probability" % p)
    if not 0 <= seed < 1 << 64 or not 0 <= stream < 1 << 32:
        raise RuntimeError("seed (%d) and stream (%d) are unsigned, of 64 and 32 bits" % (seed, stream))
    if stream_offset is not None:
        ops._check_input(stream_offset, "stream_offset", ops._I32)
        if stream_offset.numel() != 1:
            raise RuntimeError("stream_offset must hold one int32")
        ops._same_device(x, stream_offset)
    if not training:
        if not relu:
            return x
        p, stream_offset = 0.0, None
    if not (torch.is_grad_enabled() and x.requires_grad):
        return _drop(x, p, seed, stream, relu, stream_offset)
    return _Dropout.apply(x, p, seed, stream, bool(relu), stream_offset)


class Dropout(nn.Module):
    """``dropout`` as a layer: ``seed`` makes the masks of a run, every call in training takes the next stream (``calls`` counts them;
    set it to repeat or resume a run).  Layers of one model take a seed each, or share one instance.  ``relu=True``: the activation before it goes with it, in
    evaluation too.  ``stream_offset``: as for ``dropout``, for calls that are captured in a graph (whose stream numbers are those of the
    capture: advance it by more than the calls that one replay makes)."""

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
