"""Dropout between layers (the reference's ``nn.Dropout``, GraphConv.py:71,84-85) whose mask is never stored: whether an element is
kept is a function of its position, a seed and a stream number (``fgl_dropout``), formed again in the backward pass.  Runs are
reproducible from the seed alone, whatever else draws random numbers, and a layer's activation goes with it in one pass.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.utils._python_dispatch import _disable_current_modes

from . import _lib as L
from . import ops

_TAG = 0x44524F50  # the counter's last word: "DROP"


def _drawn_seed():
    """A seed from torch's generator (of the CPU: ``torch.manual_seed`` governs it)."""
    with _disable_current_modes():  # (a number, also where tensors hold none)
        return int(torch.randint(0, 2 ** 63 - 1, (), device="cpu"))


def _kept(x, p, seed, stream, stream_offset):
    """Which elements of ``x`` are kept, in torch's operators: the generator's rounds on whole numbers of 64 bits."""
    low, n = 0xFFFFFFFF, x.numel()
    quad = torch.arange((n + 3) // 4, device=x.device)
    c0, c1, c2, c3 = quad & low, quad >> 32, torch.full_like(quad, stream), torch.full_like(quad, _TAG)
    if stream_offset is not None:
        c2 = (c2 + stream_offset.long()) & low
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (modulo 2^64: either half is the product's)
        c0, c1, c2, c3 = (b >> 32) & low ^ c1 ^ k0, b & low, (a >> 32) & low ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return (torch.stack([c0, c1, c2, c3], 1).view(-1)[:n] >= round(p * 2.0 ** 32)).view(x.shape)


def _by_operators(x, p, seed, stream, relu, stream_offset):
    """The same values in torch's operators, for who has to see those: some hundred launches."""
    if x.dtype not in ops._FEAT:
        raise RuntimeError("x must have dtype in %s, got %s" % ([str(t) for t in ops._FEAT], x.dtype))
    if not 0.0 <= p <= 1.0:
        raise RuntimeError("p (%g) is no probability" % p)
    if stream_offset is not None and stream_offset.numel() != 1:
        raise RuntimeError("stream_offset must hold one int32")
    v = torch.relu(x) if relu else x
    if p == 0.0:
        return v.clone() if v is x else v
    scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    return torch.where(_kept(x, p, seed, stream, stream_offset), v.float() * scale, 0.0).to(x.dtype)


def dropout(x, p=0.5, seed=None, stream=0, relu=False, training=True, stream_offset=None):
    """``x`` (``relu``: ``max(x, 0)``) with each element kept with probability ``1 - p`` and divided by it, zero otherwise, whatever it
    holds.  Element ``i`` of ``x`` in row-major order is kept if word ``i % 4`` of ``philox4x32_10(counter=(i // 4 low, i // 4 high, stream,
    0x44524F50), key=seed)`` is at least ``round(p * 2**32)``: calls that share a ``seed`` take a ``stream`` (32 bits) of their own each.
    ``seed=None``: another one for each call, from torch's generator (a captured call keeps the one of its capture).
    ``stream_offset``: a one-element int32 device tensor that is added to ``stream`` when the kernels run; a captured call draws
    another mask at every replay before which the caller changes it (after the backward pass, which reads it again).
    ``x``: float32 or bfloat16 on the GPU, contiguous or a matrix whose rows lie apart.  ``training=False``: ``x`` itself, or its ``relu``.
    Under tracing, forward-mode differentiation, transforms of ``torch.func`` and modes that follow the operators: the same values by
    torch's operators (``_by_operators``); a traced call keeps the seed and stream of its trace."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    if seed is None:
        seed = _drawn_seed() if training and 0.0 < p < 1.0 else 0
    if not 0 <= seed < 1 << 64 or not 0 <= stream < 1 << 32:
        raise RuntimeError("seed (%d) and stream (%d) are unsigned, of 64 and 32 bits" % (seed, stream))
    if stream_offset is not None:
        ops._check_input(stream_offset, "stream_offset", ops._I32)
    if not training:
        if not relu:
            return x
        p, stream_offset = 0.0, None
    if ops._unseen(x, stream_offset):
        return _by_operators(x, p, seed, stream, relu, stream_offset)
    return L.host().dropout(x, p, seed, stream, relu, stream_offset)


class Dropout(nn.Module):
    """``dropout`` as a layer: ``seed`` makes the masks of a run, every call in training takes the next stream (``calls`` counts them;
    set it to repeat a run).  Both are in ``state_dict()``, so that a run that is resumed goes on with the next stream; a state without them leaves
    them as they are.  Layers of one model take a seed each, or share one instance; ``seed=None``: one from torch's generator
    when the layer is made.  ``relu=True``: the activation before it goes with it, in
    evaluation too.  ``stream_offset``: as for ``dropout``, for calls that are captured in a graph (whose stream numbers are those of the
    capture: advance it by more than the calls that one replay makes).  A layer that is computed anew for its backward pass (activation
    checkpoints) would take another stream there: call ``dropout`` with a ``stream`` of its own in such a layer."""

    def __init__(self, p=0.5, seed=None, relu=False):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("p (%g) is no probability" % p)
        if seed is not None and not 0 <= int(seed) < 1 << 64:
            raise ValueError("seed (%d) is unsigned, of 64 bits" % seed)
        self.p, self.seed, self.relu = float(p), _drawn_seed() if seed is None else int(seed), bool(relu)
        self.calls = 0
        self.stream_offset = None

    def forward(self, x, relu=None):
        """``relu``: in the place of the layer's own, if given."""
        relu = self.relu if relu is None else relu
        if not self.training:
            return dropout(x, 0.0, relu=relu, training=False)
        stream = self.calls & 0xFFFFFFFF
        self.calls += 1
        return dropout(x, self.p, self.seed, stream, relu, True, self.stream_offset)

    def get_extra_state(self):
        return torch.tensor([self.seed - (self.seed >> 63 << 64), self.calls], dtype=torch.int64, device="cpu")

    def set_extra_state(self, state):
        seed, self.calls = state.tolist()
        self.seed = seed % (1 << 64)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if prefix + "_extra_state" in missing_keys:  # (the state of a model without a seed)
            missing_keys.remove(prefix + "_extra_state")

    def extra_repr(self):
        return "p=%g, seed=%d%s" % (self.p, self.seed, ", relu=True" if self.relu else "")
