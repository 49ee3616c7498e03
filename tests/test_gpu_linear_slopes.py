"""The derivatives that linear keeps for gelu and silu beside bf16, one by one: with the identity for a weight, and gradients of one, the input's gradient is the derivative
itself, rounded once to the type."""
import numpy as np
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def slopes(z, act):
    """act'(z) and what the kernel's formula of it may be off by: the exponential's argument is rounded (a part of |z| U, or z^2 U, of the exponential), the instructions
    and the products each by some U; gelu's distribution function is off by 0.75e-7."""
    if act == "silu":
        e = np.exp(-np.abs(z))
        p = np.where(z < 0, e / (1 + e), 1 / (1 + e))
        q = np.where(z < 0, 1 / (1 + e), e / (1 + e))
        return p * (1 + z * q), (2 * np.abs(z) + 12) * U * p * (1 + np.abs(z) * q) + 4 * U * p * np.abs(z)
    density = np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    cdf = 0.5 * torch.erfc(-torch.from_numpy(z) / 2 ** 0.5).numpy()
    return cdf + z * density, 0.75e-7 + (z * z + 12) * U * np.abs(z) * density + 12 * U * cdf


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("n", [700, 120_000])
def test_of_sums_that_are_not_rounded(cuda, act, n):
    """z = x + b has more bits than bf16.  Off by half a step of fp16 (2^-11) of the derivative, which is held times 2^15: below 2^-29 of half its smallest step, 2^-40; and by
    the one rounding to bf16.  Near its zero a derivative tells a rounded z by a hundred times that."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    d = 64
    x = torch.empty((n, d), device=cuda)
    x[:, :16] = torch.rand((n, 16), generator=gen, device=cuda) * 30 - 24
    x[:, 16:32] = (-1.2785 if act == "silu" else -0.7518) + 0.03 * torch.randn((n, 16), generator=gen, device=cuda)
    x[:, 32:] = 3 * torch.randn((n, 32), generator=gen, device=cuda)
    x = x.bfloat16().requires_grad_()
    b = (0.004 * torch.randn(d, generator=gen, device=cuda)).bfloat16()
    w = torch.eye(d, device=cuda).bfloat16()
    g, = torch.autograd.grad(fastgl.linear(x, w, b, act), x, torch.ones((n, d), device=cuda, dtype=torch.bfloat16))
    z = x.detach().cpu().double().numpy() + b.cpu().double().numpy()
    slope, off = slopes(z, act)
    off = off + U * np.abs(z)  # (the sum's rounding; derivatives change by at most 0.8 times what z does)
    off = off if act == "gelu" else np.where(z < -4, off - U * np.abs(z) + U * np.abs(z) * np.abs(slope) * 1.5, off)  # (there by 1.5 times the derivative)
    bound = (2.0 ** -11 * np.abs(slope) + 2.0 ** -40 + off) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(slope)
    far = np.abs(g.cpu().double().numpy() - slope) - bound
    assert (far <= 0).all(), (far.max(), z.flat[far.argmax()])


def test_small_derivatives_are_not_lost(cuda):
    """silu's at -12 .. -24, 7e-5 to 9e-10: within a hundredth, as bf16 holds them."""
    z = -torch.linspace(12, 24, 64, device=cuda).bfloat16()
    x = z.expand(40, 64).contiguous().requires_grad_()
    g, = torch.autograd.grad(fastgl.linear(x, torch.eye(64, device=cuda).bfloat16(), None, "silu"), x, torch.ones_like(x))
    t = z.double()
    want = torch.exp(t) * (1 + t)
    assert ((g.double() - want).abs() <= 0.01 * want.abs()).all()
