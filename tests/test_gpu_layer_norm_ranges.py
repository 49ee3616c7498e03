"""layer_norm of rows at the ends of the types' range, with no eps or a tiny one: the normed values are of ordinary size, and so are the weights' gradients, where a row's spread, one
over it, or a difference from the mean is past what fp32 holds."""
import numpy as np
import pytest
import torch

import fastgl
from held8 import held

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def rows(cuda, n, d, power, dtype):
    """Multiples of 2^power up to 100 times it, exact in both types; and a column far from the others."""
    gen = torch.Generator(device=cuda).manual_seed(n + d)
    x = torch.randint(-100, 101, (n, d), generator=gen, device=cuda).double()
    x[:, d // 2] = 127
    x[1::2] = x[1::2].clamp(max=-60)  # (rows whose mean is far from zero)
    x[1::2, d // 2] = 127
    return (x * 2.0 ** power).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu,keep8", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("power", [-133, -130, -110, -60, 0, 60, 120, 121])
@pytest.mark.parametrize("n,d", [(40, 30), (300, 100), (70, 602), (9, 2048)])
def test_values_and_gradients(cuda, dtype, relu, keep8, power, n, d):
    """The bounds are those of rows of ordinary size: y one rounding of h, two of the product and sum; h in 64 bits, rounded once; sums of d and of n values in fp32, each rounding
    off by U of the sum of magnitudes.  dy is so small (large) where the rows are that dx is of ordinary size; below 2^-126 half of a type's smallest value more."""
    x = rows(cuda, n, d, power, dtype).requires_grad_()
    gen = torch.Generator(device=cuda).manual_seed(power + 200)
    w, b = (t.to(dtype).requires_grad_() for t in (1 + 0.3 * torch.randn(d, generator=gen, device=cuda), 0.3 * torch.randn(d, generator=gen, device=cuda)))
    dy = (torch.randn((n, d), generator=gen, device=cuda) * 2.0 ** min(max(power / 2, -60), 60)).to(dtype)
    y = fastgl.layer_norm(x, w, b, eps=0.0, relu=relu, keep8=keep8)
    got = torch.autograd.grad(y, (x, w, b), dy)
    X, W, B, DY = (t.detach().cpu().double().numpy() for t in (x, w, b, dy))
    c = X - X.mean(1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True))
    h = c * r
    want = h * W + B
    half = HALF[dtype]
    near = relu & (np.abs(want) < 1e-13)  # (64 bits here and there)
    assert not near.any()
    if relu:
        DY = np.where(want <= 0, 0.0, DY)
        want = np.where(want <= 0, 0.0, want)
    off = half * np.abs(want) + 4 * U * (np.abs(h * W) + np.abs(B))
    assert (np.abs(y.detach().cpu().double().numpy() - want) <= off).all()
    if keep8:
        h = held(h)
    g = DY * W
    H, G = np.abs(h), np.abs(g)
    dx = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    sums = (d + 8) * U * (G.mean(1, keepdims=True) + H * (G * H).mean(1, keepdims=True))
    least = 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150
    off = half * np.abs(dx) + r * (8 * U * (G + G.mean(1, keepdims=True) + H * (G * H).mean(1, keepdims=True)) + sums) + least
    assert (np.abs(got[0].cpu().double().numpy() - dx) <= off).all()
    for t, terms in ((got[1], DY * h), (got[2], DY)):
        e = terms.sum(0)
        assert (np.abs(t.cpu().double().numpy() - e) <= half * np.abs(e) + (n + 8) * U * np.abs(terms).sum(0)).all()


def test_rows_of_one_value_and_a_tiny_eps(cuda):
    """Nothing to norm: the values are zeros, whatever 1 / sqrt(eps) is."""
    x = torch.full((40, 100), 3.5, device=cuda, requires_grad=True)
    w, b = torch.randn(100, device=cuda, requires_grad=True), torch.randn(100, device=cuda, requires_grad=True)
    for eps in (1e-60, 1e-100, 1e-300):
        y = fastgl.layer_norm(x, w, b, eps=eps)
        gw, gb = torch.autograd.grad(y, (w, b), torch.ones_like(y))
        assert torch.equal(y, b.expand(40, 100)) and not gw.any() and torch.equal(gb, torch.full_like(gb, 40))
