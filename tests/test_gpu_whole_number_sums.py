"""Gradients of norm and dense layers over many rows, of whole numbers: their sums stay below 2^24 and are exact, in whatever order they are formed, so that one row left out or
taken twice shows, wherever it is."""
import numpy as np
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu


def whole(gen, cuda, most, *size):
    """1 .. most and their negatives."""
    return torch.randint(1, most + 1, size, generator=gen, device=cuda) * (1 - 2 * torch.randint(0, 2, size, generator=gen, device=cuda))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,stride", [(1, 2, 2), (63, 32, 34), (70_001, 64, 64), (40_000, 100, 101), (300_000, 8, 8), (66_003, 256, 256), (9001, 602, 602), (20_011, 1000, 1000), (4099, 2048, 2048), (8200, 34, 40)])
def test_norm(cuda, dtype, relu, keep8, n, d, stride):
    """Rows of as many ones as minus ones, times a power of two: the normed values are 1 and -1, exactly, without eps."""
    gen = torch.Generator(device=cuda).manual_seed(n + d)
    signs = torch.ones((n, d), device=cuda)
    signs[:, ::2] = -1
    signs = signs * (1 - 2 * torch.randint(0, 2, (n, 1), generator=gen, device=cuda)).float()
    signs = signs[:, torch.randperm(d, generator=gen, device=cuda)]
    x = torch.empty((n, stride), device=cuda, dtype=dtype)[:, :d]
    x.copy_(signs * torch.exp2(torch.randint(-3, 4, (n, 1), generator=gen, device=cuda).float()))
    w, b = torch.full((d,), 2.0, device=cuda, dtype=dtype), torch.full((d,), 1.0, device=cuda, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x.detach(), w, b)]
    dy = whole(gen, cuda, 3, n, d).to(dtype)
    y = fastgl.layer_norm(*leaves, eps=0.0, relu=relu, keep8=keep8)
    want = 2 * signs + 1
    assert torch.equal(y, (want.clamp(min=0) if relu else want).to(dtype))
    g = torch.autograd.grad(y, leaves, dy)
    dz = dy.double() * (signs > 0 if relu else 1)
    assert torch.equal(g[1], (dz * signs.double()).sum(0).float().to(dtype)) and torch.equal(g[2], dz.sum(0).float().to(dtype))


SIZES = [(1, 1, 1), (2, 3, 5), (15, 33, 47), (63, 64, 64), (65, 64, 64), (8000, 100, 256), (40_000, 64, 128), (40_001, 33, 62), (107_003, 100, 256), (8192, 602, 256), (3001, 416, 96), (5003, 1030, 70),
         (110_255, 64, 30), (140_001, 100, 40), (26_999, 640, 128), (26_192, 1217, 60), (26_300, 2400, 24), (100_193, 17, 129), (50_001, 104, 68), (87_000, 256, 512)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,out", SIZES)
def test_linear(cuda, dtype, act, keep8, n, d, out):
    """x of 1 .. 7, gradients of 1 .. 3, weights of 1 .. 3: what 8 bits hold of x is x.  (Sums of the largest magnitudes here: 21 n < 2^24.)"""
    gen = torch.Generator(device=cuda).manual_seed(n + d + out)
    x, w = whole(gen, cuda, 7, n, d), whole(gen, cuda, 3, out, d)
    b, dy = whole(gen, cuda, 9, out), whole(gen, cuda, 3, n, out)
    leaves = [t.to(dtype).requires_grad_() for t in (x, w, b)]
    y = fastgl.linear(*leaves, activation=act, keep8=keep8)
    g = torch.autograd.grad(y, leaves, dy.to(dtype))
    X, W, DZ = (t.cpu().double().numpy() for t in (x, w, dy))
    z = X @ W.T + b.cpu().double().numpy()
    if act == "relu":
        DZ = DZ * (z > 0)
        z = np.maximum(z, 0)
    for name, got, want in zip(("y", "x", "w", "b"), (y, *g), (z, DZ @ W, DZ.T @ X, DZ.sum(0))):
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(dtype)), name
