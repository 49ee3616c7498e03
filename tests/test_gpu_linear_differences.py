"""linear's gradients against differences of its outputs, and infinite values in fp32."""
import numpy as np
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("act", [None, "gelu", "silu"])
@pytest.mark.parametrize("n,d,out", [(40, 30, 20), (500, 100, 64)])
def test_gradients_are_those_of_differences(cuda, act, n, d, out):
    """y along a direction, by two steps, against the gradient's product with it.  What the differences are off by: the roundings of y (gelu's of 1.5e-7 |z| among them) over the step, and the
    third derivative, below 2, times the cube of what z changes by.  Both together are below a hundredth of what the terms of the product are."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    normal = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    leaves = [normal(n, d).requires_grad_(), (normal(out, d) / d ** 0.5).requires_grad_(), normal(out).requires_grad_(), normal(n, out).requires_grad_()]
    dy = normal(n, out)
    f = lambda m: fastgl.linear(m[0], m[1], m[2], act, m[3])  # noqa: E731
    grads = torch.autograd.grad(f(leaves), leaves, dy)
    x, w, b, r = (t.detach().double() for t in leaves)
    z = x @ w.t() + b
    slope = {None: torch.ones_like(z), "silu": torch.sigmoid(z) * (1 + z * torch.sigmoid(-z)),
             "gelu": 0.5 * torch.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5}[act]
    h = 2.0 ** -5
    for i, t in enumerate(leaves):
        v = normal(*t.shape) / (d ** 0.5 if i == 1 else 1.0)  # (z changes by about one)
        up, down = (f([u.detach() + (s * h * v if j == i else 0) for j, u in enumerate(leaves)]).double() for s in (1, -1))
        got, want = float(((up - down) / (2 * h) * dy).sum()), float((grads[i].double() * v).sum())
        e = v.double()
        change = [lambda: e @ w.t(), lambda: x @ e.t(), lambda: e.expand(n, out), lambda: torch.zeros_like(z)][i]()
        cubes = torch.zeros_like(z) if act is None else change.abs() ** 3
        # y's roundings: those of z (d + 8 of its terms; fewer are in a chain), the activation's, the residual's; the inputs' own when they are moved
        terms = (x.abs() @ w.abs().t() + b.abs()) * 1.13 * (d + 8) * U + z.abs() * 1.5e-7 + (r.abs() + z.abs()) * 4 * U
        allowed = float((dy.abs().double() * (terms / h + 2 * h * h / 6 * cubes)).sum())
        size = float((dy.abs().double() * (e.abs() if i == 3 else (slope * change).abs())).sum())
        assert allowed < 0.01 * size, (i, allowed, size)
        assert abs(got - want) < allowed, (i, got, want, allowed)


@pytest.mark.parametrize("n", [300, 27_000])
@pytest.mark.parametrize("d,out", [(96, 130), (100, 64), (129, 130), (250, 256), (16, 40), (1000, 47)])
def test_infinite_values_in_fp32(cuda, n, d, out):
    """A row with one infinite value is infinite by its weights' signs, wherever in the row that is, and its gradient's by theirs; all others are what they were."""
    gen = torch.Generator(device=cuda).manual_seed(n + d)
    x, w, dy = torch.randn((n, d), generator=gen, device=cuda), torch.randn((out, d), generator=gen, device=cuda), torch.randn((n, out), generator=gen, device=cuda)
    w[w.abs() < 2.0 ** -10] = 0.5
    places = [(0, d - 1), (1, d - 2), (70, d - 8), (133, 0), (n - 1, d - 5)]
    for row, c in places:
        x[row, c] = float("inf")
        dy[row, c % out] = float("-inf")
    x.requires_grad_()
    y, z = fastgl.linear(x, w), fastgl.linear(x, w, None, "relu")
    gx, = torch.autograd.grad(y, x, dy)
    good = torch.ones(n, dtype=torch.bool, device=cuda)
    for row, c in places:
        assert torch.equal(y[row], float("inf") * w[:, c].sign())
        assert torch.equal(z[row], torch.where(w[:, c] > 0, float("inf"), 0.0))
        assert torch.equal(gx[row], float("-inf") * w[c % out].sign())
        good[row] = False
    X, W, DY = (t.detach()[good].double() if t is not w else w.double() for t in (x, w, dy))
    for got, want, terms, k in ((y, X @ W.t(), X.abs() @ W.abs().t(), d), (gx, DY @ W, DY.abs() @ W.abs(), out)):
        assert ((got[good].double() - want).abs() <= (k + 8) * U * terms).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [300, 30_000])
@pytest.mark.parametrize("d,out", [(96, 130), (129, 130), (250, 256), (1000, 47)])
def test_infinite_weights(cuda, dtype, n, d, out):
    """An output column with one infinite weight is infinite by its rows' signs, and so is that weight's column of the input's gradient."""
    gen = torch.Generator(device=cuda).manual_seed(n + d)
    x, w, dy = (torch.randn(s, generator=gen, device=cuda) for s in ((n, d), (out, d), (n, out)))
    x, dy = torch.where(x.abs() < 2.0 ** -10, 0.5, x).to(dtype).requires_grad_(), torch.where(dy.abs() < 2.0 ** -10, 0.5, dy).to(dtype)
    places = [(0, d - 1), (31, d - 3), (out - 1, 0)]
    for j, c in places:
        w[j, c] = float("inf")
    w = w.to(dtype)
    y = fastgl.linear(x, w)
    gx, = torch.autograd.grad(y, x, dy)
    columns, rows = torch.ones(out, dtype=torch.bool, device=cuda), torch.ones(d, dtype=torch.bool, device=cuda)
    for j, c in places:
        assert torch.equal(y[:, j].float(), float("inf") * x[:, c].detach().float().sign()) and torch.equal(gx[:, c].float(), float("inf") * dy[:, j].float().sign())
        columns[j] = rows[c] = False
    assert y[:, columns].isfinite().all() and gx[:, rows].isfinite().all()
