"""fastgl.layer_norm against the formula in 64 bits: values and all gradients, at the sizes where lanes, loads and rows end, with what is kept in full and in
8 bits."""
import numpy as np
import pytest
import torch

import fastgl
from held8 import held

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def formula(x, w, b, dy, eps, relu, keep8):
    """y, dx, dw, db in float64, and for the tolerances: the normed values, 1 / sqrt, the gradient by h."""
    x, w, b, dy = (t.detach().cpu().double().numpy() for t in (x, w, b, dy))
    c = x - x.mean(1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    h = c * r
    y = h * w + b
    if relu:
        dy = np.where(y <= 0, 0.0, dy)
        y = np.where(y <= 0, 0.0, y)
    if keep8:
        h = held(h)
    g = dy * w
    dx = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return y, dx, (dy * h).sum(0), dy.sum(0), dict(h=h, r=r, g=g, dy=dy)


def close(got, want, bound, dtype):
    got = got.detach().cpu().double().numpy()
    assert got.shape == want.shape
    far = np.abs(got - want) - (HALF[dtype] * np.abs(want) + bound)
    assert (far <= 0).all(), (np.abs(got - want).max(), far.max())


def check(x, w, b, dy, eps, relu, keep8, y, grads):
    """Errors: y one rounding of h, two of the product and sum; sums of d values in fp32, each rounding off by U of the sum of magnitudes; sums over n rows by
    U n of theirs (fewer roundings are in a chain).  h: (x - mean) in 64 bits, rounded, times a rounded 1 / sqrt: 3 U of it."""
    dtype, n, d = x.dtype, x.shape[0], x.shape[1]
    want_y, want_dx, want_dw, want_db, m = formula(x, w, b, dy, eps, relu, keep8)
    W, B = (t.detach().cpu().double().numpy() for t in (w, b))
    H = np.abs(m["h"])
    close(y, want_y, 4 * U * (H * np.abs(W) + np.abs(B)), dtype)
    G = np.abs(m["g"])
    sums = (d + 8) * U * (G.mean(1, keepdims=True) + H * (G * H).mean(1, keepdims=True))
    close(grads[0], want_dx, m["r"] * (8 * U * (G + G.mean(1, keepdims=True) + H * (G * H).mean(1, keepdims=True)) + sums), dtype)
    close(grads[1], want_dw, (n + 8) * U * (np.abs(m["dy"]) * H).sum(0), dtype)
    close(grads[2], want_db, (n + 8) * U * np.abs(m["dy"]).sum(0), dtype)


def problem(cuda, n, d, dtype, stride=None, seed=0, mean=1.0):
    gen = torch.Generator(device=cuda).manual_seed(1000 * seed + n + d)
    normal = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    x = (normal(n, stride or d) * (0.1 + 2 * torch.rand((n, 1), generator=gen, device=cuda)) + mean * normal(n, 1)).to(dtype)[:, :d]
    return x.requires_grad_(), (1 + 0.3 * normal(d)).to(dtype).requires_grad_(), (0.3 * normal(d)).to(dtype).requires_grad_(), normal(n, d).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,stride", [(1, 1, 1), (1, 2, 3), (3, 7, 7), (5, 31, 33), (33, 32, 32), (70, 33, 35), (129, 47, 47), (40, 63, 64), (100, 64, 100), (17, 65, 65),
                                        (515, 100, 100), (50, 128, 129), (31, 129, 130), (1000, 256, 256), (9, 257, 300), (66, 512, 512), (13, 513, 513), (21, 602, 602),
                                        (7, 1024, 1025), (5, 1025, 1025), (4, 2047, 2047), (3, 2048, 2050)])
def test_values_and_gradients(cuda, dtype, relu, keep8, n, d, stride):
    x, w, b, dy = problem(cuda, n, d, dtype, stride)
    y = fastgl.layer_norm(x, w, b, eps=1e-5, relu=relu, keep8=keep8)
    assert y.is_contiguous() and y.dtype == dtype
    grads = torch.autograd.grad(y, (x, w, b), dy)
    check(x, w, b, dy, 1e-5, relu, keep8, y, grads)
    assert torch.equal(fastgl.layer_norm(x.detach(), w, b.detach(), relu=relu), y) and torch.equal(fastgl.layer_norm(x.detach(), w.detach(), b.detach(), relu=relu), y)


@pytest.mark.parametrize("keep8", [False, True])
def test_many_rows_are_the_same_on_every_run(cuda, keep8):
    for n, d, dtype in ((70_001, 64, torch.float32), (40_000, 100, torch.bfloat16), (300_000, 8, torch.float32)):
        x, w, b, dy = problem(cuda, n, d, dtype)
        runs = []
        for _ in range(3):
            y = fastgl.layer_norm(x, w, b, relu=True, keep8=keep8)
            runs.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
        check(x, w, b, dy, 1e-5, True, keep8, runs[0][0], runs[0][1:])
        assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r))


def test_rows_far_from_zero(cuda):
    x, w, b, dy = problem(cuda, 200, 100, torch.float32)
    x = (x.detach() + 4096.0).requires_grad_()  # (values are exact: what they differ in is theirs)
    y = fastgl.layer_norm(x, w, b)
    check(x, w, b, dy, 1e-5, False, False, y, torch.autograd.grad(y, (x, w, b), dy))


def test_offsets_beyond_32_bits(cuda):
    n, d = (1 << 32) // 512 + 37, 512
    x = torch.empty((n, d), device=cuda, dtype=torch.bfloat16).normal_().requires_grad_()
    w, b = torch.randn(d, device=cuda).bfloat16().requires_grad_(), torch.randn(d, device=cuda).bfloat16().requires_grad_()
    y = fastgl.layer_norm(x, w, b, relu=True, keep8=True)
    dy = torch.zeros((n, d), device=cuda, dtype=torch.bfloat16)
    some = torch.cat([torch.arange(40), torch.arange(n - 90, n)]).to(cuda)
    dy[some] = torch.randn((130, d), device=cuda).bfloat16()
    g = torch.autograd.grad(y, (x, w, b), dy)
    xs = x.detach()[some].clone().requires_grad_()
    ys = fastgl.layer_norm(xs, w, b, relu=True, keep8=True)
    assert torch.equal(ys, y[some])
    s = torch.autograd.grad(ys, (xs, w, b), dy[some])
    assert torch.equal(s[0], g[0][some]) and not g[0][100:1000].any()
    for p, q in zip(g[1:], s[1:]):  # (sums in another order, each rounded)
        assert torch.allclose(p.float(), q.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_constant_rows_and_no_eps(cuda):
    x = torch.full((6, 40), 3.5, device=cuda, requires_grad=True)
    w, b = torch.randn(40, device=cuda), torch.randn(40, device=cuda)
    y = fastgl.layer_norm(x, w, b)
    assert torch.equal(y, b.expand(6, 40))
    g, = torch.autograd.grad(y, x, torch.randn_like(y))
    assert g.isfinite().all()
    assert fastgl.layer_norm(x, eps=0.0).isnan().all()


@pytest.mark.parametrize("keep8", [False, True])
def test_values_that_are_no_numbers_stay_in_their_row(cuda, keep8):
    x, w, b, dy = problem(cuda, 37, 100, torch.float32)
    x = x.detach().clone()
    x[3, 50], x[5, 0], x[36, 99] = float("nan"), float("inf"), -float("inf")
    x.requires_grad_()
    y = fastgl.layer_norm(x, w, b, relu=True, keep8=keep8)
    bad = torch.zeros(37, dtype=torch.bool, device=cuda)
    bad[[3, 5, 36]] = True
    assert y[bad].isnan().all() and y[~bad].isfinite().all()
    g = torch.autograd.grad(y, (x, w, b), dy)
    assert g[0][bad].isnan().all() and g[0][~bad].isfinite().all() and g[1].isnan().all() and g[2].isfinite().all()


@pytest.mark.parametrize("keep8", [False, True])
def test_which_gradients_are_asked_for(cuda, keep8):
    x, w, b, dy = problem(cuda, 300, 47, torch.float32)
    whole = torch.autograd.grad(fastgl.layer_norm(x, w, b, relu=True, keep8=keep8), (x, w, b), dy)
    for keep in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        leaves = [t.detach().clone().requires_grad_(i in keep) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(fastgl.layer_norm(*leaves, relu=True, keep8=keep8), [leaves[i] for i in keep], dy)
        assert all(torch.equal(got[j], whole[i]) for j, i in enumerate(keep))
    for weight, bias in ((None, None), (w, None), (None, b)):
        y = fastgl.layer_norm(x, weight, bias, keep8=keep8)
        ones, zeros = torch.ones_like(w).requires_grad_(), torch.zeros_like(b).requires_grad_()
        z = fastgl.layer_norm(x, ones if weight is None else weight, zeros if bias is None else bias, keep8=keep8)
        assert torch.equal(y, z) and torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(z, x, dy)[0])


def test_any_shape_order_and_gradients_from_views(cuda):
    x, w, b, dy = problem(cuda, 24, 36, torch.float32)
    y = fastgl.layer_norm(x, w, b, relu=True)
    g = torch.autograd.grad(y, (x, w, b), dy)
    for view in (x.detach().view(2, 3, 4, 36), x.detach().t().contiguous().t()):  # (another order is copied)
        v = view.requires_grad_()
        z = fastgl.layer_norm(v, w, b, relu=True)
        assert z.shape == v.shape and torch.equal(z.reshape(24, 36), y)
        gz = torch.autograd.grad(z, (v, w, b), dy.t().contiguous().t().reshape(z.shape))
        assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(gz, g))
    one = x.detach()[0].clone().requires_grad_()
    z = fastgl.layer_norm(one, w, b, relu=True)
    assert z.shape == (36,) and torch.equal(z, y[0])
    gx, = torch.autograd.grad(fastgl.layer_norm(x, w, b).sum(), x)  # (an expanded gradient)
    assert torch.equal(gx, torch.autograd.grad(fastgl.layer_norm(x, w, b), x, torch.ones_like(dy))[0])
    row = torch.randn(36, device=cuda, requires_grad=True)
    gr, = torch.autograd.grad(fastgl.layer_norm(row.expand(24, 36), w, b), row, dy)  # (24 rows that are one)

    rep = row.detach().repeat(24, 1).requires_grad_()
    ge, = torch.autograd.grad(fastgl.layer_norm(rep, w, b), rep, dy)
    assert torch.allclose(gr, ge.sum(0), rtol=1e-5, atol=1e-5)
    for shape in ((0, 36), (2, 0, 36)):
        e = torch.zeros(shape, device=cuda, requires_grad=True)
        z = fastgl.layer_norm(e, w, b, keep8=True)
        assert z.shape == shape
        ge = torch.autograd.grad(z, (e, w, b), torch.zeros(shape, device=cuda))
        assert ge[0].shape == shape and not ge[1].any() and not ge[2].any()


def test_refusals(cuda):
    x = torch.zeros((4, 8), device=cuda)
    w = torch.ones(8, device=cuda)
    for bad in (dict(x=x.half()), dict(x=x.double()), dict(weight=w[:7]), dict(weight=w.bfloat16()), dict(bias=w[None]), dict(eps=-1.0), dict(eps=float("nan")),
                dict(x=torch.zeros((2, 2049), device=cuda), weight=None), dict(x=torch.zeros((2, 0), device=cuda), weight=None), dict(x=torch.zeros((), device=cuda), weight=None),
                dict(weight=w.cpu()), dict(x=x.cpu())):
        with pytest.raises(RuntimeError):
            fastgl.layer_norm(**{**dict(x=x, weight=w), **bad})
    with pytest.raises(RuntimeError, match="columns"):
        fastgl.LayerNorm(9).to(cuda)(x)
    y = fastgl.layer_norm(x.requires_grad_(), w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(g.sum(), x)


def test_input_changed_in_between_is_an_error(cuda):
    x = torch.randn((8, 16), device=cuda, requires_grad=True)
    t = x * 1
    y = fastgl.layer_norm(t)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    t = x * 1
    y = fastgl.layer_norm(t, keep8=True)  # (nothing of it is kept)
    t.add_(1)
    y.sum().backward()


@pytest.mark.parametrize("keep8", [False, True])
def test_many_gradients_at_once(cuda, keep8):
    x, w, b, _ = problem(cuda, 9, 20, torch.float32)
    y = fastgl.layer_norm(x, w, b, relu=True, keep8=keep8)
    many = torch.randn((5, 9, 20), device=cuda)
    got = torch.autograd.grad(y, (x, w, b), many, is_grads_batched=True, retain_graph=True)
    for i in range(5):
        one = torch.autograd.grad(y, (x, w, b), many[i], retain_graph=True)
        assert all(torch.equal(p[i], q) for p, q in zip(got, one))


def test_followed_and_under_autocast(cuda):
    x, w, b, dy = problem(cuda, 30, 50, torch.float32)
    y = fastgl.layer_norm(x, w, b, relu=True)
    f = lambda t: fastgl.layer_norm(t, w, b, relu=True)  # noqa: E731
    assert torch.allclose(torch.func.vmap(f)(x.detach()), y, rtol=1e-6, atol=1e-6)
    _, tangent = torch.func.jvp(f, (x.detach(),), (dy,))
    gx, = torch.autograd.grad(y, x, dy, retain_graph=True)
    v = torch.randn_like(dy)
    gv, = torch.autograd.grad(y, x, v)
    assert torch.allclose((tangent * v).sum(), (gv * dy).sum(), rtol=1e-4, atol=1e-4) and gx.isfinite().all()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        z = fastgl.layer_norm(x.detach().bfloat16(), w, b)
    assert z.dtype == torch.float32 and torch.equal(z, fastgl.layer_norm(x.detach().bfloat16().float(), w, b))


def test_captured_on_another_stream(cuda):
    x, w, b, dy = problem(cuda, 500, 100, torch.float32)
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    step = lambda: (lambda y: (y, *torch.autograd.grad(y, (x, w, b), dy)))(fastgl.layer_norm(x, w, b, relu=True, keep8=True))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
