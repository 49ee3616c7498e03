"""fastgl.linear against its formulas in 64 bits: the output and all gradients, for each activation, with and without bias and residual, with the input kept
in full and in 8 bits."""
import numpy as np
import pytest
import torch

import fastgl
from held8 import held

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24
ERF = 1.5e-7  # the error function's, absolute


def normal_cdf(z):
    return 0.5 * torch.erfc(-torch.from_numpy(z) / 2 ** 0.5).numpy()


def act_of(z, act):
    """act(z) and its derivative."""
    if act is None:
        return z, np.ones_like(z)
    if act == "relu":
        return np.maximum(z, 0), (z > 0).astype(z.dtype)
    if act == "gelu":
        p = normal_cdf(z)
        return z * p, p + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    p = 1 / (1 + np.exp(-z))
    return z * p, p * (1 + z * (1 - p))


def check(x, w, b, r, dy, act, keep8, y, grads):
    """A sum of d products is off by (d + 8) U of the sum of magnitudes.  The activations' slopes are at most 1.13 and change by at most 0.8 times what z does (relu's
    by 1 where z is nearer to zero than it is off); the functions themselves are off by 4 U, gelu by ERF, of |z|, the slopes by 8 U, gelu's by ERF.  In bf16 the
    slope is taken of the rounded z, and dz is rounded."""
    dtype = x.dtype
    half = HALF[dtype]
    X, W, DY = (t.detach().cpu().double().numpy() for t in (x, w, dy))
    n, d, out = X.shape[0], X.shape[1], W.shape[0]
    B = np.zeros(out) if b is None else b.detach().cpu().double().numpy()
    R = np.zeros((n, out)) if r is None else r.detach().cpu().double().numpy()
    z = X @ W.T + B
    off = (d + 8) * U * (np.abs(X) @ np.abs(W).T + np.abs(B))
    value, slope = act_of(z, act)
    want = value + R
    bound = 1.13 * off + (8 * U + (ERF if act == "gelu" else 0)) * np.abs(z) + U * np.abs(want) + half * np.abs(want)
    far = np.abs(y.detach().cpu().double().numpy() - want) - bound
    assert (far <= 0).all(), ("y", far.max())
    if act is None:
        dz, dz_off = DY, np.zeros_like(DY)
    else:
        dz = DY * slope
        if act == "relu":
            s_off = (np.abs(z) <= off).astype(float)
        else:
            s_off = 0.8 * (off + (half * np.abs(z) if dtype == torch.bfloat16 else U * np.abs(z))) + 8 * U * (1 + np.abs(z)) + (ERF if act == "gelu" else 0)
        dz_off = np.abs(DY) * s_off + half * np.abs(dz)
    names = ["x", "w"] + ([] if b is None else ["b"]) + ([] if r is None else ["r"])
    H = held(X) if keep8 else X
    for name, g in zip(names, grads):
        assert g.dtype == dtype
        g = g.detach().cpu().double().numpy()
        if name == "x":
            e, o = dz @ W, dz_off @ np.abs(W) + (out + 8) * U * (np.abs(dz) @ np.abs(W))
        elif name == "w":
            e, o = dz.T @ H, dz_off.T @ np.abs(H) + (n + 8) * U * (np.abs(dz).T @ np.abs(H))
        elif name == "b":
            e, o = dz.sum(0), dz_off.sum(0) + (n + 8) * U * np.abs(dz).sum(0)
        else:
            e, o = DY, 0.0
        far = np.abs(g - e) - (o * (1 + half) + half * np.abs(e))
        assert g.shape == e.shape and (far <= 0).all(), (name, far.max())


def problem(cuda, n, d, out, dtype, bias=True, residual=False, stride=None):
    gen = torch.Generator(device=cuda).manual_seed(n + 31 * d + 7 * out)
    normal = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    x = normal(n, stride or d).to(dtype)[:, :d].requires_grad_()
    w = (normal(out, d) / d ** 0.5).to(dtype).requires_grad_()
    b = (0.3 * normal(out)).to(dtype).requires_grad_() if bias else None
    r = normal(n, out).to(dtype).requires_grad_() if residual else None
    return x, w, b, r, normal(n, out).to(dtype)


SIZES = [(1, 1, 1), (2, 3, 5), (33, 47, 31), (100, 64, 47), (257, 100, 256), (64, 33, 129), (1000, 256, 64), (8000, 100, 256), (4100, 602, 64), (130, 512, 513), (17, 1025, 40),
         (2500, 256, 300), (5000, 130, 66), (40_000, 64, 128), (3001, 416, 96), (40_001, 33, 62)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,out", SIZES)
def test_values_and_gradients(cuda, dtype, act, keep8, n, d, out):
    bias, residual = (n + d) % 3 != 0, (d + out) % 2 == 0
    x, w, b, r, dy = problem(cuda, n, d, out, dtype, bias, residual, stride=d + (n % 3))
    y = fastgl.linear(x, w, b, activation=act, residual=r, keep8=keep8)
    assert y.shape == (n, out) and y.dtype == dtype and y.is_contiguous()
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    check(x, w, b, r, dy, act, keep8, y, grads)
    with torch.no_grad():
        assert torch.equal(fastgl.linear(x, w, b, activation=act, residual=r), y)


# bf16 with the weights kept on the CUs, from 3.3 M outputs on (and 100 K rows where k is short): columns and lanes at the ends of tiles, vectors and pairs, k at the ends of a piece of 8 and a chunk of 64, and as
# long as 128, 64 and 32 columns of weights have room
@pytest.mark.parametrize("act", [None, "relu", "gelu"])
@pytest.mark.parametrize("n,d,out", [(100_000, 16, 64), (100_193, 17, 129), (120_000, 47, 33), (110_255, 64, 30), (26_999, 640, 128), (20_200, 641, 132), (26_000, 1216, 62), (26_192, 1217, 60),
                                     (26_300, 2400, 24), (12_321, 96, 260), (26_999, 128, 127), (50_001, 104, 68), (60_000, 512, 256), (30_000, 4096, 8), (26_193, 15, 40), (140_001, 100, 40)])
def test_many_rows_in_bf16(cuda, act, n, d, out):
    x, w, b, r, dy = problem(cuda, n, d, out, torch.bfloat16, True, out % 4 != 1, stride=d + d % 2 + 2 * (n % 2))
    y = fastgl.linear(x, w, b, activation=act, residual=r)
    check(x, w, b, r, dy, act, False, y, torch.autograd.grad(y, [t for t in (x, w, b, r) if t is not None], dy))


def test_offsets_beyond_32_bits(cuda):
    n = (1 << 32) // 256 + 70
    w, b = torch.randn((256, 16), device=cuda).bfloat16().requires_grad_(), torch.randn(256, device=cuda).bfloat16().requires_grad_()
    x = torch.randn((n, 16), device=cuda).bfloat16().requires_grad_()
    y = fastgl.linear(x, w, b, "relu", keep8=True)
    d = torch.zeros((n, 256), device=cuda, dtype=torch.bfloat16)
    some = torch.cat([torch.arange(40), torch.arange(n - 90, n)]).to(cuda)
    d[some] = torch.randn((130, 256), device=cuda).bfloat16()
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), d)
    xs = x.detach()[some].clone().requires_grad_()
    ys = fastgl.linear(xs, w, b, "relu", keep8=True)
    assert torch.equal(ys, y[some])
    sx, sw, sb = torch.autograd.grad(ys, (xs, w, b), d[some])
    assert torch.equal(sx, gx[some]) and not gx[100:1000].any()
    for p, q in ((gw, sw), (gb, sb)):  # (sums in another order, each rounded)
        assert torch.allclose(p.float(), q.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_from_several_threads_on_streams_of_their_own(cuda):
    import threading

    x, w, b, r, dy = problem(cuda, 9000, 100, 130, torch.float32, True, True)
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, (x, w, b, r), dy)))(fastgl.linear(x, w, b, "gelu", r, keep8=True))  # noqa: E731
    want = step()
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = [step() for _ in range(5)]
            torch.cuda.current_stream().synchronize()
        results[i] = out

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(p, q) for out in results for one in out for p, q in zip(one, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("keep8", [False, True])
def test_the_same_on_every_run_and_which_gradients_are_asked_for(cuda, dtype, act, keep8):
    x, w, b, r, dy = problem(cuda, 3000, 100, 130, dtype, True, True)
    leaves = [x, w, b, r]
    whole = torch.autograd.grad(fastgl.linear(x, w, b, act, r, keep8), leaves, dy)
    for keep in ((0, 1, 2, 3), (0,), (1,), (2,), (3,), (0, 2), (1, 3), (0, 3)):
        some = [t.detach().clone().requires_grad_(i in keep) for i, t in enumerate(leaves)]
        got = torch.autograd.grad(fastgl.linear(some[0], some[1], some[2], act, some[3], keep8), [some[i] for i in keep], dy)
        assert all(torch.equal(got[j], whole[i]) for j, i in enumerate(keep)), keep


def test_any_shape_order_and_gradients_from_views(cuda):
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, r, dy = problem(cuda, 24, 35, 33, dtype, True, True)
        y = fastgl.linear(x, w, b, "relu", r)
        g = torch.autograd.grad(y, (x, w, b, r), dy)
        for lead in ((2, 3, 4), (24,)):
            v = x.detach().reshape(*lead, 35).requires_grad_()
            s = r.detach().reshape(*lead, 33).requires_grad_()
            z = fastgl.linear(v, w, b, "relu", s)
            assert z.shape == (*lead, 33) and torch.equal(z.reshape(24, 33), y)
            gz = torch.autograd.grad(z, (v, w, b, s), dy.reshape(z.shape))
            assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(gz, g))
        turned = [t.detach().t().contiguous().t().requires_grad_() for t in (x, w, r)]
        z = fastgl.linear(turned[0], turned[1], b, "relu", turned[2])
        gz = torch.autograd.grad(z, (turned[0], turned[1], b, turned[2]), dy.t().contiguous().t())
        assert torch.equal(z, y) and all(torch.equal(p, q) for p, q in zip(gz, g))
        gs, = torch.autograd.grad(fastgl.linear(x, w, b).sum(), x)  # (an expanded gradient)
        assert torch.equal(gs, torch.autograd.grad(fastgl.linear(x, w, b), x, torch.ones_like(dy))[0])
        one = fastgl.linear(x.detach()[3], w, b, "relu", r.detach()[3])
        assert one.shape == (33,) and torch.equal(one, fastgl.linear(x.detach()[3:4], w, b, "relu", r.detach()[3:4])[0])
        for keep8 in (False, True):
            e = torch.zeros((0, 35), device=cuda, dtype=dtype, requires_grad=True)
            z = fastgl.linear(e, w, b, "gelu", keep8=keep8)
            ge = torch.autograd.grad(z, (e, w, b), torch.zeros((0, 33), device=cuda, dtype=dtype))
            assert z.shape == (0, 33) and ge[0].shape == (0, 35) and not ge[1].any() and not ge[2].any()


def test_gradients_are_those_of_differences(cuda):
    """y along a direction, forward by two steps in 64 bits of the formula's arguments, against the gradient's product with it."""
    for act in ("gelu", "silu"):
        x, w, b, r, dy = problem(cuda, 40, 30, 20, torch.float32, True, True)
        y = fastgl.linear(x, w, b, act, r)
        grads = torch.autograd.grad(y, (x, w, b, r), dy)
        for i, t in enumerate((x, w, b, r)):
            v = torch.randn_like(t)
            h = 2.0 ** -8
            moved = [[u.detach() + (s * h * v if j == i else 0) for j, u in enumerate((x, w, b, r))] for s in (1, -1)]
            up, down = (fastgl.linear(m[0], m[1], m[2], act, m[3]).double() for m in moved)
            slope, want = float(((up - down) / (2 * h) * dy).sum()), float((grads[i].double() * v).sum())
            # rounding: 2^-24 of values below 8 over 2 h, 800 of them times dy; the third derivative (below 2) times h^2 / 6
            size = float(dy.abs().sum())
            third = 2 * h * h / 6 * size * float((v.abs().max() * (1 + w.abs().sum(1).max())) ** 3)
            assert abs(slope - want) < 8 * 2.0 ** -24 / h * size + third


@pytest.mark.parametrize("keep8", [False, True])
def test_values_that_are_no_numbers(cuda, keep8):
    x, w, b, r, dy = problem(cuda, 300, 70, 40, torch.float32, True, False)
    x = x.detach().clone()
    x[7, 33], x[200, 2] = float("nan"), float("inf")
    x.requires_grad_()
    for act in (None, "relu", "gelu"):
        y = fastgl.linear(x, w, b, act, keep8=keep8)
        bad = torch.zeros(300, dtype=torch.bool, device=cuda)
        bad[[7, 200]] = True
        assert y[7].isnan().all() and not y[200].isfinite().all() and y[~bad].isfinite().all()
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
        assert gx[~bad].isfinite().all()
        columns = torch.ones(70, dtype=torch.bool, device=cuda)
        if keep8:  # (32 columns are held together)
            columns[32:64] = columns[:32] = False
        else:
            columns[[33, 2]] = False
        if act is None:
            assert gw[:, columns].isfinite().all() and gb.isfinite().all()
        assert not gw[:, ~columns].isfinite().any()


@pytest.mark.parametrize("n", [300, 27_000])
@pytest.mark.parametrize("d", [96, 100, 129, 250])
def test_infinite_values_in_bf16(cuda, n, d):
    """A row with one infinite value is infinite by its weights' signs, wherever in the row that is, and its gradient's by theirs."""
    x, w, b, r, dy = problem(cuda, n, d, 130, torch.bfloat16, True, False)
    x, dy, w = x.detach().clone(), dy.clone(), w.detach().clone()
    w[w.abs() < 2.0 ** -10] = 0.5
    places = [(0, d - 1), (1, d - 2), (70, d - 8), (133, 0), (n - 1, d - 5)]
    for row, c in places:
        x[row, c] = float("inf")
        dy[row, 130 - d + c if c > d - 10 else 0] = float("-inf")
    x.requires_grad_()
    y = fastgl.linear(x, w, b)
    z = fastgl.linear(x, w, b, "relu")
    gx, = torch.autograd.grad(y, x, dy)
    bad = torch.zeros(n, dtype=torch.bool, device=cuda)
    for row, c in places:
        assert torch.equal(y[row].float(), float("inf") * w[:, c].sign().float())
        assert torch.equal(z[row].float(), torch.where(w[:, c] > 0, float("inf"), 0.0))
        assert torch.equal(gx[row].float(), float("-inf") * w[130 - d + c if c > d - 10 else 0].sign().float())
        bad[row] = True
    assert y[~bad].isfinite().all() and gx[~bad].isfinite().all()


@pytest.mark.parametrize("act", [None, "silu"])
def test_magnitudes_that_have_no_three_parts(cuda, act):
    """Gradients below 2^-110 and rows of zeros beside large ones, kept in 8 bits: each sum to its own terms' precision."""
    x, w, b, r, dy = problem(cuda, 4000, 96, 64, torch.float32, True, False)
    dy = dy.clone()
    dy[:, 5] *= 2.0 ** -115
    dy[:, 9] *= 2.0 ** 60
    dy[100:200] = 0
    x = x.detach().clone()
    x[:, 64:] *= 2.0 ** -100
    x[:, :32] = 0
    x.requires_grad_()
    y = fastgl.linear(x, w, b, act, keep8=True)
    gw, gb = torch.autograd.grad(y, (w, b), dy)
    H = held(x.detach().cpu().double().numpy())
    z = x.detach().cpu().double().numpy() @ w.detach().cpu().double().numpy().T + b.detach().cpu().double().numpy()
    slope = act_of(z, act)[1]
    dz = dy.cpu().double().numpy() * slope
    e, o = dz.T @ H, (4008 * U + 1e-5) * (np.abs(dz).T @ np.abs(H)) + 2.0 ** -149
    assert (np.abs(gw.cpu().double().numpy() - e) <= o).all()
    assert (gw[:, :32] == 0).all()


def test_refusals(cuda):
    x, w = torch.zeros((4, 8), device=cuda), torch.zeros((5, 8), device=cuda)
    for bad in (dict(x=x.half()), dict(x=x.bfloat16()), dict(weight=w[:, :7]), dict(weight=w[0]), dict(bias=torch.zeros(4, device=cuda)), dict(bias=torch.zeros(5)),
                dict(bias=torch.zeros(5, device=cuda).bfloat16()), dict(activation="tanh"), dict(residual=torch.zeros((4, 4), device=cuda)),
                dict(residual=torch.zeros((1, 5), device=cuda)), dict(residual=torch.zeros((4, 5), device=cuda).double()), dict(x=x.cpu()), dict(weight=torch.zeros((0, 8), device=cuda)),
                dict(weight=torch.zeros((4097, 8), device=cuda)), dict(x=torch.zeros((4, 0), device=cuda), weight=torch.zeros((5, 0), device=cuda))):
        with pytest.raises(RuntimeError):
            fastgl.linear(**{**dict(x=x, weight=w), **bad})
    y = fastgl.linear(x.requires_grad_(), w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(g.sum(), x)
    r = torch.zeros((4, 5), device=cuda, requires_grad=True)
    v = torch.ones((4, 5), device=cuda, requires_grad=True)
    d, = torch.autograd.grad(fastgl.linear(x, w, residual=r), r, v, create_graph=True)
    assert torch.equal(torch.autograd.grad(d.sum(), v)[0], torch.ones_like(v))  # (the residual's are the output's own)


def test_input_changed_in_between_is_an_error(cuda):
    x, w, b, _, dy = problem(cuda, 8, 16, 4, torch.float32)
    t = x * 1
    y = fastgl.linear(t, w, b)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(dy)
    t = x * 1
    y = fastgl.linear(t, w, b, keep8=True)  # (nothing of it is kept)
    t.add_(1)
    y.backward(dy)


@pytest.mark.parametrize("keep8", [False, True])
def test_many_gradients_at_once(cuda, keep8):
    x, w, b, r, _ = problem(cuda, 9, 20, 6, torch.float32, True, True)
    y = fastgl.linear(x, w, b, "gelu", r, keep8)
    many = torch.randn((5, 9, 6), device=cuda)
    got = torch.autograd.grad(y, (x, w, b, r), many, is_grads_batched=True, retain_graph=True)
    for i in range(5):
        one = torch.autograd.grad(y, (x, w, b, r), many[i], retain_graph=True)
        assert all(torch.equal(p[i], q) for p, q in zip(got, one))


def test_followed_and_under_autocast(cuda):
    x, w, b, r, dy = problem(cuda, 30, 50, 20, torch.float32, True, True)
    for act in (None, "relu", "gelu", "silu"):
        y = fastgl.linear(x, w, b, act, r)
        f = lambda t: fastgl.linear(t, w, b, act, r)  # noqa: E731
        _, tangent = torch.func.jvp(f, (x.detach(),), (torch.ones_like(x),))
        gx, = torch.autograd.grad(y, x, dy)
        assert torch.allclose((tangent * dy).sum(), gx.sum(), rtol=1e-3, atol=1e-3)
    assert torch.allclose(torch.func.vmap(lambda t, s: fastgl.linear(t, w, b, "silu", s))(x.detach(), r.detach()), fastgl.linear(x, w, b, "silu", r), rtol=1e-5, atol=1e-5)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        z = fastgl.linear(x, w, b, "relu", r)
    half = [t.detach().bfloat16() for t in (x, w, b, r)]
    assert z.dtype == torch.bfloat16 and torch.equal(z, fastgl.linear(half[0], half[1], half[2], "relu", half[3]))


def test_captured_on_another_stream(cuda):
    x, w, b, r, dy = (None if t is None else t.detach().requires_grad_(i < 4) for i, t in enumerate(problem(cuda, 3000, 100, 130, torch.float32, True, True)))

    def step():
        y = fastgl.linear(x, w, b, "relu", r, keep8=True)
        return (y, *torch.autograd.grad(y, (x, w, b, r), dy))

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
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
