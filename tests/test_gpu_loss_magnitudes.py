"""fastgl.linear_cross_entropy in fp32 where magnitudes lie far apart: columns, classes and rows with values many powers of two beside the others.
Every limit is that of the terms a result is the sum of, none of a largest value of the matrix.

Limits.  u = 2^-24, M the largest sum of magnitudes sum_d |x_id w_vd| + |b_v| of a row.  A value is the sum of three bf16 values, v = h + m + l, |m| <=
2^-8 |v|, |l| <= 2^-17 |v|, exactly; of a product m l', l m' and l l' are left out, 2^-24 of it and little more.  Six instructions add up 16 columns, and
each is off by u of the sum of magnitudes: a logit is off by (c - 2) u M, c = 3 + 6 d / 16, and the bias's and the label's roundings make it c u M.  So a
share is off by eps = 4 u (c + 4) (M + 4) of itself (twice that error, with its own exponential's, for itself and for the sum that divides it) and a loss by eps
(1 + loss), where a sum of V shares adds one rounding for each tile of 32 and log-many: (V / 32 + 8) u.  A gradient is a sum of shares times values: each
term off by 2 eps of itself, twelve instructions for a tile's 32 terms, and at last a rounding: (2 eps + (12 k / 32 + 16) u) of the sum of its k terms'
magnitudes.  A share below 2^-110 has bits that bf16 does not, below 2^-126 none at all: 2^-126 times the other factor more, for each term."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [(300, 200, 64), (150, 170, 300), (140, 170, 340), (150, 270, 500), (40_000, 130, 48), (130, 40_000, 48)]


def normal(cuda, seed, *size):
    return torch.randn(size, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda)


def problem(cuda, n, v, d):
    x, w, b = normal(cuda, n + d, n, d) / 2, normal(cuda, v + d, v, d) / d ** 0.5, normal(cuda, v, v)
    y = torch.randint(0, v, (n,), generator=torch.Generator(device=cuda).manual_seed(3), device=cuda)
    return x, w, b, y


def check(x, w, b, y, reduction="none", g=None, left_out=None):
    n, d, v = x.size(0), x.size(1), w.size(0)
    if g is None:
        g = torch.rand(n if reduction == "none" else (), generator=torch.Generator(device=x.device).manual_seed(4), device=x.device) + 0.5
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction=reduction)
    grads = torch.autograd.grad(loss, leaves, g)
    if left_out is not None:  # (their gradients, none, apart; the others' as if they were not there)
        assert (grads[1][left_out] == 0).all() and (grads[2][left_out] == 0).all()
        stay = (~left_out).nonzero()[:, 0]
        name = torch.full((v,), -1, device=x.device)
        name[stay] = torch.arange(stay.numel(), device=x.device)
        w, b, y, grads, v = w[stay], b[stay], name[y], (grads[0], grads[1][stay], grads[2][stay]), stay.numel()
    X, W, B = x.double(), w.double(), b.double()
    s = X @ W.t() + B
    rows = torch.arange(n, device=x.device)
    others = (s - s[rows, y][:, None]).exp().scatter(1, y[:, None], 0.0).sum(1)
    losses = torch.log1p(others)
    p = (s - torch.logsumexp(s, 1, keepdim=True)).exp()
    p[rows, y] = torch.expm1(-losses)
    scale = g.double().expand(n) / (n if reduction == "mean" else 1)
    p *= scale[:, None]
    most = float((X.abs() @ W.abs().t() + B.abs()).max())
    eps = 4 * U * (3 + 6 * d / 16 + 4) * (most + 4) + (v / 32 + 8) * U
    assert eps < 2e-3  # (or the limits would say nothing)
    want = losses if reduction == "none" else losses.sum() / (n if reduction == "mean" else 1)
    limit = eps * (1 + losses) if reduction == "none" else eps * (1 + losses).sum() / (n if reduction == "mean" else 1)
    off = (loss.detach().double() - want).abs()
    assert (off <= limit).all(), ("loss", float((off / limit).max()))
    least = 2.0 ** -126 * float(scale.abs().max())
    for what, got, exact, terms, k, floor in (("dx", grads[0], p @ W, p.abs() @ W.abs(), v, least * W.abs().sum(0)), ("dw", grads[1], p.t() @ X, p.abs().t() @ X.abs(), n, least * X.abs().sum(0)),
                                              ("db", grads[2], p.sum(0), p.abs().sum(0), n, least * n)):
        limit = (2 * eps + (12 * k / 32 + 16) * U) * terms + U * exact.abs() + floor + 2.0 ** -126
        off = (got.double() - exact).abs()
        assert (off <= limit).all(), (what, float((off / limit).max()), float((off / (exact.abs() + 1e-300)).max()))


@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("power", [0, 20, 30, 60])
def test_one_column_of_another_scale(cuda, n, v, d, power):
    """The same logits: a column of x times 2^power, that of the weights times its inverse."""
    x, w, b, y = problem(cuda, n, v, d)
    x[:, 3] *= 2.0 ** power
    w[:, 3] *= 2.0 ** -power
    check(x, w, b, y)


@pytest.mark.parametrize("n,v,d", SIZES)
def test_columns_of_many_scales(cuda, n, v, d):
    x, w, b, y = problem(cuda, n, v, d)
    scale = 2.0 ** torch.randint(-40, 41, (d,), generator=torch.Generator(device=cuda).manual_seed(5), device=cuda).float()
    check(x * scale, w / scale, b, y, reduction="mean")


@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("size", [1e4, 1e7])
def test_classes_that_are_left_out_may_have_large_weights(cuda, n, v, d, size):
    x, w, b, y = problem(cuda, n, v, d)
    out = torch.zeros(v, dtype=torch.bool, device=cuda)
    out[0] = out[v // 2] = True
    w[out] *= size
    b[out] = float("-inf")
    y = torch.where(out[y], torch.full_like(y, 1), y)
    check(x, w, b, y, left_out=out)


@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("size", [1e5, 1e9])
def test_a_large_weight_of_a_class_of_small_share(cuda, n, v, d, size):
    x, w, b, y = problem(cuda, n, v, d)
    x[:, 5] = 0.0
    w[1, 5] = size
    b[1] = -26.0
    check(x, w, b, torch.where(y == 1, torch.full_like(y, 2), y))


@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("size", [1e6, 1e9])
def test_a_large_value_of_one_row(cuda, n, v, d, size):
    x, w, b, y = problem(cuda, n, v, d)
    w[:, 5] = 0.0
    x[1, 5] = size
    check(x, w, b, y)


@pytest.mark.parametrize("n,v,d", SIZES)
@pytest.mark.parametrize("power", [-90, 60])
def test_gradients_of_losses_of_any_magnitude(cuda, n, v, d, power):
    x, w, b, y = problem(cuda, n, v, d)
    check(x, w, b, y, g=normal(cuda, 6, n) * 2.0 ** power)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [40, 300, 500])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), 1e30])
def test_what_classes_that_are_left_out_hold_is_nobodys_matter(cuda, dtype, d, what):
    """A table of classes that is longer than what it holds: the same bits as with zeros there."""
    x, w, b, y = problem(cuda, 150, 170, d)
    out = torch.arange(170, device=cuda) % 5 == 1
    out[128:] = True  # (a whole tile and the last ones)
    y = torch.where(out[y], torch.full_like(y, 2), y)
    for bias in (float("-inf"), torch.finfo(dtype).min):
        results = []
        for fill in (0.0, what):
            leaves = [t.to(dtype).detach() for t in (x, torch.where(out[:, None], fill, w), torch.where(out, bias, b))]
            for t in leaves:
                t.requires_grad_()
            loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
            results.append([loss.detach(), *torch.autograd.grad(loss, leaves), fastgl.linear_cross_entropy(*(t.detach() for t in leaves[:2]), y, leaves[2].detach())])
        assert all(torch.isfinite(t).all() and torch.equal(t, u) for t, u in zip(*results))
        assert (results[1][2][out] == 0).all() and (results[1][3][out] == 0).all()


@pytest.mark.parametrize("n,v,d", [(12_900, 230, 340), (230, 12_900, 500), (20_000, 3000, 400), (3000, 20_000, 330), (1, 1, 321), (65, 33, 512), (70_000, 40, 450), (33, 100_000, 350)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_many_columns_in_whole_and_in_cut_groups(cuda, n, v, d, reduction):
    """Two waves share their rows from 321 columns on: groups that a workgroup has alone, that several share, and that are cut anywhere."""
    print("linear_cross_entropy %d x %d, %d classes" % (n, d, v), flush=True)
    check(*problem(cuda, n, v, d), reduction=reduction)


@pytest.mark.parametrize("d", [330, 500])
def test_many_columns_captured_and_replayed(cuda, d):
    x, w, b, y = problem(cuda, 900, 700, d)
    y[::5] = -100
    held, one = [x.clone(), w.clone(), b.clone()], torch.ones((), device=cuda)

    def step():
        leaves = [t.detach().requires_grad_() for t in held]
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
        return loss.detach(), *torch.autograd.grad(loss, leaves, one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        for t, u in zip(held, (x, w, b)):
            t.copy_(u * (1 + k / 2))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
