"""fastgl.linear_cross_entropy against the definition in float64.

Tolerances.  Let u = 2^-24 and M the largest sum of magnitudes sum_d |x_id w_vd| + |b_v| of a row.  bf16: products are exact, and added up one
instruction of 16 columns after another: a logit is off by at most c u M, c = 2 + d / 16.  fp32: a value is taken as the sum of two fp16 values, off by
2^-22 of it (half a step of the second, 2^-11, times 2^-11 for the first), and the product of the two second parts, 2^-22, is left out: 3 * 2^-22 = 12 u of
each product; three instructions for 16 columns: c = 14 + 3 d / 16.  A value whose scaled second part is below fp16's normal numbers is off by
2^-25 of 2^-14 times the matrix's largest: 2^-39 of it, once for either factor: 2^-38 d max|x| max|w| more.  The exponentials are off by 2 u and by u
times their argument in powers of two, at most 2 M log2(e), more.  So a share p is off by eps = 4 u (c + 4) (M + 4) of itself and a loss by eps, and a sum
of n shares adds one rounding for each tile of 32 and log-many: (n / 32 + 8) u.  Gradients are sums of p times finite values: bf16: p is
rounded, 2^-8 more of each term; fp32: 3 * 2^-22 more and six instructions for a tile's 32 terms, (6 n / 32 + 8) u, and as p is scaled by its row's largest, or by sixteen times that, 2^-25 of 2^-14 of those:
2^-35 of the largest term's p, times the largest value, for each term.  At last half a step of the result."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def definition(x, w, b, y, ignore, reduction, g):
    """(loss, dx, dw, db) in 64 bits, and the sums of the magnitudes of the gradients' terms."""
    x, w = x.detach().double(), w.detach().double()
    s = x @ w.t()
    if b is not None:
        s = s + b.detach().double()
    valid = y != ignore
    label = torch.where(valid, y, torch.zeros_like(y)).long()
    rows = torch.arange(x.size(0), device=x.device)
    log_p = s - torch.logsumexp(s, 1, keepdim=True)
    # (in 64 bits too, a loss of e^-30 has few bits left as a difference of logits)
    others = (s - s[rows, label][:, None]).exp().scatter(1, label[:, None], 0.0).sum(1)
    own = torch.where(others < 1e100, torch.log1p(others), -log_p[rows, label])
    losses = torch.where(valid, own, 0.0)
    count = valid.sum()
    loss = losses if reduction == "none" else losses.sum() / (count if reduction == "mean" else 1)
    d = log_p.exp()
    d[rows, label] = torch.expm1(-own)
    d *= torch.where(valid, g.double() / (count if reduction == "mean" else 1), 0.0)[:, None] if reduction != "none" else torch.where(valid, g.double(), 0.0)[:, None]
    d[~valid] = 0.0
    # of the gradients' terms: the sums of their magnitudes, and the largest of a row times the largest value that p meets
    sums = d.abs() @ w.abs(), d.abs().t() @ x.abs(), d.abs().sum(0)
    largest = (d.abs().amax(1)[:, None] * w.abs().max(), d.abs().amax(0)[:, None] * x.abs().max(), 0.0) if min(d.shape) else (0.0, 0.0, 0.0)
    return (losses, loss, d @ w, d.t() @ x, d.sum(0)), sums, largest


def share_error(x, w, b, n_terms):
    u, d = 2.0 ** -24, x.size(1)
    # (magnitudes of a few thousand classes at a time)
    most = max(float((x.detach().abs().double() @ w.detach()[k:k + 4096].abs().double().t()).max()) for k in range(0, w.size(0), 4096))
    if b is not None:
        most += float(b.detach().double().abs().masked_fill(b.detach().isinf(), 0.0).max())
    c = 14 + 3 * d / 16 if x.dtype == torch.float32 else 2 + d / 16
    scaled = 2.0 ** -38 * d * float(x.detach().abs().max()) * float(w.detach().abs().max()) if x.dtype == torch.float32 else 0.0
    return 4 * u * (c + 4) * (most + 4) + (n_terms / 32 + 8) * u + 4 * scaled


def check(x, w, b, y, reduction="mean", ignore=-100, g=None, limit_scale=1.0):
    gen = torch.Generator(device=x.device).manual_seed(1)
    n = x.size(0)
    if g is None:
        g = torch.rand(n if reduction == "none" else (), generator=gen, device=x.device) + 0.5
    leaves = [t.detach().requires_grad_() for t in (x, w) + (() if b is None else (b,))]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2] if b is not None else None, ignore, reduction)
    assert loss.dtype == torch.float32 and loss.shape == ((n,) if reduction == "none" else ())
    grads = torch.autograd.grad(loss, leaves, g)
    (losses, want, *want_grads), sums, largest = definition(x, w, b, y, ignore, reduction, g)
    eps = share_error(x, w, b, w.size(0))
    loss_limit = eps * (1 + losses) if reduction == "none" else eps * (1 + losses.max()) * (n if reduction == "sum" else 1)
    assert ((loss.detach().double() - want).abs() <= loss_limit).all(), float((loss.detach().double() - want).abs().max())
    half = HALF[x.dtype]
    for name, got, exact, total, most in zip(("dx", "dw", "db"), grads, want_grads, sums, largest):
        assert got.dtype == x.dtype and got.shape == exact.shape
        terms = n if name != "dx" else w.size(0)
        limit = (2 * eps + ((6 if x.dtype == torch.float32 else 2) * terms / 32 + 16) * 2.0 ** -24 + (half if x.dtype == torch.bfloat16 else 12 * half)) * total + half * exact.abs() + 2.0 ** -120
        if x.dtype == torch.float32:
            limit = limit + terms * 2.0 ** -35 * most
        off = (got.double() - exact).abs()
        assert (off <= limit).all(), (name, float((off / limit).max()))
    with torch.no_grad():  # nobody records: the loss alone
        alone = fastgl.linear_cross_entropy(x, w, y, b, ignore, reduction)
    assert ((alone.double() - want).abs() <= loss_limit).all()
    return loss.detach(), grads


def make(cuda, n, v, d, dtype, bias=True, ignored=0.2, seed=0, label_dtype=torch.int64):
    gen = torch.Generator(device=cuda).manual_seed(seed + n + 7 * v + 31 * d)
    normal = lambda *size: torch.randn(size, generator=gen, device=cuda)  # noqa: E731
    w = normal(v, d) / d ** 0.5
    y = torch.randint(0, v, (n,), generator=gen, device=cuda)
    x = normal(n, d) + w[y] * 8 * torch.rand((n, 1), generator=gen, device=cuda)
    y = torch.where(torch.rand(n, generator=gen, device=cuda) < ignored, torch.full_like(y, -100), y)
    if ignored < 1:
        y[0] = v - 1
    return x.to(dtype), w.to(dtype), normal(v).to(dtype) if bias else None, y.to(label_dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 2, 3), (2, 33, 31), (31, 32, 32), (33, 31, 33), (100, 47, 64), (128, 64, 65), (129, 129, 96), (257, 172, 100), (64, 1000, 128),
                                   (300, 161, 160), (500, 300, 192), (96, 4097, 200), (1000, 47, 256), (40, 500, 257), (70, 333, 300), (130, 100, 384), (33, 700, 400),
                                   (200, 65, 512), (150, 140, 350), (90, 1000, 288), (5, 20011, 64), (4100, 5, 16), (2500, 2100, 48),
                                   (12900, 230, 300), (230, 12900, 300), (40_000, 500, 250), (500, 90_000, 250), (33_000, 70, 30)])
def test_losses_and_gradients(cuda, dtype, n, v, d):
    print("linear_cross_entropy %d x %d, %d classes, %s" % (n, d, v, dtype), flush=True)
    check(*make(cuda, n, v, d, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("label_dtype", [torch.int32, torch.int64])
def test_reductions_biases_and_labels(cuda, dtype, reduction, bias, label_dtype):
    check(*make(cuda, 150, 75, 70, dtype, bias=bias, label_dtype=label_dtype), reduction=reduction)
    x, w, b, y = make(cuda, 60, 75, 70, dtype, bias=bias, label_dtype=label_dtype, ignored=0.0)
    y[3:9] = 7
    check(x, w, b, y, reduction=reduction, ignore=7)
    g = torch.randn(60, device=cuda) if reduction == "none" else torch.tensor(-3.0, device=cuda)
    check(x, w, b, y, reduction=reduction, ignore=-1, g=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(cuda, dtype):
    x, w, b, y = make(cuda, 77, 90, 45, dtype)
    want_loss, want = check(x, w, b, y)
    wide = torch.zeros((77, 61), dtype=dtype, device=cuda)
    wide[:, 3:48] = x
    for xs in (wide[:, 3:48], x.t().contiguous().t()):
        for ws in (w.t().contiguous().t(), torch.stack([w, w], 2)[:, :, 0]):
            loss, grads = check(xs, ws, b, y)
            assert torch.equal(loss, want_loss) and all(torch.equal(p, q) for p, q in zip(grads, want))
    row = x[5:6].expand(77, 45)  # (one row many times)
    check(row, w, b, y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_some_gradients(cuda, dtype):
    x, w, b, y = make(cuda, 90, 200, 64, dtype)
    _, (dx, dw, db) = check(x, w, b, y)
    for needs in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), needs)]
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
        gen = torch.Generator(device=cuda).manual_seed(1)
        loss.backward(torch.rand((), generator=gen, device=cuda) + 0.5)
        for t, k, want in zip(leaves, needs, (dx, dw, db)):
            assert t.grad is None if not k else torch.equal(t.grad, want)


def test_two_backward_passes_and_no_third_order(cuda):
    x, w, b, y = make(cuda, 90, 200, 64, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    twice = torch.autograd.grad(loss, leaves, torch.tensor(2.0, device=cuda), retain_graph=True)
    again = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(2 * p, q) for p, q in zip(first, twice)) and all(torch.equal(p, q.detach()) for p, q in zip(first, again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(again[0].sum(), leaves)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_certain_of_their_label_keep_their_bits(cuda, dtype):
    # every loss about e^-20: a difference of logits would have none of its bits
    x, w, _, y = make(cuda, 64, 40, 32, dtype, bias=False, ignored=0.0)
    x = (w[y].float() / w[y].float().square().sum(1, keepdim=True) * 24).to(dtype)
    w = (w.float() * 0.2).to(dtype)
    for r in range(64):
        w[y[r]] = (x[r].float() / 24 ).to(dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    losses = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, reduction="none")
    g = torch.ones(64, device=cuda)
    dx, = torch.autograd.grad(losses, leaves[:1], g)
    (exact, _, want, _, _), (total, _, _), (largest, _, _) = definition(x, w, None, y, -100, "none", g)
    eps = share_error(x, w, None, 40)
    small = exact < 1e-3
    assert int(small.sum()) > 8
    assert ((losses.detach().double() - exact).abs()[small] <= 3 * eps * exact[small]).all()
    assert ((dx.double() - want).abs()[small] <= (3 * eps + (2 if dtype == torch.bfloat16 else 14) * HALF[dtype]) * total[small] + HALF[dtype] * want.abs()[small] + 40 * 2.0 ** -35 * largest[small] + 2.0 ** -120).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lowest", [True, False])
def test_masked_classes(cuda, dtype, lowest):
    x, w, b, y = make(cuda, 70, 300, 40, dtype, ignored=0.0)
    off = torch.arange(300, device=cuda) % 3 == 1
    off[:64] = True  # (whole tiles, the first among them)
    y = torch.where(off[y], torch.full_like(y, 68), y)
    assert not off[68]
    b = torch.where(off, torch.full_like(b, torch.finfo(dtype).min if lowest else float("-inf")), b)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    kept = (~off).nonzero()[:, 0]
    names = torch.full((300,), -1, device=cuda, dtype=torch.int64)
    names[kept] = torch.arange(kept.numel(), device=cuda)
    (_, want, dx, dw, db), (tx, tw, tb), largest = definition(x, w[kept], b[kept], names[y], -100, "mean", torch.ones((), device=cuda))
    eps = share_error(x, w[kept], b[kept], 300)
    assert abs(float(loss.detach()) - float(want)) <= eps * (1 + 2 * float(want) + 8)
    for got, exact, total, most in zip((grads[0], grads[1][kept], grads[2][kept]), (dx, dw, db), (tx, tw, tb), largest):
        assert ((got.double() - exact).abs() <= (2 * eps + (2 if dtype == torch.bfloat16 else 14) * HALF[dtype]) * total + HALF[dtype] * exact.abs() + 300 * 2.0 ** -35 * most + 1e-30).all()
    assert (grads[1][off] == 0).all() and (grads[2][off] == 0).all()
    # a label that is left out
    y2 = y.clone()
    y2[0] = 0
    loss = fastgl.linear_cross_entropy(x, w, y2, b, reduction="none")
    assert float(loss[0]) == float("inf") and torch.isfinite(loss[1:]).all()
    # no class that is not
    assert fastgl.linear_cross_entropy(x, w, y, torch.full_like(b, float("-inf")), reduction="none").isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_labels_and_bad_ones(cuda, dtype):
    x, w, b, y = make(cuda, 50, 30, 20, dtype, ignored=0.0)
    none = torch.full_like(y, -100)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], none, leaves[2])
    assert torch.isnan(loss)
    assert all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
    assert float(fastgl.linear_cross_entropy(x, w, none, b, reduction="sum")) == 0
    bad = y.clone()
    bad[7], bad[9] = 30, -3
    losses = fastgl.linear_cross_entropy(x, w, bad, b, reduction="none")
    assert losses.isnan().nonzero()[:, 0].tolist() == [7, 9]
    # a row that is not a number is the row's matter in the losses and in dx, an ignored one nobody's
    x2 = x.clone()
    x2[4] = float("nan")
    leaves = [t.detach().requires_grad_() for t in (x2, w, b)]
    losses = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="none")
    assert losses.isnan().nonzero()[:, 0].tolist() == [4]
    dx, dw = torch.autograd.grad(losses.sum(), leaves[:2])
    assert dx.isnan().any(1).nonzero()[:, 0].tolist() == [4] and dw.isnan().all()
    # nothing at all
    for reduction, want in (("none", []), ("sum", 0.0)):
        leaves = [t.detach().requires_grad_() for t in (x[:0], w, b)]
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y[:0], leaves[2], reduction=reduction)
        assert loss.tolist() == want
        dx, dw, db = torch.autograd.grad(loss.sum(), leaves)
        assert dx.shape == (0, 20) and (dw == 0).all() and (db == 0).all()
    assert torch.isnan(fastgl.linear_cross_entropy(x[:0], w, y[:0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_against_differences(cuda, dtype):
    x, w, b, y = make(cuda, 9, 12, 7, torch.float32, ignored=0.1)
    leaves = [t.to(dtype).detach().requires_grad_() for t in (x, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    h = 2.0 ** -3  # (central differences of third order: off by h^4 / 30 times a fifth derivative of the order of the gradients' own scale)
    for t, g in zip(leaves, grads):
        flat = t.detach().reshape(-1)
        for i in range(0, flat.numel(), 5):
            def at(step):
                moved = [u.detach().double() for u in leaves]
                k = [u is t for u in leaves].index(True)
                moved[k].reshape(-1)[i] += step
                s = moved[0] @ moved[1].t() + moved[2]
                keep = y != -100
                return float(torch.nn.functional.cross_entropy(s[keep], y[keep], reduction="sum"))
            slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
            assert abs(float(g.reshape(-1)[i]) - slope) <= 2e-2 * (1 + abs(slope))


def test_values_beyond_2_to_the_31(cuda):
    """A weight of 2^31 values and more: classes at its far end, against sums over pieces of the classes."""
    n, v, d = 40, (1 << 31) // 256 + 3000, 256
    gen = torch.Generator(device=cuda).manual_seed(2)
    w = torch.empty((v, d), dtype=torch.bfloat16, device=cuda)
    for k in range(0, v, 1 << 20):
        w[k:k + (1 << 20)] = torch.randn((min(1 << 20, v - k), d), generator=gen, device=cuda) / 16
    y = torch.randint(0, v, (n,), generator=gen, device=cuda)
    y[:20] = v - 1 - torch.arange(20, device=cuda) * 97
    x = torch.randn((n, d), generator=gen, device=cuda).bfloat16()
    x[:20] += w[y[:20]] * 6
    x, w = x.requires_grad_(), w.requires_grad_()
    losses = fastgl.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(losses, (x, w), torch.ones(n, device=cuda))
    with torch.no_grad():
        total = torch.zeros(n, dtype=torch.float64, device=cuda)
        want_dx = torch.zeros((n, d), dtype=torch.float64, device=cuda)
        for k in range(0, v, 1 << 19):
            s = (x.float() @ w[k:k + (1 << 19)].float().t()).double()
            total += s.exp().sum(1)
            want_dx += (s.exp().float() @ w[k:k + (1 << 19)].float()).double()
        own = (x.double() * w[y].double()).sum(1)
        # (fp32 sums of 256 products on either side, shares rounded to bf16 on this: 2^-8 of sums of magnitudes, which are ten times the sums here)
        assert ((losses.double() - (total.log() - own)).abs() <= 1e-5 * losses.abs()).all()
        want_dx = want_dx / total[:, None] - w[y].double()
        assert (dx.double() - want_dx).norm() <= 2.0 ** -7 * want_dx.norm()
        last = slice(v - 2000, v)
        p = (x.double() @ w[last].double().t()).exp() / total[:, None]
        p[torch.arange(20, device=cuda), y[:20] - (v - 2000)] -= 1
        want_dw = p.t() @ x.double()
        assert (dw[last].double() - want_dw).norm() <= 2.0 ** -7 * want_dw.norm()
        assert (dw[last].double() - want_dw).abs().amax() <= 2.0 ** -7 * want_dw.abs().amax()


def test_refusals(cuda):
    x, w, b, y = make(cuda, 10, 6, 8, torch.float32)
    ce = fastgl.linear_cross_entropy
    for bad in (lambda: ce(x, w[:, :7], y), lambda: ce(x[0], w, y), lambda: ce(x, w.bfloat16(), y), lambda: ce(x, w, y, b.bfloat16()), lambda: ce(x.half(), w.half(), y),
                lambda: ce(x, w, y, b[:5]), lambda: ce(x, w, y, torch.stack([b, b], 1)[:, 0]), lambda: ce(x, w, y[:9]), lambda: ce(x, w, y.float()),
                lambda: ce(x, w, y.short()), lambda: ce(x, w, y.cpu()), lambda: ce(x, w, torch.stack([y, y], 1)[:, 0]), lambda: ce(x, w, y, reduction="max"),
                lambda: ce(x, w[:0], y), lambda: ce(x[:, :0], w[:, :0], y), lambda: ce(torch.zeros((3, 513), device=cuda), torch.zeros((4, 513), device=cuda), y[:3])):
        with pytest.raises(RuntimeError):
            bad()


def test_autocast_takes_its_type(cuda):
    x, w, b, y = make(cuda, 40, 20, 16, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
    assert torch.equal(loss, fastgl.linear_cross_entropy(x.bfloat16(), w.bfloat16(), y, b.bfloat16()))
    assert all(g.dtype == torch.float32 for g in torch.autograd.grad(loss, leaves))


def test_same_bits_on_every_run_and_on_another_stream(cuda):
    x, w, b, y = make(cuda, 700, 900, 128, torch.float32)
    run = lambda: check(x, w, b, y)  # noqa: E731
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first[0], second[0]) and all(torch.equal(p, q) for p, q in zip(first[1], second[1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(cuda, dtype):
    x, w, b, y = make(cuda, 300, 180, 100, dtype)
    d = torch.ones((), device=cuda)
    held = [x.clone(), w.clone(), b.clone(), y.clone()]

    def step():
        leaves = [t.detach().requires_grad_() for t in held[:3]]
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], held[3], leaves[2])
        return loss.detach(), torch.autograd.grad(loss, leaves, d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for k in range(4):
        nx, nw, nb, ny = make(cuda, 300, 180, 100, dtype, seed=50 + k)
        for t, u in zip(held, (nx, nw, nb, ny)):
            t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        want_loss, want = step()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and all(torch.equal(p, q) for p, q in zip(grads, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_far_apart(cuda, dtype):
    # maxima that move many times, and far: classes in ascending order of their logits
    n, v = 40, 2000
    w = torch.zeros((v, 8), device=cuda)
    w[:, 0] = torch.linspace(-100, 100, v, device=cuda)
    x = torch.zeros((n, 8), device=cuda)
    x[:, 0] = torch.linspace(-4, 4, n, device=cuda)
    y = torch.randint(0, v, (n,), generator=torch.Generator(device=cuda).manual_seed(3), device=cuda)
    check(x.to(dtype), w.to(dtype), None, y, reduction="none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), 1e30])
def test_what_padded_rows_hold_is_nobodys_matter(cuda, dtype, what):
    x, w, b, y = make(cuda, 200, 130, 72, dtype, ignored=0.4)
    x[y == -100] = 0.0
    want_loss, want = check(x, w, b, y)
    padded = x.clone()
    padded[y == -100] = what
    leaves = [t.detach().requires_grad_() for t in (padded, w, b)]
    loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2])
    gen = torch.Generator(device=cuda).manual_seed(1)
    grads = torch.autograd.grad(loss, leaves, torch.rand((), generator=gen, device=cuda) + 0.5)
    assert torch.equal(loss.detach(), want_loss) and all(torch.equal(p, q) for p, q in zip(grads, want))


@pytest.mark.parametrize("far", [(0, 0), (-30, 10), (60, -50), (-90, 20)])
def test_rows_and_classes_of_many_magnitudes(cuda, far):
    """fp32: two kinds of rows and of classes in any order, powers of two apart, each with columns of its own; a kind's products are near 1.  A row's or
    class's values that are within 2^12 of their tile's largest are taken with 2^-25 / 2^2 of their own largest, others with less: 2^-27 of it for either
    factor, 2^-26 d max|x_i| max|w_v| for a logit."""
    n, v, d = 150, 170, 64
    gen = torch.Generator(device=cuda).manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen, device=cuda) for s in ((n, d), (v, d), (v,)))
    w /= 4
    scaled = torch.zeros(n, dtype=torch.float64, device=cuda)
    rows, classes = (torch.randint(0, 2, (k,), generator=gen, device=cuda) for k in (n, v))
    columns = torch.arange(d, device=cuda) // (d // 2)
    power = 2.0 ** torch.tensor(far, device=cuda, dtype=torch.float64)
    for k in (0, 1):
        most = x[rows == k][:, columns == k].abs().amax(1).double() * float(w[classes == k][:, columns == k].abs().max())
        scaled[rows == k] = 2.0 ** -26 * d * most
    x = torch.where(rows[:, None] == columns, x * power[rows][:, None], 0.0).float()
    w = torch.where(classes[:, None] == columns, w / power[classes][:, None], 0.0).float()
    y = torch.randint(0, v, (n,), generator=gen, device=cuda)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    losses = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction="none")
    g = torch.ones(n, device=cuda)
    grads = torch.autograd.grad(losses, leaves, g)
    (want, _, *want_grads), sums, largest = definition(x, w, b, y, -100, "none", g)
    u = 2.0 ** -24
    most = (x.abs().double() @ w.abs().double().t()).amax(1) + float(b.abs().max())
    eps = 4 * u * (14 + 3 * d / 16 + 4) * (most + 4) + (v / 32 + 8) * u + 4 * scaled
    assert ((losses.detach().double() - want).abs() <= eps * (1 + want)).all(), float(((losses.detach().double() - want).abs() / eps).max())
    for name, got, exact, total, top in zip(("dx", "dw", "db"), grads, want_grads, sums, largest):
        terms = n if name != "dx" else v
        limit = (2 * eps.max() + (6 * terms / 32 + 16) * u + 12 * u) * total + u * exact.abs() + terms * 2.0 ** -35 * top + 2.0 ** -120
        assert ((got.double() - exact).abs() <= limit).all(), (name, float(((got.double() - exact).abs() / limit).max()))


def test_layer(cuda):
    torch.manual_seed(0)
    layer = fastgl.LinearCrossEntropy(48, 37).to(cuda)
    x, _, _, y = make(cuda, 80, 37, 48, torch.float32)
    want = torch.nn.functional.cross_entropy(layer.logits(x), y)
    loss = layer(x, y)
    assert torch.allclose(loss, want, rtol=1e-5)
    loss.backward()
    assert layer.weight.grad.shape == (37, 48) and layer.bias.grad.shape == (37,)
    assert fastgl.LinearCrossEntropy(48, 37, bias=False).bias is None
