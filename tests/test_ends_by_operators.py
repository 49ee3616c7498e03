"""Dropout and the loss of a last layer as they are formed where torch's operators have to be seen (tracing, forward mode, transforms): the same
values as the kernels', here on the CPU, against the generator restated on whole numbers and torch's own loss in 64 bits."""
import pytest
import torch

from fastgl import dropouts, losses
from test_gpu_dropout import words

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("shape", [(1,), (33, 47), (3, 5, 7), (0, 5)])
def test_dropout(dtype, relu, p, shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    if x.numel() > 50:
        x.view(-1)[:8] = float("nan")
    x.requires_grad_()
    seed, stream = 2 ** 63 + 12345, 2 ** 32 - 2
    y = dropouts._by_operators(x, p, seed, stream, relu, None)
    n = x.numel()
    kept = torch.from_numpy(words(0, (n + 3) // 4 * 4, seed, stream)[:n] >= round(p * 2.0 ** 32)).view(shape)
    scale = torch.tensor(1 / (1 - p) if p < 1 else 0.0, dtype=torch.float32)
    want = torch.where(kept, (x.detach().float().clamp(min=0) if relu else x.detach().float()) * scale, 0.0).to(dtype)
    assert torch.equal(y.detach().nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(y.isnan(), want.isnan())
    d = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    g, = torch.autograd.grad(y, x, d)
    passed = kept & ~(x.detach() <= 0) if relu else kept
    assert torch.equal(g, torch.where(passed, d.float() * scale, 0.0).to(dtype))
    offset = torch.tensor([-5], dtype=torch.int32)
    moved = dropouts._by_operators(x, p, seed, 3, relu, offset)
    assert torch.equal(moved.nan_to_num(9.0), dropouts._by_operators(x, p, seed, 2 ** 32 - 2, relu, None).nan_to_num(9.0))


def test_dropout_refuses():
    for bad in (dict(x=torch.zeros(3, dtype=torch.float16)), dict(p=1.5), dict(p=float("nan")), dict(stream_offset=torch.zeros(2, dtype=torch.int32))):
        call = dict(x=torch.zeros(3), p=0.5, seed=0, stream=0, relu=False, stream_offset=None)
        with pytest.raises(RuntimeError):
            dropouts._by_operators(**{**call, **bad})


def problem(dtype, n=60, v=33, d=20, label_dtype=torch.int64):
    gen = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen).to(dtype) for s in ((n, d), (v, d), (v,)))
    y = torch.randint(0, v, (n,), generator=gen)
    y[::7] = -100
    x[0] = float("nan")  # (a row without a label)
    return x, w, b, y.to(label_dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("label_dtype", [torch.int32, torch.int64])
def test_loss(dtype, reduction, label_dtype):
    x, w, b, y = problem(dtype, label_dtype=label_dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = losses._by_operators(x, w, y, b, -100, reduction)
    X, W, B = (torch.nan_to_num(t.detach().double()).requires_grad_() for t in leaves)
    want = torch.nn.functional.cross_entropy(X @ W.t() + B, y.long(), reduction=reduction)
    # Sums of d products and of v shares in fp32, each rounding off by u of the sum of magnitudes, at most M for a logit; the exponential's argument
    # makes u M more: eps of a share and, of 1 + loss, of a loss.  A gradient's terms: 2 eps, and a sum of at most 60 of them.
    most = float((X.detach().abs() @ W.detach().abs().t() + B.detach().abs()).max())
    eps = (20 + 33 + 16) * U * (most + 4)
    assert loss.dtype == torch.float32 and ((loss.double() - want).abs() <= eps * (1 + want) * (60 if reduction == "sum" else 1)).all()
    got, exact = torch.autograd.grad(loss.sum(), leaves), torch.autograd.grad(want.sum(), (X, W, B))
    half = 2.0 ** -8 if dtype == torch.bfloat16 else U
    for g, e in zip(got, exact):
        # (the terms' magnitudes: at most 60 shares of at most 1 times values of at most 5)
        assert g.dtype == dtype and ((g.double() - e).abs() <= (2 * eps + 60 * U) * 60 * 5 + half * e.abs()).all()
    assert (got[0][0] == 0).all()


def test_loss_of_labels_and_classes_that_are_not():
    x, w, b, y = problem(torch.float32)
    y[1], y[2] = 33, -3
    assert losses._by_operators(x, w, y, b, -100, "none").isnan().nonzero()[:, 0].tolist() == [1, 2]
    y[1], y[2] = 4, 5
    for out in (float("-inf"), torch.finfo(torch.float32).min, -1e30):
        b[9] = out
        y[y == 9] = 8
        w[9] = float("nan")
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        loss = losses._by_operators(leaves[0], leaves[1], y, leaves[2], -100, "mean")
        got = torch.autograd.grad(loss, leaves)
        assert torch.isfinite(loss) and (got[1][9] == 0).all() and got[2][9] == 0 and torch.isfinite(got[0]).all()
    none = torch.full_like(y, -100)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = losses._by_operators(leaves[0], leaves[1], none, leaves[2], -100, "mean")
    assert loss.isnan() and all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
    assert losses._by_operators(x, w, none, b, -100, "sum") == 0
    assert losses._by_operators(x[:0], w, y[:0], b, -100, "mean").isnan() and losses._by_operators(x[:0], w, y[:0], b, -100, "none").shape == (0,)


def test_loss_refuses():
    x, w, b, y = problem(torch.float32)
    for bad in ((x, w[:, :7], y, b), (x[1], w, y, b), (x, w.bfloat16(), y, b), (x, w, y, b.bfloat16()), (x.half(), w.half(), y, None), (x, w, y, b[:5]), (x, w, y[:9], b), (x, w, y.float(), b),
                (x, w, y.short(), b), (x, w[:0], y, None), (x[:, :0], w[:, :0], y, None), (torch.zeros(3, 513), torch.zeros(4, 513), y[:3], None)):
        with pytest.raises(RuntimeError):
            losses._by_operators(*bad, -100, "mean")
