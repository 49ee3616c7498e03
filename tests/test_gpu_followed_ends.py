"""Dropout and the loss of a last layer where somebody follows torch's operators: forward mode, tracing, transforms of torch.func, modes and
tensor subclasses see what they would of torch's own, and the values are the kernels'."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.flop_counter import FlopCounterMode

import fastgl

pytestmark = pytest.mark.gpu


def make(cuda, dtype=torch.float32, n=60, v=33, d=24):
    gen = torch.Generator(device=cuda).manual_seed(5)
    x, w, b = (torch.randn(s, generator=gen, device=cuda).to(dtype) for s in ((n, d), (v, d), (v,)))
    y = torch.randint(0, v, (n,), generator=gen, device=cuda)
    y[::7] = -100
    return x, w, b, y


class Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def close(a, b, eps=2.0 ** -10):
    """Either side's shares are off by (24 + 33 + 16) u (M + 4) of themselves, for sums of 24 products and 33 shares and logits' magnitudes M below 60: 2^-11.8;
    a gradient's terms by twice that, and its own roundings are little beside it."""
    return a.shape == b.shape and a.dtype == b.dtype and (a.double() - b.double()).abs().max() <= eps * (1 + b.double().abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
def test_dropout_by_operators_is_the_kernels(cuda, dtype, relu):
    x = make(cuda, dtype)[0]
    x[3] = float("nan")
    offset = torch.tensor([-7], dtype=torch.int32, device=cuda)
    for p in (0.0, 0.3, 1.0):
        for more in (dict(stream=2 ** 32 - 1), dict(stream=5, stream_offset=offset)):
            want = fastgl.dropout(x, p, seed=2 ** 64 - 3, relu=relu, **more)
            with Watch() as watch:
                got = fastgl.dropout(x, p, seed=2 ** 64 - 3, relu=relu, **more)
            assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0)) and torch.equal(got.isnan(), want.isnan())
            assert watch.seen and not any("aten.empty" in s for s in watch.seen)


@pytest.mark.parametrize("record", [False, True])
@pytest.mark.parametrize("relu", [False, True])
def test_dropout_in_forward_mode(cuda, record, relu):
    x = make(cuda)[0]
    t = torch.randn_like(x)
    want = fastgl.dropout(x, 0.4, seed=3, relu=relu)
    with torch.set_grad_enabled(record), forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(record), t)
        y, tangent = forward_ad.unpack_dual(fastgl.dropout(dual, 0.4, seed=3, relu=relu))
        assert torch.equal(y.detach(), want)
        kept = fastgl.dropout(torch.ones_like(x), 0.4, seed=3) != 0
        if relu:
            kept = kept & (x > 0)
        assert torch.allclose(tangent, torch.where(kept, t / 0.6, 0.0), rtol=2.0 ** -22)


@pytest.mark.parametrize("record", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_in_forward_mode(cuda, record, reduction):
    x, w, b, y = make(cuda)
    t = torch.randn_like(x)
    want, want_tangent = torch.func.jvp(
        lambda x: torch.nn.functional.cross_entropy(x @ w.double().t() + b.double(), y, reduction=reduction), (x.double(),), (t.double(),))
    with torch.set_grad_enabled(record), forward_ad.dual_level():
        loss = fastgl.linear_cross_entropy(forward_ad.make_dual(x.clone().requires_grad_(record), t), w, y, b, reduction=reduction)
        loss, tangent = forward_ad.unpack_dual(loss)
    assert close(loss.detach(), want.float()) and close(tangent.detach(), want_tangent.float())


@pytest.mark.parametrize("relu", [False, True])
def test_traced_dropout(cuda, relu):
    x = make(cuda)[0]
    layer = fastgl.Dropout(0.4, seed=9, relu=relu)
    traced = torch.jit.trace(layer, (x,), check_trace=False)
    stream = layer.calls - 1
    other = torch.randn(31, 24, device=cuda)
    for k in range(3):
        junk = torch.full((400, 24), float("nan"), device=cuda)  # noqa: F841 (memory that a later allocation takes)
        del junk
        assert torch.equal(traced(other), fastgl.dropout(other, 0.4, 9, stream, relu=relu))
    layer.eval()
    assert torch.equal(torch.jit.trace(layer, (x,))(other), other.clamp(min=0) if relu else other)


def test_traced_loss(cuda):
    x, w, b, y = make(cuda)
    torch.manual_seed(0)
    head = fastgl.LinearCrossEntropy(24, 33).to(cuda)
    traced = torch.jit.trace(head, (x, y))
    other, labels = torch.randn(17, 24, device=cuda), y[:17].clone()
    loss = traced(other, labels)
    assert close(loss, head(other, labels))
    got, want = torch.autograd.grad(loss, list(head.parameters())), torch.autograd.grad(head(other, labels), list(head.parameters()))
    assert all(close(p, q) for p, q in zip(got, want))


def test_modes_see_the_operators(cuda):
    x, w, b, y = make(cuda)
    want = fastgl.linear_cross_entropy(x, w, y, b)
    with FlopCounterMode(display=False) as counter:
        assert close(fastgl.linear_cross_entropy(x, w, y, b), want)
    assert counter.get_total_flops() == 2 * x.numel() * w.size(0)

    class Calls(torch.overrides.TorchFunctionMode):
        names = []

        def __torch_function__(self, func, types, args=(), kwargs=None):
            self.names.append(getattr(func, "__name__", ""))
            return func(*args, **(kwargs or {}))

    with Calls():
        assert close(fastgl.linear_cross_entropy(x, w, y, b), want)
        fastgl.dropout(x, 0.5)
    assert "linear" in Calls.names and "where" in Calls.names
    with torch.device(cuda):  # (a default device is a mode too, and follows nothing: the kernel's own bits)
        assert torch.equal(fastgl.linear_cross_entropy(x, w, y, b), want)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as fake:
        a = [fake.from_tensor(t) for t in (x, w, y, b)]
        assert fastgl.linear_cross_entropy(*a, reduction="none").shape == (60,) and fastgl.dropout(a[0], 0.5).shape == x.shape


def test_transforms(cuda):
    x, w, b, y = make(cuda)
    many = torch.stack([x, 2 * x, -x])
    keep = lambda t: fastgl.dropout(t, 0.4, seed=1, stream=2)  # noqa: E731
    assert torch.equal(torch.func.vmap(keep)(many), torch.stack([keep(t) for t in many]))
    loss = lambda t: fastgl.linear_cross_entropy(t, w, y, b)  # noqa: E731
    assert close(torch.func.vmap(loss)(many), torch.stack([loss(t) for t in many]))
    head = fastgl.LinearCrossEntropy(24, 33).to(cuda)
    got = torch.func.grad(lambda p: torch.func.functional_call(head, p, (keep(x), y)))(dict(head.named_parameters()))
    want = torch.autograd.grad(head(keep(x), y), list(head.parameters()))
    assert close(got["weight"], want[0]) and close(got["bias"], want[1])


def test_tensors_that_take_their_operators_themselves(cuda):
    class Named(torch.Tensor):
        pass

    x, w, b, y = make(cuda)
    named = x.as_subclass(Named)
    assert type(fastgl.dropout(named, 0.3, seed=4)) is Named and torch.equal(fastgl.dropout(named, 0.3, seed=4).as_subclass(torch.Tensor), fastgl.dropout(x, 0.3, seed=4))
    loss = fastgl.linear_cross_entropy(named, w, y, b)
    assert type(loss) is Named and close(loss.as_subclass(torch.Tensor), fastgl.linear_cross_entropy(x, w, y, b))


def test_a_models_evaluation_traced(cuda):
    """The activation of a seeded SAGE is the dropout layer's, in evaluation too."""
    layer = fastgl.Dropout(0.5, seed=1, relu=True).eval()
    x = make(cuda)[0]
    with forward_ad.dual_level(), torch.no_grad():
        y, tangent = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, torch.ones_like(x))))
        assert torch.equal(y, x.clamp(min=0)) and torch.equal(tangent, (x > 0).float())


def test_autocast(cuda):
    x, w, b, y = make(cuda)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = fastgl.linear_cross_entropy(x, w, y, b)
        with Watch():
            got = fastgl.linear_cross_entropy(x, w, y, b)
    assert close(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("p", [0.4, 1.0])
def test_batched_gradients_of_dropout(cuda, dtype, relu, p):
    """The same bits as one after another: a product in fp32, rounded once."""
    x = make(cuda, dtype)[0].requires_grad_()
    y = fastgl.dropout(x, p, seed=3, stream=8, relu=relu)
    v = torch.randn(5, 60, 24, device=cuda).to(dtype)
    got, = torch.autograd.grad(y, x, v, is_grads_batched=True, retain_graph=True)
    assert torch.equal(got, torch.stack([torch.autograd.grad(y, x, t, retain_graph=True)[0] for t in v]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("needs", [(1, 1, 1), (1, 0, 0), (0, 0, 1)])
def test_batched_gradients_of_the_loss(cuda, dtype, reduction, needs):
    x, w, b, y = make(cuda, dtype)
    leaves = [t.requires_grad_(bool(k)) for t, k in zip((x, w, b), needs)]
    loss = fastgl.linear_cross_entropy(x, w, y, b, reduction=reduction)
    v = torch.randn(4, *loss.shape, device=cuda)
    wanted = [t for t, k in zip(leaves, needs) if k]
    got = torch.autograd.grad(loss, wanted, v, is_grads_batched=True, retain_graph=True)
    want = [torch.autograd.grad(loss, wanted, t, retain_graph=True) for t in v]
    assert all(torch.equal(g, torch.stack(e)) for g, e in zip(got, zip(*want)))


def test_vectorized_jacobian(cuda):
    x, w, b, y = make(cuda, n=6)
    f = lambda t: fastgl.linear_cross_entropy(t, w, y, b, reduction="none")  # noqa: E731
    want = torch.autograd.functional.jacobian(f, x)
    assert torch.equal(torch.autograd.functional.jacobian(f, x, vectorize=True), want)
    g = lambda t: fastgl.dropout(t, 0.5, seed=1)  # noqa: E731
    assert torch.equal(torch.autograd.functional.jacobian(g, x, vectorize=True), torch.autograd.functional.jacobian(g, x))


def test_vectorized_jacobian_with_a_graph(cuda):
    x, w, b, y = make(cuda, n=6)
    f = lambda t: fastgl.linear_cross_entropy(t, w, y, b, reduction="none")  # noqa: E731
    x.requires_grad_()
    made = torch.autograd.functional.jacobian(f, x, create_graph=True, vectorize=True)
    assert torch.equal(made.detach(), torch.autograd.functional.jacobian(f, x))
    with pytest.raises(RuntimeError, match="no gradients of its gradients"):
        torch.autograd.grad(made.sum() + (x * x).sum(), x)
    g = lambda t: fastgl.dropout(t, 0.5, seed=1, relu=True)  # noqa: E731
    assert torch.equal(torch.autograd.functional.jacobian(g, x, create_graph=True, vectorize=True).detach(), torch.autograd.functional.jacobian(g, x))


def test_a_traced_model(cuda):
    """A whole seeded SAGE in evaluation, blocks held: another input than that of the trace."""
    edge_ptr, edge_src = fastgl.graph.rmat_csr(2000, 20000, seed=3, device=cuda)
    sampler = fastgl.FusedMapSampler([3, 3], rng_seed=1).set_graph(edge_ptr, edge_src)
    inputs, _, blocks = sampler.sample_blocks(None, torch.arange(50, dtype=torch.int32, device=cuda) * 31)
    x = torch.randn(inputs.numel(), 8, device=cuda)
    seeded = fastgl.SAGE(8, 16, 5, 2, dropout=0.5, dropout_seed=4).to(cuda).eval()
    with torch.no_grad(), forward_ad.dual_level():
        y, tangent = forward_ad.unpack_dual(seeded._between(forward_ad.make_dual(x, torch.ones_like(x))))
    assert torch.equal(y, x.clamp(min=0)) and torch.equal(tangent, (x > 0).float())


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradients_of_gradients_are_refused_wherever_they_are_asked_for(cuda, reduction):
    """A penalty on a gradient beside something that has second derivatives: the sum must not come back without the penalty's part."""
    leaves = [t.requires_grad_() for t in make(cuda)[:3]]
    y = make(cuda)[3]
    d = torch.ones(60 if reduction == "none" else (), device=cuda, requires_grad=True)
    for k in range(3):
        loss = fastgl.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction=reduction)
        grads = torch.autograd.grad(loss, leaves, d, create_graph=True)
        assert all(torch.equal(p.detach(), q) for p, q in zip(grads, torch.autograd.grad(loss, leaves, d.detach(), retain_graph=True)))
        total = grads[k].square().sum() + sum(t.square().sum() for t in leaves) + d.sum()
        for of in (leaves[0], leaves[1], leaves[2], d):
            with pytest.raises(RuntimeError, match="no gradients of its gradients"):
                torch.autograd.grad(total, of, retain_graph=True)
        with pytest.raises(RuntimeError, match="no gradients of its gradients"):
            total.backward(retain_graph=True)
    # of the losses themselves there is one
    assert torch.isfinite(torch.autograd.grad(loss.sum() + leaves[0].square().sum(), leaves[0])[0]).all()
