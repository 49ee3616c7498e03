"""What fastgl.linear, the models' norms and blocks, and the layers' entry points refuse, on the host and before anything is launched; what torch's operators give in
linear's place."""
import pytest
import torch

import fastgl
from fastgl import layers


def test_operator_refuses():
    x, w = torch.zeros(4, 8), torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.linear(x, w)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.Linear(8, 5)(x)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.FeedForward(8, 16)(x)
    for make in (lambda: fastgl.Linear(8, 5, activation="tanh"), lambda: fastgl.FeedForward(8, 16, activation="x")):
        with pytest.raises(ValueError):
            make()
    assert "gelu" in repr(fastgl.Linear(8, 5, activation="gelu")) and "keep8" in repr(fastgl.Linear(8, 5, keep8=True))
    fastgl.Linear(8, 5).load_state_dict(torch.nn.Linear(8, 5).state_dict())


def test_models_refuse_and_keep_their_state():
    for model in (lambda **k: fastgl.GCN(8, 16, 4, 3, None, True, 0.1, **k), lambda **k: fastgl.GIN(8, 16, 4, 3, None, True, 0.1, **k), lambda **k: fastgl.SAGE(8, 16, 4, 3, **k)):
        for bad in (dict(norm="batch"), dict(feed_forward=-1), dict(keep8=True)):
            with pytest.raises(ValueError):
                model(**bad)
        plain, deep = model(), model(norm="layer", feed_forward=32, keep8=True)
        assert not any("norms" in k or "blocks" in k for k in plain.state_dict())
        assert len(deep.norms) == len(deep.blocks_between) == 2
        deep.load_state_dict(model(norm="layer", feed_forward=32).state_dict())


def test_entry_points_refuse():
    lib = fastgl.lib()

    def forward(n=4, d=8, out=6, ldx=None, ldw=None, ldr=None, ldy=None, dtype=0, act=2, keep8=1, x=256, w=256, r=256, y=256, state=256, size=1 << 20):
        return lib.fgl_linear(x, d if ldx is None else ldx, w, d if ldw is None else ldw, None, r, out if ldr is None else ldr, n, d, out, dtype, act, keep8, y,
                              out if ldy is None else ldy, state, size, None)

    def backward(n=4, d=8, out=6, ldx=None, ldw=None, lddy=None, lddx=None, dtype=0, act=2, keep8=0, x=256, w=256, dy=256, dx=256, dw=256, db=256, state=256, size=1 << 20,
                 ws=256, room=1 << 30):
        return lib.fgl_linear_backward(dy, out if lddy is None else lddy, x, d if ldx is None else ldx, w, d if ldw is None else ldw, n, d, out, dtype, act, keep8, state, size,
                                       dx, d if lddx is None else lddx, dw, db, ws, room, None)

    for call in (forward, backward):
        for bad in (dict(n=-1), dict(n=1 << 31), dict(d=0), dict(d=4097), dict(out=0), dict(out=4097), dict(dtype=2), dict(act=-1), dict(act=4), dict(ldx=7), dict(ldx=1 << 24),
                    dict(ldw=7), dict(ldw=1 << 24), dict(x=None), dict(w=None), dict(dtype=1, x=258), dict(dtype=1, ldx=9)):
            assert call(**bad) == 1, bad
        assert call(size=8) == 2 and b"state" in lib.fgl_last_error()
        assert call(state=264) == 2
    for bad in (dict(ldy=5), dict(ldy=1 << 24), dict(ldr=5), dict(ldr=1 << 24), dict(y=None), dict(dtype=1, w=258), dict(dtype=1, ldw=9)):
        assert forward(**bad) == 1, bad
    assert forward(n=0) == 0
    for bad in (dict(n=0), dict(dy=None), dict(lddy=5), dict(lddx=7), dict(lddx=1 << 24), dict(dtype=1, act=0, dy=258), dict(dtype=1, act=0, lddy=7)):
        assert backward(**bad) == 1, bad
    assert backward(state=None) == 2 and backward(room=64) == 2 and backward(ws=None) == 2 and backward(ws=260) == 2
    assert backward(dx=None, dw=None, db=None) == 0


def test_sizes_of_state_and_workspace():
    lib = fastgl.lib()
    state, ws = lib.fgl_linear_state_bytes, lib.fgl_linear_workspace_bytes
    assert state(-1, 8, 8, 0, 0, 0) == 0 and state(4, 4097, 8, 0, 0, 0) == 0 and state(4, 8, 8, 0, 4, 0) == 0 and ws(4, 8, 8, 3, 0, 0, 1, 1) == 0
    n, d, out = 100_000, 256, 512
    assert state(n, d, out, 0, 0, 0) == 0 and state(n, d, out, 0, 1, 0) <= n * out // 8 + 256 and state(n, d, out, 1, 2, 0) <= n * out * 2 + 256
    assert state(n, d, out, 0, 0, 1) <= n * d * 33 // 32 + 1024
    assert ws(n, d, out, 0, 0, 0, 0, 0) == 0 and 0 < ws(n, d, out, 0, 0, 0, 1, 0) < 300 << 20 and 0 < ws(n, d, out, 0, 0, 1, 1, 1) < 300 << 20
    for k in (1, 63, 64, 1000, 100_000):
        for m in (1, 31, 47, 256, 4096):
            for dtype in (0, 1):
                assert ws(k, 100, m, dtype, 0, 1, 1, 1) > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
def test_by_operators(dtype, activation):
    gen = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(s, generator=gen).to(dtype) for s in ((5, 30), (20, 30), (20,), (5, 20), (5, 20)))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = layers._linear_by_operators(x, w, b, activation, r)
    got = torch.autograd.grad(y, leaves, dy)
    X, W, B, R = (t.detach().double().requires_grad_() for t in leaves)
    z = X @ W.t() + B
    want = {None: lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[activation](z) + R
    half = torch.finfo(dtype).eps / 2
    size = (X.detach().abs() @ W.detach().abs().t() + B.detach().abs()).max()
    assert y.dtype == dtype and ((y.double() - want).abs() <= half * want.abs() + 60 * 2.0 ** -24 * (size + 4)).all()
    for g, e in zip(got, torch.autograd.grad(want, (X, W, B, R), dy.double())):
        assert ((g.double() - e).abs() <= half * e.abs() + 200 * 2.0 ** -24 * (size + 4)).all()
    for bad in (dict(x=x.detach().double()), dict(weight=w.detach()[:, :5]), dict(bias=b.detach()[:3]), dict(residual=r.detach()[:1])):
        with pytest.raises(RuntimeError):
            layers._linear_by_operators(**{**dict(x=x, weight=w, bias=b, activation=activation, residual=r), **bad})
