"""What fastgl.layer_norm and its entry points refuse, on the host and before anything is launched; what torch's operators give in its place."""
import pytest
import torch

import fastgl
from fastgl import layers


def test_operator_refuses():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.LayerNorm(8)(x)
    with pytest.raises(RuntimeError, match="columns"):
        fastgl.LayerNorm(9)(x)
    with pytest.raises(ValueError):
        fastgl.LayerNorm((3, 4))
    assert "relu" in repr(fastgl.LayerNorm(8, relu=True)) and "keep8" in repr(fastgl.LayerNorm(8, keep8=True))
    fastgl.LayerNorm(8).load_state_dict(torch.nn.LayerNorm(8).state_dict())


def test_entry_points_refuse():
    lib = fastgl.lib()

    def forward(n=4, d=8, ld=8, dtype=0, eps=1e-5, x=256, y=256, state=256, size=1 << 20, keep8=0):
        return lib.fgl_layer_norm(x, ld, None, None, n, d, dtype, eps, 0, keep8, y, state, size, None)

    def backward(n=4, d=8, ld=8, ldx=8, dtype=0, x=256, dy=256, state=256, size=1 << 20, dw=256, ws=256, room=1 << 20, keep8=0):
        return lib.fgl_layer_norm_backward(dy, ld, x, ldx, None, n, d, dtype, 0, keep8, state, size, 256, dw, None, ws, room, None)

    for call in (forward, backward):
        for bad in (dict(n=-1), dict(n=(1 << 31) + 1), dict(d=0), dict(d=2049), dict(dtype=2), dict(ld=7), dict(x=None)):
            assert call(**bad) == 1, bad
        assert call(size=8) == 2 and b"state" in lib.fgl_last_error()
        assert call(state=264) == 2
    for bad in (dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(y=None)):
        assert forward(**bad) == 1, bad
    assert forward(n=0) == 0
    for bad in (dict(n=0), dict(dy=None), dict(state=None), dict(ldx=7)):
        assert backward(**bad) == 1, bad
    assert backward(room=63) == 2 and backward(ws=None) == 2 and backward(ws=260) == 2


def test_sizes_of_state_and_workspace():
    lib = fastgl.lib()
    state, ws = lib.fgl_layer_norm_state_bytes, lib.fgl_layer_norm_workspace_bytes
    assert state(-1, 8, 0, 0) == 0 and state(4, 2049, 0, 0) == 0 and ws(4, 0, 0) == 0 and ws(4, 8, 2) == 0
    n, d = 100_000, 256
    assert state(n, d, 0, 0) <= n * 12 + 512 and state(n, d, 1, 0) <= n * (12 + 32) + 1024 and state(n, d, 0, 1) <= n * (4 + 256 + 8) + 1024
    assert 0 < ws(n, d, 0) <= 1024 * 2 * 4 * d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("relu", [False, True])
def test_by_operators(dtype, relu):
    gen = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(s, generator=gen).to(dtype) for s in ((5, 30), (30,), (30,), (5, 30)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(layers._norm_by_operators(x, w, b, 1e-5, relu), leaves, dy)
    y = layers._norm_by_operators(x, w, b, 1e-5, relu)
    X, W, B = (t.detach().double().requires_grad_() for t in leaves)
    want = torch.nn.functional.layer_norm(X, (30,), W, B, 1e-5)
    want = want.relu() if relu else want
    half = torch.finfo(dtype).eps / 2
    assert y.dtype == dtype and ((y.double() - want).abs() <= half * want.abs() + 1e-12).all()
    for g, e in zip(got, torch.autograd.grad(want, (X, W, B), dy.double())):
        assert ((g.double() - e).abs() <= half * e.abs() + 1e-12).all()
    for bad in (dict(x=x.detach().double()), dict(weight=w.detach()[:5]), dict(eps=-1.0)):
        with pytest.raises(RuntimeError):
            layers._norm_by_operators(**{**dict(x=x, weight=w, bias=b, eps=1e-5, relu=False), **bad})
