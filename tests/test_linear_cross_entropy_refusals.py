"""What fastgl.linear_cross_entropy and its entry points refuse, on the host and before anything is launched."""
import pytest
import torch

import fastgl


def test_operator_refuses():
    x, w, y = torch.zeros(4, 8), torch.zeros(3, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.linear_cross_entropy(x, w, y)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        fastgl.LinearCrossEntropy(8, 3)(x, y)
    assert fastgl.LinearCrossEntropy(8, 3).logits(x).shape == (4, 3)


def test_entry_points_refuse():
    lib = fastgl.lib()

    def forward(n=4, v=3, d=8, dtype=0, reduction=2, want=3, at=256, state=1 << 30, ws=1 << 30):
        return lib.fgl_linear_cross_entropy(at, d, 1, at, d, 1, None, at, 1, -100, n, v, d, dtype, reduction, want, at, at, state, at, ws, None)

    def backward(n=4, v=3, d=8, dtype=0, reduction=2, want=3, at=256, dx=256, dw=256, db=256, state=1 << 30, ws=1 << 30):
        return lib.fgl_linear_cross_entropy_backward(at, n, v, d, dtype, reduction, want, at, state, dx, dw, db, at, ws, None)

    for call in (forward, backward):
        for bad in (dict(n=0), dict(n=-1), dict(n=1 << 31), dict(v=0), dict(v=1 << 31), dict(d=0), dict(d=513), dict(dtype=2), dict(reduction=3), dict(want=4), dict(at=None)):
            assert call(**bad) == 1, bad
        assert call(state=64) == 2 and b"state" in lib.fgl_last_error()
        assert call(at=257) == 2 and b"256-byte" in lib.fgl_last_error()
    assert forward(ws=64) == 2
    assert backward(want=0) == 1 and backward(want=1) == 1 and backward(want=2) == 1 and backward(dw=None) == 1  # (bias without weight)


def test_sizes_of_state_and_workspace():
    lib = fastgl.lib()
    state, ws = lib.fgl_linear_cross_entropy_state_bytes, lib.fgl_linear_cross_entropy_workspace_bytes
    assert state(0, 3, 8, 0, 3) == 0 and state(4, 3, 600, 0, 3) == 0 and ws(4, 0, 8, 0, 3, 0) == 0
    logits = 8192 * 100_000 * 2
    assert 0 < state(8192, 100_000, 256, 1, 3) < logits // 10 and 0 < ws(8192, 100_000, 256, 1, 3, 0) < logits // 10
    # the loss alone keeps nothing, and each gradient what it needs
    assert state(8192, 100, 256, 1, 0) <= 256 < state(8192, 100, 256, 1, 1) < state(8192, 100, 256, 1, 3) and ws(8192, 100, 256, 1, 1, 1) == 0
    for n in (1, 31, 32, 33, 128, 129, 8192, 100_000):
        for v in (1, 2, 33, 4097, 1_000_000):
            for d in (1, 32, 100, 256, 257, 512):
                for dtype in (0, 1):
                    for want in (0, 1, 2, 3):
                        assert state(n, v, d, dtype, want) > 0 and ws(n, v, d, dtype, want, 0) > 0


def test_sizes_beyond_a_launch_are_refused_before_the_forward_pass():
    lib = fastgl.lib()
    for n, v, d in ((1 << 29, 3, 8), (3, 1 << 29, 8), (1 << 28, 1 << 28, 8), (1 << 24, 3, 512), (1 << 28, 3, 32)):
        assert lib.fgl_linear_cross_entropy_state_bytes(n, v, d, 1, 3) == 0 and lib.fgl_linear_cross_entropy_workspace_bytes(n, v, d, 1, 3, 1) == 0
        assert lib.fgl_linear_cross_entropy(256, d, 1, 256, d, 1, None, 256, 1, -100, n, v, d, 1, 2, 3, 256, 256, 1 << 40, 256, 1 << 40, None) == 1
    assert lib.fgl_linear_cross_entropy_state_bytes((1 << 24) - 32, 3, 512, 1, 3) > 0 and lib.fgl_linear_cross_entropy_state_bytes((1 << 28) - 32, 1 << 20, 32, 1, 3) > 0
