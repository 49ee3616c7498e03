"""What fastgl.dropout and fgl_dropout refuse, on the host and before anything is launched."""
import pytest
import torch

import fastgl
from fastgl import _lib as L


def test_operator_refuses():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fastgl.dropout(torch.zeros(4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fastgl.dropout([1.0])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fastgl.Dropout(0.5)(torch.zeros(4))
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            fastgl.Dropout(p)


def test_entry_points_refuse():
    lib = fastgl.lib()
    call = lambda ldx=8, rows=2, cols=8, dtype=0, p=0.5, x=None: lib.fgl_dropout(x, ldx, rows, cols, dtype, p, 0, 0, None, 0, x, None)  # noqa: E731
    assert call(dtype=2) == 1 and b"dtype" in lib.fgl_last_error()
    assert call(p=1.5) == 1 and call(p=-0.5) == 1 and call(p=float("nan")) == 1 and b"probability" in lib.fgl_last_error()
    assert call(rows=-1) == 1 and call(cols=-1) == 1 and b"negative" in lib.fgl_last_error()
    assert call(rows=0) == 0 and call(cols=0) == 0
    assert call() == 1 and b"null" in lib.fgl_last_error()
    assert call(ldx=7, x=64) == 1 and b"stride" in lib.fgl_last_error()
    assert call(ldx=1 << 32, cols=1 << 31, x=64) == 1 and b"columns" in lib.fgl_last_error()
    assert call(ldx=1 << 20, rows=1 << 16, cols=1 << 20, x=64) == 1 and b"2^35" in lib.fgl_last_error()
    back = lambda n, dtype=0, p=0.5: lib.fgl_dropout_relu_backward(None, None, n, dtype, p, None, None)  # noqa: E731
    assert back(0) == 0 and back(1) == 1 and back(-1) == 1 and back((1 << 35) + 1) == 1 and back(1, dtype=9) == 1 and back(1, p=2.0) == 1


def test_layer_counts_nothing_in_evaluation():
    layer = fastgl.Dropout(0.5, seed=3, relu=True).eval()
    with pytest.raises(RuntimeError):
        layer(torch.zeros(3))
    assert layer.calls == 0 and "seed=3" in repr(layer) and "relu" in repr(layer)
    assert L.SIGNATURES["fgl_dropout"][0] is L._i32
