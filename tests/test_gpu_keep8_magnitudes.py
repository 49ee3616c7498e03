"""What is held in 8 bits at the ends of the range: values next to the largest finite one, whose 128 steps would be 2^128, and the smallest."""
import numpy as np
import pytest
import torch

import fastgl
from held8 import held

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,out", [(300, 70, 40), (4000, 96, 64), (5000, 256, 130)])
@pytest.mark.parametrize("power", [-117, 0, 120, 127])
def test_weight_gradient_of_rows_of_any_size(cuda, dtype, n, d, out, power):
    """Every third row's first 32 columns lie below 2^(power + 1), one of them next to it; zeros among them stay zeros.  A sum of n products in fp32, of values that
    are exact: n + 8 roundings of the sum of magnitudes, and the result's own."""
    gen = torch.Generator(device=cuda).manual_seed(n + d + out + power)
    x = torch.randn((n, d), generator=gen, device=cuda)
    big = (torch.rand((n, 32), generator=gen, device=cuda) - 0.5) * 2.0 ** -2
    big[:, 7] = 0.8125
    big[:, 3] = 0
    x[::3, :32] = big[::3] * 2.0 ** power * 2.0
    x[1::3, :32] = 0
    x[2::3, :32] = 0
    x = x.to(dtype)
    w = (torch.randn((out, d), generator=gen, device=cuda) / d ** 0.5).to(dtype).requires_grad_()
    dy = torch.randn((n, out), generator=gen, device=cuda) * (2.0 ** -20 if power > 100 else 1.0)
    dy = dy.to(dtype)
    assert x.isfinite().all()
    gw, = torch.autograd.grad(fastgl.linear(x, w, keep8=True), w, dy)
    H, DY = held(x.cpu().double().numpy()), dy.cpu().double().numpy()
    want = DY.T @ H
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    bound = (n + 8) * U * (np.abs(DY).T @ np.abs(H)) + half * np.abs(want) + 2.0 ** -133
    got = gw.cpu().double().numpy()
    assert (np.abs(got - want) <= bound).all()
    assert (got[:, 3] == 0).all() and (np.abs(got[:, 7]) > 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_groups_with_what_is_no_number_are_none(cuda, dtype):
    """Each of 32 columns of a row with one infinite value or no number, whatever its own was; the others stay."""
    x = torch.ones((40, 96), device=cuda)
    x[:, 40:50] = 0
    x[3, 33], x[9, 70] = float("inf"), float("nan")
    x = x.to(dtype)
    w = torch.ones((40, 96), device=cuda, dtype=dtype, requires_grad=True)
    dy = torch.eye(40, device=cuda, dtype=dtype)
    y = fastgl.linear(x, w, keep8=True)
    gw, = torch.autograd.grad(y, w, dy)
    bad = torch.zeros((40, 96), dtype=torch.bool, device=cuda)
    bad[:, 32:96] = True  # (a row's zeros of dy times no number are none either)
    assert gw[bad].isnan().all() and torch.equal(gw[~bad], x[~bad])
    h = torch.randn((40, 96), device=cuda).to(dtype)
    h[3, 33] = float("inf")
    h.requires_grad_()
    g, = torch.autograd.grad(fastgl.layer_norm(h, keep8=True), h, torch.ones_like(h))
    assert g[3].isnan().all() and g[torch.arange(40) != 3].isfinite().all()
