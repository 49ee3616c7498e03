"""A weight's gradient where the last vector of a row of the operands is moved back to end with it and repeats columns of the tile before: each column is stored by the
one tile that it belongs to.  Tiles form their sums again, in another order, where they meet values that have no three parts; a column's bits must not hang on what
its neighbour's tile met."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [float("inf"), 2.0 ** -130])
@pytest.mark.parametrize("keep8,n,d,out,side", [(True, 4000, 64, 193, "out"), (True, 9001, 96, 129, "out"), (False, 4000, 64, 193, "out"), (False, 4000, 193, 64, "in")])
def test_a_column_is_its_own_tiles(cuda, keep8, n, d, out, side, odd):
    """Columns before the last one, beside a last one that is formed again, have the bits that they have beside one that is not."""
    gen = torch.Generator(device=cuda).manual_seed(n + d + out)
    x, w = torch.randn((n, d), generator=gen, device=cuda), torch.randn((out, d), generator=gen, device=cuda)
    dy = torch.randn((n, out), generator=gen, device=cuda)

    def gradient(x, dy):
        v = w.clone().requires_grad_()
        return torch.autograd.grad(fastgl.linear(x, v, keep8=keep8), v, dy)[0]

    want = gradient(x, dy)
    if side == "out":
        dy = dy.clone()
        if odd == float("inf"):
            dy[n // 2, out - 1] = odd
        else:
            dy[:, out - 1] *= odd
    else:
        x = x.clone()
        if odd == float("inf"):
            x[n // 2, d - 1] = odd
        else:
            x[:, d - 1] *= odd
    for _ in range(20):
        got = gradient(x, dy)
        if side == "out":
            assert torch.equal(got[:out - 1], want[:out - 1])
        else:
            assert torch.equal(got[:, :d - 1], want[:, :d - 1])
