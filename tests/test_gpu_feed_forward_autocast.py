"""FeedForward under autocast: rows of fp32 that pass through it stay fp32, as beside torch's modules."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep8", [False, True])
def test_rows_keep_their_type(cuda, keep8):
    torch.manual_seed(3)
    block = fastgl.FeedForward(64, 96, keep8=keep8).to(cuda)
    x = (torch.randn((500, 64), device=cuda) * 100).requires_grad_()  # (with bits that bf16 has not, and far above what the block adds)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x)
        z = block(y)
        added = block.down(block.up(block.norm(x)))
    assert y.dtype == z.dtype == torch.float32 and added.dtype == torch.bfloat16
    assert torch.equal(y, x + added)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert gx.dtype == torch.float32
    # the same in torch's modules
    up, down = (torch.nn.Linear(a, b).to(cuda) for a, b in ((64, 96), (96, 64)))
    up.load_state_dict(block.up.state_dict()), down.load_state_dict(block.down.state_dict())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = x + down(torch.nn.functional.gelu(up(torch.nn.functional.layer_norm(x, (64,)))))
    assert want.dtype == torch.float32
    # bf16 of what is added, once here, three times there, and of the weights' products: eight roundings of values below the largest
    assert (y - want).abs().max() < 8 * 2.0 ** -8 * added.abs().max()
    gt, = torch.autograd.grad(want, x, torch.ones_like(want))
    assert torch.allclose(gx, gt, rtol=2.0 ** -6, atol=2.0 ** -6)


def test_rows_of_autocasts_type_go_through_at_once(cuda):
    torch.manual_seed(4)
    block = fastgl.FeedForward(64, 96).to(cuda)
    x = torch.randn((500, 64), device=cuda).bfloat16().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x)
        want = block.down(block.up(block.norm(x)), residual=x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, want)
    plain = fastgl.FeedForward(64, 96).to(cuda)
    h = torch.randn((50, 64), device=cuda)
    assert torch.equal(plain(h), plain.down(plain.up(plain.norm(h)), residual=h))
