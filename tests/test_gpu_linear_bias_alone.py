"""A dense layer whose bias, or residual, has a gradient and whose weight has none: neither needs anything of the input, and the residual's nothing at all."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu


def problem(cuda, n, d, out, dtype, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed + n + d + out)
    normal = lambda *s: torch.randn(s, generator=gen, device=cuda)  # noqa: E731
    return normal(n, d).to(dtype), (normal(out, d) / d ** 0.5).to(dtype), normal(out).to(dtype).requires_grad_(), normal(n, out).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,out", [(1, 1, 1), (3, 5, 2), (15, 64, 33), (300, 47, 130), (3000, 100, 193), (8192, 602, 256), (40_001, 33, 62), (100_001, 64, 47), (1000, 1024, 1030)])
def test_has_the_bits_that_it_has_beside_the_weights(cuda, dtype, act, keep8, n, d, out):
    x, w, b, dy = problem(cuda, n, d, out, dtype)
    want, = torch.autograd.grad(fastgl.linear(x, w.clone().requires_grad_(), b, act, keep8=keep8), b, dy)
    got, = torch.autograd.grad(fastgl.linear(x, w, b, act, keep8=keep8), b, dy)
    both = x.clone().requires_grad_()
    gx, gb = torch.autograd.grad(fastgl.linear(both, w, b, act, keep8=keep8), (both, b), dy)
    assert torch.equal(got, want) and torch.equal(gb, want)
    assert gx.shape == x.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,out,stride", [(1, 1, 1), (63, 31, 40), (64, 33, 34), (65, 64, 64), (257, 65, 70), (70_001, 130, 131), (30_003, 1025, 1025), (300_000, 8, 8)])
def test_whole_numbers_are_exact(cuda, dtype, n, out, stride):
    """Gradients of 1 to 3 and their negatives: sums of fewer than 2^24 are exact in fp32, and a row left out or taken twice shows."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    dy = (torch.randint(1, 4, (n, stride), generator=gen, device=cuda) * (1 - 2 * torch.randint(0, 2, (n, stride), generator=gen, device=cuda))).to(dtype)[:, :out]
    x, w, b = torch.zeros((n, 8), device=cuda, dtype=dtype), torch.zeros((out, 8), device=cuda, dtype=dtype), torch.zeros(out, device=cuda, dtype=dtype, requires_grad=True)
    g, = torch.autograd.grad(fastgl.linear(x, w, b), b, dy)
    assert torch.equal(g, dy.double().sum(0).float().to(dtype))


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_keeps_nothing_of_the_input(cuda, act, keep8):
    x, w, b, dy = problem(cuda, 20_000, 512, 16, torch.float32)
    h = x * 1
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = fastgl.linear(h, w, b, act, keep8=keep8)
    room = 20_000 * 16 * 4
    assert torch.cuda.memory_allocated() - before < (2.5 if act else 1.5) * room  # (the output, and behind an activation its derivative)
    want, = torch.autograd.grad(fastgl.linear(x, w.clone().requires_grad_(), b, act, keep8=keep8), b, dy)
    h.add_(1)  # (nobody reads it any more)
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got, = torch.autograd.grad(y, b, dy)
    assert torch.equal(got, want)
    assert torch.cuda.max_memory_allocated() - held < (2.5 if act else 1) * room + (1 << 20)  # (no gradient of the weight)


def test_residual_alone_keeps_nothing(cuda):
    x, w, b, dy = problem(cuda, 20_000, 64, 64, torch.float32)
    b, r = b.detach(), torch.randn((20_000, 64), device=cuda, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = fastgl.linear(x, w, b, "gelu", r, keep8=True)
    assert torch.cuda.memory_allocated() - before < 1.5 * 20_000 * 64 * 4  # (the output)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)
    with torch.no_grad():
        assert torch.equal(fastgl.linear(x, w, b, "gelu", r), y)


def test_captured(cuda):
    x, w, b, dy = problem(cuda, 3000, 100, 130, torch.float32)

    def step():
        return torch.autograd.grad(fastgl.linear(x, w, b, "relu", keep8=True), b, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=cuda).manual_seed(seed), device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_many_gradients_at_once(cuda):
    x, w, b, _ = problem(cuda, 9, 20, 6, torch.float32)
    y = fastgl.linear(x, w, b, "gelu", keep8=True)
    many = torch.randn((5, 9, 6), device=cuda)
    got, = torch.autograd.grad(y, b, many, is_grads_batched=True, retain_graph=True)
    for i in range(5):
        assert torch.equal(got[i], torch.autograd.grad(y, b, many[i], retain_graph=True)[0])


@pytest.mark.parametrize("act", [0, 1, 3])
@pytest.mark.parametrize("code,dtype", [(0, torch.float32), (1, torch.bfloat16)])
@pytest.mark.parametrize("n,d,out", [(1, 1, 1), (37, 47, 33), (2500, 100, 130), (9001, 600, 257)])
def test_entry_point_without_the_input(cuda, act, code, dtype, n, d, out):
    """Neither x nor 8 bits of it: the state of a forward pass without keep8, workspaces to the byte and full of no numbers, nothing written past the outputs."""
    from fastgl import _lib as L

    lib = L.lib()
    gen = torch.Generator(device=cuda).manual_seed(n)
    even, wide = d + d % 2, out + out % 2
    x, w, dy = (torch.randn(s, generator=gen, device=cuda).to(dtype) for s in ((n, even), (out, even), (n, wide)))
    y = torch.empty((n, out), device=cuda, dtype=dtype)
    for keep8 in (0, 1):
        held = []
        for kept, need_w in ((keep8, 1), (keep8, 0), (0, 0)):
            size = lib.fgl_linear_state_bytes(n, d, out, code, act, kept)
            room = lib.fgl_linear_workspace_bytes(n, d, out, code, act, keep8, need_w, 1)
            state, ws = (torch.full((b + 256,), 255, device=cuda, dtype=torch.uint8) for b in (size, room))
            db, dw, dx = (torch.full((c + 64,), 7.0, device=cuda, dtype=dtype) for c in (out, out * d, n * d))
            L.check(lib.fgl_linear(x.data_ptr(), even, w.data_ptr(), even, None, None, 0, n, d, out, code, act, kept, y.data_ptr(), out, state.data_ptr(), size, L.stream_handle()))
            L.check(lib.fgl_linear_backward(dy.data_ptr(), wide, x.data_ptr() if need_w else None, even if need_w else 0, w.data_ptr(), even, n, d, out, code, act, keep8,
                                            state.data_ptr(), size, dx.data_ptr(), d, dw.data_ptr() if need_w else None, db.data_ptr(), ws.data_ptr(), room, L.stream_handle()))
            assert (state[size:] == 255).all() and (ws[room:] == 255).all() and (db[out:] == 7).all() and (dx[n * d:] == 7).all()
            held.append((db[:out].clone(), dx[:n * d].clone()))
        assert all(torch.equal(p, q) for one in held[1:] for p, q in zip(one, held[0])) and held[0][0].isfinite().all()
