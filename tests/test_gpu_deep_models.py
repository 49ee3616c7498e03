"""Norms, dense layers and 8 bits together as models use them: the feed-forward block and models with blocks and norms between their layers, against
torch's modules in 64 bits with the same parameters; what is kept of a forward pass; training by the command."""
import pytest
import torch
from torch.nn import functional as F

import fastgl
from held8 import held
from test_gpu_train import load_train

pytestmark = pytest.mark.gpu


def plain_block(block, x, keep8=False):
    """The block in torch's operators in 64 bits; with keep8 the weights' gradients and the norm's are of the held values."""
    as_held = lambda t: t if not keep8 else t + (torch.from_numpy(held(t.detach().cpu().numpy())).to(t.device) - t).detach()  # noqa: E731

    class Held(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t, w, b):
            ctx.save_for_backward(as_held(t), w)
            return t @ w.t() + b

        @staticmethod
        def backward(ctx, g):
            t, w = ctx.saved_tensors
            return g @ w, g.t() @ t, g.sum(0)

    class HeldNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t, w, b, eps):
            c = t - t.mean(1, keepdim=True)
            r = torch.rsqrt(c.square().mean(1, keepdim=True) + eps)
            ctx.save_for_backward(as_held(c * r), r, w)
            return c * r * w + b

        @staticmethod
        def backward(ctx, g):
            h, r, w = ctx.saved_tensors
            gw = g * w
            return r * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True)), (g * h).sum(0), g.sum(0), None

    n, u, d = block.norm, block.up, block.down
    p = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
    h = HeldNorm.apply(x, p["norm.weight"], p["norm.bias"], n.eps)
    h = {"gelu": F.gelu, "silu": F.silu, "relu": torch.relu, None: lambda t: t}[u.activation](Held.apply(h, p["up.weight"], p["up.bias"]))
    assert d.activation is None
    return x + Held.apply(h, p["down.weight"], p["down.bias"]), p


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("n,d,hidden", [(1, 16, 32), (700, 47, 130), (9000, 256, 512), (20_000, 64, 100)])
def test_feed_forward_block(cuda, keep8, n, d, hidden):
    torch.manual_seed(n)
    block = fastgl.FeedForward(d, hidden, keep8=keep8).to(cuda)
    with torch.no_grad():
        block.norm.weight.add_(0.2 * torch.randn_like(block.norm.weight))
        block.norm.bias.add_(0.2 * torch.randn_like(block.norm.bias))
    x = torch.randn((n, d), device=cuda, requires_grad=True)
    g = torch.randn((n, d), device=cuda)
    y = block(x)
    got = torch.autograd.grad(y, [x, *block.parameters()], g)
    X = x.detach().double().requires_grad_()
    want_y, p = plain_block(block, X, keep8)
    want = torch.autograd.grad(want_y, [X, *p.values()], g.double())
    # fp32 sums of at most 512 (rows) and n terms in pairs of tens: 2-norms to 2e-6.  With keep8 a layer's input is off by that, and a value next to the middle of two
    # steps may be held as the other: a share of about 2^7 2^-22 of the values, each by a step of 2^-6, sqrt(2^-15) 2^-6 = 1e-4 of the weights' gradients behind them.
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y, want_y) < 2e-6
    # The norm's gradients are sums over rows of terms of both signs, dz W of the first layer (times h): dz is off by 8 U and the error function's 1.5e-7 beside a slope of at
    # most 1.13, of which 4 in z, and hidden terms add (hidden + 8) U, together less than 1e-6 + (hidden + 8) U of the terms' magnitudes, which do not cancel.
    with torch.no_grad():
        dh = (g.double() @ p["down.weight"]).abs() * 1.13 @ p["up.weight"].abs()
        terms = (1e-6 + (hidden + d + 8) * 2.0 ** -24) * dh.sum(0)
        c = X - X.mean(1, keepdim=True)
        h = (c * torch.rsqrt(c.square().mean(1, keepdim=True) + block.norm.eps)).abs()
        terms = {"norm.bias": terms, "norm.weight": (1e-6 + (hidden + d + 8) * 2.0 ** -24) * (dh * h).sum(0)}
    for (name, a), b in zip([("x", got[0]), *zip(p, got[1:])], want):
        most = (1e-4 if keep8 and name in ("up.weight", "down.weight") else 4e-6) * float(b.norm()) + (float(terms[name].norm()) if name in terms else 0.0)
        assert float((a.double() - b).norm()) < most, name


def test_feed_forward_block_in_bf16(cuda):
    torch.manual_seed(1)
    block = fastgl.FeedForward(100, 256, activation="relu", keep8=True).to(cuda).bfloat16()
    x = torch.randn((5000, 100), device=cuda).bfloat16().requires_grad_()
    y = block(x)
    got = torch.autograd.grad(y, [x, *block.parameters()], torch.ones_like(y))
    X = x.detach().double().requires_grad_()
    want_y, p = plain_block(block, X)
    want = torch.autograd.grad(want_y, [X, *p.values()], torch.ones_like(want_y))
    for a, b in zip((y, *got), (want_y, *want)):  # (three roundings to bf16 in a row, and 8 bits)
        assert float((a.double() - b).norm() / b.norm()) < 0.02


def test_what_is_kept(cuda):
    n, d, hidden = 40_000, 256, 512
    x = torch.randn((n, d), device=cuda, requires_grad=True)
    kept = []
    for keep8 in (False, True):
        block = fastgl.FeedForward(d, hidden, activation="relu", keep8=keep8).to(cuda)
        before = torch.cuda.memory_allocated()
        y = block(x)
        kept.append(torch.cuda.memory_allocated() - before - y.numel() * 4)
        y.sum().backward()
        del y, block
    # the norm's output and the activation's in full, or 33 / 32 bytes a value of them and of the normed rows; a bit a value of the hidden ones for relu, 12 or 4 bytes a row
    # (torch's allocator hands out cached blocks up to 1 MiB larger than what is asked for as they are; five of them are kept at most)
    assert kept[0] < n * (4 * d + 4 * hidden + hidden // 8 + 12) + 5 * 2 ** 20 and kept[1] < n * ((2 * d + hidden) * 33 // 32 + hidden // 8 + 4) + 5 * 2 ** 20
    assert kept[1] < 0.4 * kept[0]


def sampled(cuda, seed=3):
    edge_ptr, edge_src = fastgl.graph.rmat_csr(20_000, 200_000, seed=0, device=cuda)
    sampler = fastgl.FusedMapSampler([5, 5, 4], rng_seed=seed, deterministic=True).set_graph(edge_ptr, edge_src)
    seeds = torch.randperm(20_000, generator=torch.Generator().manual_seed(seed))[:700].int().to(cuda)
    return sampler.sample_blocks(None, seeds)


@pytest.mark.parametrize("name", ["gcn", "gin", "sage"])
@pytest.mark.parametrize("norm,feed_forward", [("layer", 0), (None, 96), ("layer", 96)])
def test_models(cuda, name, norm, feed_forward):
    train = load_train()
    input_nodes, output_nodes, blocks = sampled(cuda)
    feat = torch.randn((20_000, 40), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    x = feat.index_select(0, input_nodes.long())
    torch.manual_seed(2)
    model = train.build_model(name, 40, 64, 7, 3, 0.0, None, norm, feed_forward).to(cuda)
    call = lambda m: m(blocks, x) if name == "sage" else m(blocks, x, neighbor_list=[5, 5, 4])  # noqa: E731
    y = call(model)
    d = torch.randn_like(y)
    grads = torch.autograd.grad(y, list(model.parameters()), d)

    # the same with torch's modules between the layers
    torch.manual_seed(2)
    other = train.build_model(name, 40, 64, 7, 3, 0.0, None, norm, feed_forward).to(cuda)

    class Block(torch.nn.Module):
        def __init__(self, of):
            super().__init__()
            self.of = of

        def forward(self, h):
            of = self.of
            t = F.layer_norm(h, (h.size(1),), of.norm.weight, of.norm.bias, of.norm.eps)
            return h + F.linear(F.gelu(F.linear(t, of.up.weight, of.up.bias)), of.down.weight, of.down.bias)

    class Norm(torch.nn.Module):
        def __init__(self, of):
            super().__init__()
            self.of = of

        def forward(self, h, relu=False):
            t = F.layer_norm(h, (h.size(1),), self.of.weight, self.of.bias, self.of.eps)
            return torch.relu(t) if relu else t

    leaves = list(other.parameters())
    if feed_forward:
        other.blocks_between = torch.nn.ModuleList(map(Block, other.blocks_between))
    if norm:
        other.norms = torch.nn.ModuleList(map(Norm, other.norms))
    z = call(other)
    want = torch.autograd.grad(z, leaves, d)
    assert float((y - z).norm() / z.norm()) < 2e-5
    for a, b in zip(grads, want):  # (sums over thousands of rows in two orders; relu's border)
        assert float((a - b).norm()) < 2e-3 * float(b.norm()) + 1e-5


@pytest.mark.parametrize("name", ["gcn", "gin", "sage"])
@pytest.mark.parametrize("dropout_seed", [None, 5])
def test_gradients_with_8_bits_are_near_those_without(cuda, name, dropout_seed):
    train = load_train()
    input_nodes, output_nodes, blocks = sampled(cuda)
    x = torch.randn((input_nodes.numel(), 40), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    got = []
    for keep8 in (False, True):
        torch.manual_seed(2)
        model = train.build_model(name, 40, 64, 7, 3, 0.3 if dropout_seed else 0.0, dropout_seed, "layer", 96, keep8).to(cuda)
        y = model(blocks, x) if name == "sage" else model(blocks, x, neighbor_list=[5, 5, 4])
        got.append((y.detach(), torch.autograd.grad(y, list(model.parameters()), torch.ones_like(y))))
    assert torch.equal(got[0][0], got[1][0])  # (the forward pass is the same)
    for a, b in zip(got[0][1], got[1][1]):  # (held values are off by 2^-7 of their 32's largest at most, about a quarter of that in the mean square)
        assert float((a - b).norm()) < 0.05 * float(a.norm()) + 1e-5


@pytest.mark.parametrize("model", ["sage", "gcn"])
def test_training_by_the_command(cuda, model, tmp_path):
    train = load_train()
    args = train.parse_args(["--model", model, "--nodes", "20000", "--draws", "200000", "--feat_dim", "32", "--classes", "4", "--num_hidden", "32", "--batch_size", "512",
                             "--fanout", "5", "5", "--num_epoch", "1", "--train_frac", "0.2", "--dropout", "0.2", "--dropout_seed", "3", "--norm", "layer", "--feed_forward", "64",
                             "--keep8", "1"])
    result, losses = train.run(args)
    assert all(x == x and x < 1e3 for x in losses)
    with pytest.raises(ValueError):
        train.build_model("gat", 8, 8, 4, 2, 0.0, None, "layer")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 15, 17, 700, 13_001])
def test_memory_that_held_something_else(cuda, dtype, n):
    """States, workspaces and outputs come from torch's cache with whatever was there: not a number in all of it changes nothing."""
    torch.manual_seed(n)
    block = fastgl.FeedForward(100, 260, keep8=True).to(cuda).to(dtype)
    x = torch.randn((n, 100), device=cuda).to(dtype).requires_grad_()
    d = torch.randn((n, 100), device=cuda).to(dtype)
    step = lambda: (lambda y: [y.detach(), *torch.autograd.grad(y, [x, *block.parameters()], d)])(block(x))  # noqa: E731
    runs = []
    for fill in (0.0, float("nan"), 3e38):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        held = [torch.full((size,), fill, device=cuda) for size in (1 << 26, 1 << 17, 1 << 17, 1 << 17, 100, 100, 100, 100)]
        del held
        runs.append(step())
    assert all(torch.equal(p, q) for r in runs[1:] for p, q in zip(runs[0], r)) and all(t.isfinite().all() for t in runs[0])


def test_nothing_is_written_past_the_outputs(cuda):
    from fastgl import _lib as L

    lib = L.lib()
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for n, d, out in ((1, 1, 1), (37, 47, 33), (130, 64, 96), (2500, 100, 130), (26_000, 130, 128)):
            size = torch.finfo(dtype).bits // 8
            even = d + d % 2
            x = torch.zeros((n, even), device=cuda, dtype=dtype)
            w = torch.randn((out, even), device=cuda).to(dtype)
            x[:, :d] = torch.randn((n, d), device=cuda).to(dtype)
            dy = torch.randn((n, out + out % 2), device=cuda).to(dtype)

            def guarded(count, of=dtype):
                t = torch.full((count + 256,), 7.0, device=cuda, dtype=of) if of != torch.uint8 else torch.full((count + 4096,), 77, device=cuda, dtype=of)
                return t

            for act in (0, 1, 2):
                for keep8 in (0, 1):
                    state_bytes = lib.fgl_linear_state_bytes(n, d, out, code, act, keep8)
                    ws_bytes = lib.fgl_linear_workspace_bytes(n, d, out, code, act, keep8, 1, 1)
                    y, dx, dw, db = guarded(n * out), guarded(n * d), guarded(out * d), guarded(out)
                    state, ws = guarded(state_bytes, torch.uint8), guarded(ws_bytes, torch.uint8)
                    L.check(lib.fgl_linear(x.data_ptr(), even, w.data_ptr(), even, None, None, 0, n, d, out, code, act, keep8, y.data_ptr(), out, state.data_ptr(), state_bytes,
                                           L.stream_handle()))
                    L.check(lib.fgl_linear_backward(dy.data_ptr(), out + out % 2, x.data_ptr(), even, w.data_ptr(), even, n, d, out, code, act, keep8, state.data_ptr(), state_bytes,
                                                    dx.data_ptr(), d, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws_bytes, L.stream_handle()))
                    for t, used in ((y, n * out), (dx, n * d), (dw, out * d), (db, out)):
                        assert (t[used:] == 7.0).all() and t[:used].isfinite().all()
                    assert (state[state_bytes:] == 77).all() and (ws[ws_bytes:] == 77).all()
            for relu in (0, 1):
                for keep8 in (0, 1):
                    state_bytes, ws_bytes = lib.fgl_layer_norm_state_bytes(n, d, relu, keep8), lib.fgl_layer_norm_workspace_bytes(n, d, code)
                    y, dx, dw, db = guarded(n * d), guarded(n * d), guarded(d), guarded(d)
                    state, ws = guarded(state_bytes, torch.uint8), guarded(ws_bytes, torch.uint8)
                    L.check(lib.fgl_layer_norm(x.data_ptr(), even, None, None, n, d, code, 1e-5, relu, keep8, y.data_ptr(), state.data_ptr(), state_bytes, L.stream_handle()))
                    L.check(lib.fgl_layer_norm_backward(x.data_ptr(), even, x.data_ptr(), even, None, n, d, code, relu, keep8, state.data_ptr(), state_bytes, dx.data_ptr(),
                                                        dw.data_ptr(), db.data_ptr(), ws.data_ptr(), ws_bytes, L.stream_handle()))
                    for t, used in ((y, n * d), (dx, n * d), (dw, d), (db, d)):
                        assert (t[used:] == 7.0).all() and t[:used].isfinite().all()
                    assert (state[state_bytes:] == 77).all() and (ws[ws_bytes:] == 77).all()


def test_compiled_modules(cuda):
    """The compiler breaks its graph at the kernels' calls and makes them as they are."""
    torch.manual_seed(4)
    block = fastgl.FeedForward(48, 96).to(cuda)
    x = torch.randn((300, 48), device=cuda, requires_grad=True)
    d = torch.randn_like(x)
    y = block(x)
    want = torch.autograd.grad(y, [x, *block.parameters()], d)
    z = torch.compile(block, backend="eager")(x)
    got = torch.autograd.grad(z, [x, *block.parameters()], d)
    assert torch.equal(y, z) and all(torch.equal(p, q) for p, q in zip(got, want))


def test_computed_anew_for_the_backward_pass(cuda):
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(5)
    block = fastgl.FeedForward(48, 96, keep8=True).to(cuda)
    x = torch.randn((300, 48), device=cuda, requires_grad=True)
    d = torch.randn_like(x)
    want = torch.autograd.grad(block(x), [x, *block.parameters()], d)
    y = checkpoint(block, x, use_reentrant=False)
    got = torch.autograd.grad(y, [x, *block.parameters()], d)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_two_captured_steps(cuda):
    """Two graphs of steps over the same parameters, replayed in turn with eager steps in between."""
    torch.manual_seed(6)
    block = fastgl.FeedForward(64, 128, keep8=True).to(cuda)
    inputs = [torch.randn((n, 64), device=cuda, requires_grad=True) for n in (300, 5000)]
    grads = [torch.randn_like(t) for t in inputs]
    step = lambda i: (lambda y: [y.detach(), *torch.autograd.grad(y, [inputs[i], *block.parameters()], grads[i])])(block(inputs[i]))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for turn in range(3):
        with torch.no_grad():
            for t in inputs:
                t.copy_(torch.randn(t.shape, generator=torch.Generator(device=cuda).manual_seed(turn), device=cuda))
        for i in (turn % 2, 1 - turn % 2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(p, q) for p, q in zip(outs[i], step(i)))
