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
