"""Dropout from a seed and the loss of a last layer where they are used: between and behind a model's layers, in a captured training step, and
in the trainer."""
import importlib.util
import os
import threading

import pytest
import torch

import fastgl
from conftest import ROOT

pytestmark = pytest.mark.gpu


def batch(cuda, fanouts, n=600, nodes=20_000):
    edge_ptr, edge_src = fastgl.graph.rmat_csr(nodes, nodes * 10, seed=3, device=cuda)
    sampler = fastgl.FusedMapSampler(fanouts, rng_seed=1, deterministic=True).set_graph(edge_ptr, edge_src)
    seeds = (torch.arange(n, dtype=torch.int32, device=cuda) * 31) % nodes
    return sampler.sample_blocks(None, seeds)


def model_of(kind, cuda, dtype, seed=7):
    torch.manual_seed(0)
    args = (24, 40, 40, 3)
    if kind == "sage":
        m = fastgl.SAGE(*args, dropout=0.4, dropout_seed=seed)
    else:
        m = {"gcn": fastgl.GCN, "gin": fastgl.GIN}[kind](*args, None, True, 0.4, dropout_seed=seed)
    return m.to(cuda).to(dtype), fastgl.LinearCrossEntropy(40, 300).to(cuda).to(dtype)


def call(kind, model, blocks, x):
    return model(blocks, x) if kind == "sage" else model(blocks, x, [5, 5, 5])


class Restated(torch.nn.Module):
    """The same masks by torch's operators: of ones, an element is kept where the result is not zero."""

    def __init__(self, p, seed, relu):
        super().__init__()
        self.p, self.seed, self.relu, self.calls = p, seed, False, 0
        self.with_relu = relu

    def forward(self, h):
        mask = fastgl.dropout(torch.ones_like(h), self.p, seed=self.seed, stream=self.calls) != 0
        self.calls += 1
        return torch.where(mask, (torch.relu(h) if self.with_relu else h) * (1.0 / (1.0 - self.p)), 0.0)


@pytest.mark.parametrize("kind", ["gcn", "gin", "sage"])
def test_step_of_a_model_against_its_restatement(cuda, kind):
    input_nodes, output_nodes, blocks = batch(cuda, [5, 5, 5])
    x = torch.randn((input_nodes.numel(), 24), generator=torch.Generator(device=cuda).manual_seed(5), device=cuda)
    y = (output_nodes.long() * 7) % 300
    y[::9] = -100
    model, head = model_of(kind, cuda, torch.float32)
    params = [*model.parameters(), *head.parameters()]
    loss = head(call(kind, model, blocks, x), y)
    grads = torch.autograd.grad(loss, params)
    assert model.dropout.calls == 2
    model.dropout = Restated(0.4, 7, kind == "sage")
    if kind == "sage":
        model.activation = None
    rows = call(kind, model, blocks, x)
    logits = torch.nn.functional.linear(rows.double(), head.weight.double(), head.bias.double())
    want = torch.nn.functional.cross_entropy(logits, y)
    want_grads = torch.autograd.grad(want, params)
    # The layers are the same kernels on the same bits on both sides, so what differs is the loss's own rounding and what the layers' backward
    # passes make of it: fp32 sums of at most a few thousand terms in each of four products, each within 2^-24 sqrt(5000) < 2^-17 of its
    # largest result, which the next one carries on: 2^-15 in all.
    assert abs(float(loss.detach()) - float(want.detach())) <= 2.0 ** -17 * float(want.detach())
    for g, w in zip(grads, want_grads):
        assert (g - w).abs().max() <= 2.0 ** -15 * w.abs().max()


@pytest.mark.parametrize("kind", ["gcn", "sage"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_training_step(cuda, kind, dtype):
    input_nodes, output_nodes, blocks = batch(cuda, [5, 5, 5])
    fastgl.transpose_blocks(blocks[1:])
    x = torch.randn((input_nodes.numel(), 24), generator=torch.Generator(device=cuda).manual_seed(5), device=cuda).to(dtype)
    y = (output_nodes.long() * 7) % 300
    model, head = model_of(kind, cuda, dtype)
    offset = torch.zeros(1, dtype=torch.int32, device=cuda)
    model.dropout.stream_offset = offset

    def step():
        model.dropout.calls = 0
        loss = head(call(kind, model, blocks, x), y)
        return loss.detach(), torch.autograd.grad(loss, [*model.parameters(), *head.parameters()])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    seen = set()
    for k in range(4):
        offset.fill_(2 * k)  # (two calls a replay)
        graph.replay()
        torch.cuda.synchronize()
        want, want_grads = step()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and all(torch.equal(p, q) for p, q in zip(grads, want_grads))
        seen.add(float(loss))
    assert len(seen) == 4


def test_models_without_a_seed_are_what_they_were(cuda):
    assert type(fastgl.GCN(8, 8, 4, 2, None, True, 0.5).dropout) is torch.nn.Dropout and type(fastgl.SAGE(8, 8, 4, 2, dropout=0.5).dropout) is torch.nn.Dropout
    # with one: evaluation has the activation, and nothing else
    input_nodes, _, blocks = batch(cuda, [5, 5, 5])
    x = torch.randn((input_nodes.numel(), 24), device=cuda)
    model, _ = model_of("sage", cuda, torch.float32)
    model.eval()
    torch.manual_seed(0)
    plain = fastgl.SAGE(24, 40, 40, 3, dropout=0.4).to(cuda).eval()
    with torch.no_grad():
        assert torch.equal(model(blocks, x), plain(blocks, x)) and model.dropout.calls == 0
    other = fastgl.SAGE(24, 40, 40, 3, activation=torch.tanh, dropout=0.4, dropout_seed=1)
    assert not other.dropout.relu


def load_train():
    spec = importlib.util.spec_from_file_location("fastgl_train", os.path.join(ROOT, "fastgl-ae_amd", "train.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("model", ["sage", "gcn", "gin", "gat"])
def test_trainer_with_seeded_dropout_and_a_linear_head(cuda, model):
    """Dropout on, and two runs from one seed give the same losses bit for bit (GAT has no dropout between layers: its head alone)."""
    print("train %s" % model, flush=True)
    train = load_train()
    argv = ["--model", model, "--nodes", "20000", "--draws", "200000", "--feat_dim", "32", "--classes", "500", "--num_hidden", "32", "--batch_size", "512",
            "--fanout", "5", "5", "--num_epoch", "1", "--train_frac", "0.2", "--dropout", "0.5", "--deterministic", "1", "--prefetch", "0", "--head", "linear"]
    if model != "gat":
        argv += ["--dropout_seed", "11"]
    _, a = train.run(train.parse_args(argv))
    _, b = train.run(train.parse_args(argv))
    assert a == b and len(a) > 4 and all(v == v for v in a)
    if model == "sage":
        argv[-1] = "12"
        assert train.run(train.parse_args(argv))[1] != a
    if model == "gat":
        with pytest.raises(ValueError):
            train.run(train.parse_args(argv + ["--dropout_seed", "11"]))


def test_compiled_modules_fall_back_to_the_operators(cuda):
    x = torch.randn((50, 24), device=cuda)
    y = torch.arange(50, device=cuda) % 9
    torch.manual_seed(0)
    head = fastgl.LinearCrossEntropy(24, 9).to(cuda)
    drop = fastgl.Dropout(0.5, seed=3, relu=True)

    def loss(h, labels):
        return head(drop(h * 2.0), labels) + 1.0

    want = loss(x, y)
    drop.calls = 0
    assert torch.equal(torch.compile(loss, backend="eager")(x, y), want)


def _ends(x, w, b, y, stream):
    """Dropout and loss, forward and backward: (loss, gradients)."""
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    h = fastgl.dropout(leaves[0], 0.4, 5, stream, relu=True)
    loss = fastgl.linear_cross_entropy(h, leaves[1], y, leaves[2])
    return [loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones((), device=x.device))]


def _some(cuda, k, dtype):
    gen = torch.Generator(device=cuda).manual_seed(k)
    n, v, d = 200 + 31 * k, 90 + 500 * k, 64 + 20 * k
    normal = lambda *s: torch.randn(s, generator=gen, device=cuda).to(dtype)  # noqa: E731
    return normal(n, d), normal(v, d) / 8, normal(v), torch.randint(0, v, (n,), generator=gen, device=cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_calls_of_several_threads_at_once(cuda, dtype):
    inputs = [_some(cuda, k, dtype) for k in range(4)]
    want = [_ends(*t, stream=k) for k, t in enumerate(inputs)]
    torch.cuda.synchronize()
    got, errors = [[] for _ in inputs], []

    def work(k):
        try:
            with torch.cuda.device(cuda), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[k].append(_ends(*inputs[k], stream=k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for k, runs in enumerate(got):
        assert len(runs) == 8 and all(torch.equal(p, q) for run in runs for p, q in zip(run, want[k]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_graphs_replayed_at_once(cuda, dtype):
    inputs = [_some(cuda, k, dtype) for k in (1, 3)]
    want = [_ends(*t, stream=k) for k, t in enumerate(inputs)]
    graphs, results = [], []
    for k, t in enumerate(inputs):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _ends(*t, stream=k)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(_ends(*t, stream=k))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for r in results:
            for t in r:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for r, e in zip(results, want) for p, q in zip(r, e))
        assert all(torch.equal(p, q) for k, t in enumerate(inputs) for p, q in zip(_ends(*t, stream=k), want[k]))
