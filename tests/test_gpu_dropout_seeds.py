"""fastgl.dropout without a seed, and layers without one."""
import pytest
import torch

import fastgl

pytestmark = pytest.mark.gpu


def test_calls_without_a_seed_draw_one_each(cuda):
    x = torch.randn(40, 30, device=cuda)
    torch.manual_seed(3)
    a, b = fastgl.dropout(x, 0.5), fastgl.dropout(x, 0.5)
    torch.manual_seed(3)
    assert torch.equal(fastgl.dropout(x, 0.5), a) and not torch.equal(a, b) and torch.equal(fastgl.dropout(x, 0.5), b)
    # no draw where there is none to make
    state = torch.get_rng_state()
    assert torch.equal(fastgl.dropout(x, 0.0), x) and (fastgl.dropout(x, 1.0) == 0).all() and fastgl.dropout(x, 0.5, training=False) is x
    fastgl.dropout(x, 0.5, seed=7)
    assert torch.equal(torch.get_rng_state(), state)
    # the backward pass has the forward's
    y = x.clone().requires_grad_()
    out = fastgl.dropout(y, 0.5)
    g, = torch.autograd.grad(out, y, torch.ones_like(x))
    assert torch.equal(g != 0, out != 0)


def test_two_layers_without_a_seed_lose_different_elements(cuda):
    x = torch.ones(1000, device=cuda)
    first, second = fastgl.Dropout(0.5), fastgl.Dropout(0.5)
    # (the chance that they agree in every element: 2^-1000)
    assert not torch.equal(first(x), second(x))


def test_recomputed_for_the_backward_pass(cuda):
    """An activation checkpoint puts torch's generator back: a call without a seed draws the same one."""
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(50, 20, device=cuda, requires_grad=True)
    out = checkpoint(lambda t: fastgl.dropout(t, 0.5).sin(), x, use_reentrant=False)
    g, = torch.autograd.grad(out, x, torch.ones_like(x))
    assert torch.equal(g != 0, out != 0)


def test_compiled_without_a_seed(cuda):
    x = torch.ones(400, device=cuda)
    compiled = torch.compile(lambda t: fastgl.dropout(t * 2.0, 0.5) + 1.0, backend="eager")
    a, b = compiled(x), compiled(x)
    assert not torch.equal(a, b) and set(a.tolist()) == {1.0, 5.0}


def test_a_resumed_layer_draws_what_the_run_would_have(cuda):
    x = torch.ones(500, device=cuda)
    layer = fastgl.Dropout(0.5, seed=12)
    layer(x)
    state = layer.state_dict()
    want = [layer(x), layer(x)]
    resumed = fastgl.Dropout(0.5)
    resumed.load_state_dict(state)
    assert all(torch.equal(resumed(x), w) for w in want)


@pytest.mark.parametrize("activation", [None, torch.tanh, torch.nn.functional.relu])
@pytest.mark.parametrize("training", [False, True])
def test_an_activation_that_is_changed_is_the_one_that_is_taken(cuda, activation, training):
    edge_ptr, edge_src = fastgl.graph.rmat_csr(2000, 20000, seed=3, device=cuda)
    sampler = fastgl.FusedMapSampler([3, 3], rng_seed=1).set_graph(edge_ptr, edge_src)
    inputs, _, blocks = sampler.sample_blocks(None, torch.arange(50, dtype=torch.int32, device=cuda) * 31)
    x = torch.randn(inputs.numel(), 8, device=cuda)
    model = fastgl.SAGE(8, 16, 5, 2, dropout=0.5, dropout_seed=4).to(cuda).train(training)
    assert model.dropout.relu
    model.activation = activation
    with torch.no_grad():
        got = model(blocks, x)
        h = model.layers[0](blocks[0], x)
        h = h if activation is None else activation(h)
        h = fastgl.dropout(h, 0.5, seed=4, stream=0, training=training)
        assert torch.equal(got, model.layers[1](blocks[1], h))
        own = fastgl.Dropout(0.0, seed=1, relu=True)  # (a layer of the caller's is taken as it is)
        model.dropout, model.activation = own, None
        assert torch.equal(model(blocks, x), model.layers[1](blocks[1], model.layers[0](blocks[0], x).clamp(min=0)))
