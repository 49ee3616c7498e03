"""Seeds of fastgl.dropout and fastgl.Dropout: where none is given, one is drawn from torch's generator, and layers do not share it."""
import torch

import fastgl
from fastgl import dropouts


def test_layers_without_a_seed_have_seeds_of_their_own():
    torch.manual_seed(5)
    seeds = [fastgl.Dropout(0.5).seed for _ in range(8)]
    assert len(set(seeds)) == 8 and all(0 <= s < 2 ** 64 for s in seeds)
    torch.manual_seed(5)
    assert [fastgl.Dropout(0.5).seed for _ in range(8)] == seeds
    assert fastgl.Dropout(0.5, seed=0).seed == 0


def test_seeds_are_numbers_where_tensors_hold_none():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        assert isinstance(dropouts._drawn_seed(), int)
    with torch.device("meta"):
        assert isinstance(fastgl.Dropout(0.5).seed, int)


def test_a_given_seed_draws_nothing():
    torch.manual_seed(5)
    state = torch.get_rng_state()
    fastgl.Dropout(0.5, seed=3)
    assert torch.equal(torch.get_rng_state(), state)
