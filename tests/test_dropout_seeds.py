"""Seeds of fastgl.dropout and fastgl.Dropout: where none is given, one is drawn from torch's generator, and layers do not share it."""
import copy
import pickle

import pytest
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


def test_seeds_outside_64_bits_are_refused():
    for seed in (-1, 2 ** 64):
        with pytest.raises(ValueError, match="64 bits"):
            fastgl.Dropout(0.5, seed=seed)
        with pytest.raises(ValueError, match="64 bits"):
            fastgl.SAGE(4, 4, 4, 2, dropout=0.5, dropout_seed=seed)


@pytest.mark.parametrize("seed", [0, 7, 2 ** 63, 2 ** 64 - 1])
def test_a_saved_layer_goes_on_with_the_next_stream(seed, tmp_path):
    layer = fastgl.Dropout(0.5, seed=seed)
    layer.calls = 41
    torch.save(layer.state_dict(), tmp_path / "state.pt")
    other = fastgl.Dropout(0.5)
    other.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    assert (other.seed, other.calls) == (seed, 41)
    again = copy.deepcopy(layer)
    assert (again.seed, again.calls) == (seed, 41)


def test_states_of_models_with_and_without_a_seed():
    make = lambda **seed: fastgl.SAGE(4, 5, 3, 3, dropout=0.5, **seed)  # noqa: E731
    seeded, plain = make(dropout_seed=9), make()
    seeded.dropout.calls = 6
    assert all(isinstance(v, torch.Tensor) for v in seeded.state_dict().values())
    assert set(seeded.state_dict()) == set(plain.state_dict()) | {"dropout._extra_state"}
    state = seeded.state_dict()
    plain.load_state_dict(state)  # (strict)
    assert "dropout._extra_state" in state  # (the caller's is left as it was)
    assert torch.equal(plain.layers[0].fc_self.weight, seeded.layers[0].fc_self.weight)
    seeded.load_state_dict(make().state_dict())
    assert (seeded.dropout.seed, seeded.dropout.calls) == (9, 6)
    resumed = make(dropout_seed=9)
    resumed.load_state_dict(seeded.state_dict())
    assert resumed.dropout.calls == 6
    with pytest.raises(RuntimeError):  # (what is missing elsewhere is still missed)
        resumed.load_state_dict({"dropout._extra_state": state["dropout._extra_state"]})
    copied = pickle.loads(pickle.dumps(plain))
    copied.load_state_dict(state)
