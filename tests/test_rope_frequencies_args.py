"""What ``rope_frequencies`` makes of default devices and of entries of a scaling that it does not know (no GPU)."""
import math

import pytest
import torch

from lucid_amd.model_ops import rope_frequencies

SCALINGS = [None, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "ntk", "factor": 4.0},
            {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192},
            {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=str)
@pytest.mark.parametrize("dim", [0, 64])
def test_frequencies_are_on_the_cpu_whatever_the_default_device(scaling, dim):
    want, scale = rope_frequencies(dim, scaling=scaling)
    with torch.device("meta"):
        got, s = rope_frequencies(dim, scaling=scaling)
    assert got.device.type == "cpu" and torch.equal(got, want) and s == scale


@pytest.mark.parametrize("key", ["mscale", "mscale_all_dim", "truncate", "rope_theta", "short_factor", "beta_fats"])
@pytest.mark.parametrize("scaling", [{"rope_type": "default"}] + SCALINGS[1:], ids=str)
def test_entries_that_are_not_known_are_refused(scaling, key):
    """They would ask for another factor, ramp or base than they got."""
    with pytest.raises(ValueError, match=key):
        rope_frequencies(64, scaling=dict(scaling, **{key: 1.0}))


@pytest.mark.parametrize("scaling,key", [
    ({"rope_type": "linear", "factor": 4.0, "beta_fast": 32.0}, "beta_fast"),
    ({"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192, "attention_factor": 1.0}, "attention_factor"),
    ({"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, "low_freq_factor": 1.0}, "low_freq_factor"),
    ({"rope_type": "default", "factor": 8.0}, "factor"), ({"factor": 8.0}, "factor")], ids=str)
def test_entries_of_another_type_are_refused(scaling, key):
    with pytest.raises(ValueError, match=key):
        rope_frequencies(64, scaling=scaling)


def test_two_names_of_the_type():
    """"rope_type" and its older name may both be there, with one value."""
    both = {"rope_type": "linear", "type": "linear", "factor": 4.0}
    assert torch.equal(rope_frequencies(64, scaling=both)[0], rope_frequencies(64)[0] / 4)
    with pytest.raises(ValueError, match="type"):
        rope_frequencies(64, scaling=dict(both, type="ntk"))


def test_entries_without_a_value_are_as_if_not_there():
    yarn = dict(SCALINGS[4], attention_factor=None, beta_fast=None, beta_slow=None, mscale=None)
    got, want = rope_frequencies(64, scaling=yarn), rope_frequencies(64, scaling=SCALINGS[4])
    assert torch.equal(got[0], want[0]) and got[1] == want[1]
    with pytest.raises(ValueError, match="factor"):
        rope_frequencies(64, scaling={"rope_type": "linear", "factor": None})


def test_the_length_trained_on_may_go_with_every_type():
    """It says nothing to the types that do not use it, and configurations carry it beside them."""
    for scaling in SCALINGS[1:3]:
        got = rope_frequencies(64, scaling=dict(scaling, original_max_position_embeddings=4096))
        assert torch.equal(got[0], rope_frequencies(64, scaling=scaling)[0]) and math.isclose(got[1], 1.0)
