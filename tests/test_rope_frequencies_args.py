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
