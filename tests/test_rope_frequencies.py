"""``rope_frequencies`` against closed forms (no GPU)."""
import math

import pytest
import torch

from lucid_amd.model_ops import rope_frequencies


def test_default_linear_and_ntk():
    f, s = rope_frequencies(64)
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert f.dtype == torch.float64 and s == 1.0 and torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.equal(rope_frequencies(64, scaling={"rope_type": "default"})[0], f)
    assert torch.allclose(rope_frequencies(64, scaling={"type": "linear", "factor": 4})[0], f / 4, rtol=1e-15, atol=0)
    n, _ = rope_frequencies(64, scaling={"rope_type": "ntk", "factor": 8.0})
    assert n[0] == 1.0 and math.isclose(n[-1].item(), f[-1].item() / 8, rel_tol=1e-12)
    assert rope_frequencies(0)[0].numel() == 0


def test_llama3():
    L, factor = 8192, 8.0
    f, _ = rope_frequencies(128, 500000.0)
    g, s = rope_frequencies(128, 500000.0, {"rope_type": "llama3", "factor": factor, "low_freq_factor": 1.0,
                                            "high_freq_factor": 4.0, "original_max_position_embeddings": L})
    assert s == 1.0
    seen = set()
    for a, b in zip(f.tolist(), g.tolist()):
        wave = 2 * math.pi / a
        if wave < L / 4:
            want, kind = a, "stays"
        elif wave > L:
            want, kind = a / factor, "divided"
        else:
            smooth = (L / wave - 1.0) / 3.0
            want, kind = (1 - smooth) * a / factor + smooth * a, "between"
        seen.add(kind)
        assert math.isclose(b, want, rel_tol=1e-12)
    assert len(seen) == 3


def test_yarn():
    f, _ = rope_frequencies(64)
    g, s = rope_frequencies(64, scaling={"rope_type": "yarn", "factor": 32, "original_max_position_embeddings": 4096})
    assert math.isclose(s, 0.1 * math.log(32) + 1)
    turns = 4096 * f / (2 * math.pi)
    ratio = g / f
    assert bool((ratio[turns > 40] == 1).all())  # (the ramp's ends are whole pairs)
    assert torch.allclose(ratio[turns < 0.7], torch.full_like(ratio[turns < 0.7], 1 / 32), rtol=1e-12)
    assert bool((ratio.diff() <= 1e-15).all())  # falls from pair to pair
    assert rope_frequencies(64, scaling={"rope_type": "yarn", "factor": 32, "original_max_position_embeddings": 4096,
                                         "attention_factor": 1.5})[1] == 1.5


def test_refusals():
    for bad in ({"rope_type": "longrope"}, {"rope_type": "linear"}, {"rope_type": "yarn", "factor": 4.0},
                {"rope_type": "linear", "factor": 0.0}):
        with pytest.raises(ValueError, match="rope_frequencies"):
            rope_frequencies(64, scaling=bad)
    for dim in (-2, 3):
        with pytest.raises(ValueError, match="even"):
            rope_frequencies(dim)


@pytest.mark.parametrize("kind", ["llama3", "yarn"])
@pytest.mark.parametrize("length", [0, -8192, float("nan")])
def test_lengths_that_are_none_are_refused(kind, length):
    with pytest.raises(ValueError, match="original_max_position_embeddings"):
        rope_frequencies(64, 10000.0, {"rope_type": kind, "factor": 4.0, "original_max_position_embeddings": length})


@pytest.mark.parametrize("theta", [1.0, 0.5])
def test_yarn_without_a_spread_of_wavelengths_is_refused(theta):
    with pytest.raises(ValueError, match="theta"):
        rope_frequencies(64, theta, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
