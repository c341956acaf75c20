"""Rows of ``lucid_amd.model_ops.token_logprobs`` whose masks are finite values, between those that a model's logits
reach and the type's lowest (-1e6 .. -1e36), and finite logits that are as large: definition, tolerances and checks
of ``test_token_logprobs_gpu``.

A log probability of a masked value v is v / temperature - lse: relatively exact to 2^-22 (the temperature's inverse, the
difference and the product, 2^-24 each) as every other one.
"""
import pytest
import torch

from test_token_logprobs_gpu import _run

pytestmark = pytest.mark.gpu

MASKS = [-1e6, -1e9, -5e9, -1e10, -1e20, -1e30, -1e36]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
@pytest.mark.parametrize("V", [40, 3000, 32003, 40000])
@pytest.mark.parametrize("top", [0, 5])
def test_finite_masks(V, temperature, dtype, top):
    """A few allowed tokens (their waves beside waves that are masked as a whole), half of the row, whole segments, and
    whole rows of the mask's value."""
    print(f"case finite masks V={V} T={temperature} {dtype} top={top}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V + top)
    for mask in MASKS:
        x = 2 * torch.randn(5, V, generator=g, device="cuda")
        x[0, 7:] = mask
        x[1, :V - 3] = mask
        x[2, torch.rand(V, generator=g, device="cuda") < 0.5] = mask
        x[3] = mask
        x[4, V // 3:] = mask
        x = x.to(dtype)
        tokens = x.argmax(-1)
        tokens[4] = V - 1  # a masked token is given
        _run(x, tokens, top, temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_finite_logits(dtype):
    """Rows around large values of either sign: one maximum takes all, or several equal ones share."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for size in (1e6, 1e7, 5e9, 1e20, 1e36):
        x = size * torch.randn(4, 9001, generator=g, device="cuda")
        x[2, ::1000] = 8 * size
        x[3] = -size
        _run(x.to(dtype), x.argmax(-1), 5, 1.0)


def test_small_temperatures():
    """Ordinary logits whose quotients by the temperature are large (multiples of 1/32: a probability is that of a
    maximum or below e^-312, none where fp32 goes below its normal numbers)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = (96 * torch.randn(4, 9001, generator=g, device="cuda")).round() / 32
    x[1] -= 200.0
    for temperature in (1e-4, 1e-6, 1e-12):
        _run(x, x.argmax(-1), 3, temperature)
