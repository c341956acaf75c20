"""Rows of ``lucid_amd.model_ops.token_logprobs`` whose masks are finite values, between those that a model's logits
reach and the type's lowest (-1e6 .. -1e36), and finite logits that are as large: definition, tolerances and checks
of ``test_token_logprobs_gpu``.

A log probability of a masked value v is v / temperature - lse: relatively exact to 2^-22 (the temperature's inverse, the
difference and the product, 2^-24 each) as every other one.
"""
import pytest
import torch

from lucid_amd.model_ops import token_logprobs
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,top", [(50, 0), (9001, 4), (40000, 4)])
def test_ignored_rows_without_a_distribution_have_no_gradient(V, top, dtype):
    """A token of -100 has no gradient, whatever its row holds: nothing allowed, a NaN, an infinity.  With a gradient of
    the entropy or of an alternative such a row gives NaN, as ever, and the rows beside it are not affected."""
    print(f"case ignored rows V={V} top={top} {dtype}", flush=True)
    x0 = torch.randn(4, V, device="cuda").to(dtype)
    x0[0] = float("-inf")
    x0[1, V // 2] = float("nan")
    x0[2, V - 1] = float("inf")
    tokens = torch.tensor([-100, -100, -100, 3], device="cuda")
    x = x0.clone().requires_grad_()
    r = token_logprobs(x, tokens, top=top)
    assert r.logprobs[:3].tolist() == [0.0, 0.0, 0.0]
    dx, = torch.autograd.grad(r.logprobs.sum(), x, retain_graph=True)
    assert bool((dx[:3] == 0).all()) and bool((dx[3] != 0).any()) and bool(torch.isfinite(dx[3]).all())
    one = torch.tensor([1.0, 0.0, 0.0, 0.0], device="cuda")
    dx, = torch.autograd.grad(r.entropy, x, one, retain_graph=True)
    assert bool(torch.isnan(dx[0]).any()) and bool((dx[1:] == 0).all())
    if top:
        g = torch.zeros(4, top, device="cuda")
        g[1, 1], g[1, 2] = 1.0, -1.0
        dx, = torch.autograd.grad(r.top_logprobs, x, g)
        assert bool(torch.isnan(dx[1]).any()) and bool((dx[0] == 0).all()) and bool((dx[2:] == 0).all())
