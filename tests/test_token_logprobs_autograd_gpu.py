"""Modes of differentiation beside the backward pass: ``lucid_amd.model_ops.token_logprobs`` has no forward-mode
derivative, and says so instead of leaving a tangent out."""
import pytest
import torch
from torch.autograd import forward_ad

from lucid_amd.model_ops import token_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(grad):
    x = torch.randn(3, 500, device="cuda", requires_grad=grad)
    tokens = torch.tensor([4, -100, 7], device="cuda")
    want = token_logprobs(x.detach(), tokens, top=2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.randn_like(x))
        with pytest.raises(NotImplementedError):
            token_logprobs(dual, tokens, top=2)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            token_logprobs(dual, tokens, top=2)
        # logits without a tangent are as ever, inside the level too
        got = token_logprobs(dual.detach(), tokens, top=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(t.grad_fn is None for t in got)
