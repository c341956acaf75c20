"""Results of ``rotary`` that are changed in place, with and without a gradient.  Reference and tolerances are those of
test_rotary_gpu.py; the factor 0.5 is exact."""
import pytest
import torch

from test_rotary_gpu import BF, F32, close, make, ref

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_results_may_be_changed_in_place(dtype):
    q, k = make(2, 21, 4, 2, 68, dtype)
    pos, freq = torch.arange(21, device="cuda") * 50, O.rope_frequencies(68)[0].cuda()
    g = torch.randn(2, 4, 21, 68, device="cuda").to(dtype)
    x, y = (t.detach().requires_grad_() for t in (q, k))
    a, b = O.rotary(x, y, pos, freq)
    a.mul_(0.5)
    b[:, :, 3:].zero_()
    dq, dk = torch.autograd.grad((a, b), (x, y), (g, g[:, :2]))
    cut = g[:, :2].clone()
    cut[:, :, 3:] = 0
    close(dq, ref(0.5 * g.double(), pos, freq, False, 1.0, True), "dq")
    close(dk, ref(cut, pos, freq, False, 1.0, True), "dk")
    with torch.no_grad():
        c, d = O.rotary(q, k, pos, freq)
        c.mul_(0.5)
    assert torch.equal(a, c)
    want = ref(q, pos, freq, False, 1.0)
    close(a, (0.5 * want[0], 0.5 * want[1]), "q")
    for t, h in ((a, 4), (b, 2), (dq, 4), (dk, 2), (c, 4), (d, 2)):  # laid out by tokens, as the projections are
        assert t.stride() == (21 * h * 68, 68, h * 68, 1)
