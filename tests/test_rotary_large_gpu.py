"""Rotary results of 100 MB and more, which pass the caches by, in every layout and type, and ones that do not for their odd
widths; gradients too.  Reference and tolerances are those of test_rotary_gpu.py."""
import pytest
import torch

from test_rotary_gpu import BF, F32, close, make, ref

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,part", [(128, 128), (128, 64), (64, 64), (68, 68), (96, 24)])
def test_large_passes(d, part, inter, dtype):
    B, Hq, Hkv = 2, 24, 8
    T = 110_000_000 // (B * (Hq + Hkv) * d * (2 if dtype is BF else 4))
    print(f"case d={d} part={part} inter={inter} {dtype} T={T}", flush=True)
    q, k = make(B, T, Hq, Hkv, d, dtype)
    g = torch.randn(B, Hq, T, d, device="cuda").to(dtype)
    pos = torch.randint(0, 131072, (B, T), device="cuda")
    freq = O.rope_frequencies(part)[0].cuda()
    q = q.detach().requires_grad_()
    a, b = O.rotary(q, k, pos, freq, inter, 1.25)
    dq, = torch.autograd.grad(a, q, g)
    cut = torch.tensor([0, 1, 2, T // 3, T // 2, T - 2, T - 1], device="cuda")
    for got, x, inv, what in ((a, q, False, "q"), (b, k, False, "k"), (dq, g, True, "dq")):
        close(got[:, :, cut], ref(x[:, :, cut], pos[:, cut], freq, inter, 1.25, inv), what)
