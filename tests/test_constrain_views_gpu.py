"""Gradients of ``constrain_logits`` on views: strided, three-dimensional, transposed and offset logits, element by element against
the definition's slope (the sign of the logit of the same row and token), behind histories that are held in registers and
behind longer ones that are counted; and rows large enough to pass the caches by, in fp32.  Tolerances are those of
test_constrain_logits_gpu.py."""
import pytest
import torch

from test_constrain_logits_gpu import BF, F32, bits_of, close, history_of, ref

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu


def views(base):
    """(logits, how the rows of [2, 6] go with it)"""
    return [(base[..., :1000], lambda t: t), (base[..., 3:], lambda t: t), (base[:, ::2, 1:1001], lambda t: t[:, ::2]),
            (base.transpose(0, 1)[..., 2:1002], lambda t: t.transpose(0, 1)), (base[1, :, 1:1001], lambda t: t[1]),
            (base[1, 4, :1000], lambda t: t[1, 4]), (base[:, 2:3, 3:], lambda t: t[:, 2:3]),
            (base[:, None, :, :1000].expand(2, 3, 6, 1000)[:, 1], lambda t: t)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("N", [40, 4096, 4097, 6000])
def test_gradients_of_views(N, dtype):
    g = torch.Generator(device="cuda").manual_seed(N)
    base = torch.randn(2, 6, 1003, generator=g, device="cuda").to(dtype)
    V = 1000
    ok = torch.rand(2, 6, V, generator=g, device="cuda") < 0.5
    # few distinct tokens in each row, others in every row: a sign from another row or column shows
    h = torch.randint(0, V, (2, 6, N), generator=g, device="cuda")
    h = torch.where(h % 12 == torch.arange(12, device="cuda").view(2, 6, 1), h, -1) if N < 1000 else \
        torch.where(h % 3 == torch.arange(12, device="cuda").view(2, 6, 1) % 3, h, -1)
    rho = 0.5 + torch.rand(2, 6, generator=g, device="cuda")
    for i, (x, cut) in enumerate(views(base)):
        print(f"case N={N} {dtype} view {i} {tuple(x.shape)} {x.stride()}", flush=True)
        hh, oo, rr = cut(h), cut(ok), cut(rho)
        leaf = x.detach().requires_grad_()
        y = O.constrain_logits(leaf, history=hh, repetition=rr, presence=0.3, allowed=bits_of(oo))
        grad = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        d, = torch.autograd.grad(y, leaf, grad)
        flat = [t.reshape(-1, t.shape[-1]) for t in (x, hh, oo)]
        want, tol, slope = ref(flat[0], history=flat[1], repetition=rr.reshape(-1), presence=0.3, allowed=flat[2])
        assert slope.unique().numel() >= 3  # masked, unseen and seen tokens
        close(y.detach().reshape(-1, V), want, tol, "logits")
        gd = slope * grad.double().reshape(-1, V)
        close(d.reshape(-1, V), gd, 2 * 2.0 ** -24 * gd.abs(), "dlogits")


@pytest.mark.parametrize("N", [0, 300, 5000])
def test_large_fp32_rows_and_their_gradient(N):
    """Results of 100 MB and more pass the caches by; without a history, with tokens held, with tokens counted."""
    g = torch.Generator(device="cuda").manual_seed(N)
    R, V = 900, 32003
    x = torch.randn(R, V, generator=g, device="cuda")
    h = history_of(g, R, N, V)
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.8
    grad = torch.randn(R, V, generator=g, device="cuda")
    leaf = x.clone().requires_grad_()
    y = O.constrain_logits(leaf, history=h, repetition=1.25, presence=0.5, frequency=0.125, allowed=bits_of(ok))
    d, = torch.autograd.grad(y, leaf, grad)
    for rows in (slice(0, 40), slice(R - 40, R)):
        want, tol, slope = ref(x[rows], history=h[rows], repetition=1.25, presence=0.5, frequency=0.125, allowed=ok[rows])
        close(y[rows].detach(), want, tol, "logits")
        close(d[rows], slope * grad[rows].double(), 2 * 2.0 ** -24 * (slope * grad[rows].double()).abs(), "dlogits")
