"""What ``constrain_logits`` keeps for its backward: the logits only where the gradient depends on them, which is through their
sign where a repetition penalty applies."""
import pytest
import torch

from test_constrain_logits_gpu import BF, F32, bits_of, close, history_of, ref

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu


def make(dtype, R=5, V=9001):
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(R, V, generator=g, device="cuda").to(dtype)
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.6
    return g, x, ok, history_of(g, R, 60, V)


def cases(ok, h, per_row):
    """(arguments, those of the reference beside them, whether the gradient depends on the logits)"""
    return [(dict(allowed=bits_of(ok)), dict(allowed=ok), False),
            (dict(bias=torch.ones(ok.shape[1], device="cuda")), dict(bias=torch.ones(ok.shape[1], device="cuda")), False),
            (dict(history=h, presence=0.5, frequency=per_row), dict(history=h, presence=0.5, frequency=per_row), False),
            (dict(history=h[:, :0], repetition=1.5), dict(), False),
            (dict(history=h, repetition=1.5, allowed=bits_of(ok)), dict(history=h, repetition=1.5, allowed=ok), True),
            (dict(history=h, repetition=per_row), dict(history=h, repetition=per_row), True)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_logits_are_kept_only_where_the_gradient_asks_for_them(dtype):
    g, x, ok, h = make(dtype)
    per_row = 0.5 + torch.rand(x.shape[0], generator=g, device="cuda")
    for i, (args, want, keeps) in enumerate(cases(ok, h, per_row)):
        print(f"case {i} {dtype}", flush=True)
        leaf = x.clone().requires_grad_()
        y = O.constrain_logits(leaf, **args)
        kept = [t for t in y.grad_fn.saved_tensors if t is not None and t.data_ptr() == leaf.data_ptr()]
        assert len(kept) == keeps
        grad = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        d, = torch.autograd.grad(y, leaf, grad)
        value, tol, slope = ref(x, **want)
        close(y.detach(), value, tol, "logits")
        close(d, slope * grad.double(), 2 * 2.0 ** -24 * (slope * grad.double()).abs(), "dlogits")


def test_logits_may_change_behind_a_call_that_does_not_keep_them():
    g, x, ok, h = make(F32)
    per_row = 0.5 + torch.rand(x.shape[0], generator=g, device="cuda")
    for i, (args, want, keeps) in enumerate(cases(ok, h, per_row)):
        print(f"case {i}", flush=True)
        leaf = x.clone().requires_grad_()
        logits = leaf * 1.0
        y = O.constrain_logits(logits, **args)
        with torch.no_grad():
            logits.neg_()
        if keeps:  # (the gradient would be that of other logits)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
        else:
            y.sum().backward()
            slope = ref(x, **want)[2]
            assert torch.equal(leaf.grad.double(), slope)


def test_shapes_of_a_gradient_without_logits():
    """Logits of any shape and strides, incoming gradients likewise."""
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(2, 6, 1003, generator=g, device="cuda").to(BF)
    ok = torch.rand(1000, generator=g, device="cuda") < 0.5
    for x in (base[..., 3:], base[:, ::2, 1:1001], base.transpose(0, 1)[..., 2:1002], base[0, 0, :1000], base[:0, :, :1000]):
        print(f"case {tuple(x.shape)} {x.stride()}", flush=True)
        leaf = x.detach().requires_grad_()
        grad = torch.randn(*x.shape[:-1], 1001, generator=g, device="cuda").to(BF)[..., 1:]
        d, = torch.autograd.grad(O.constrain_logits(leaf, allowed=bits_of(ok)), leaf, grad)
        assert d.shape == x.shape and torch.equal(d, torch.where(ok, grad, 0.0).to(BF))


def test_penalties_and_histories_may_change_where_the_gradient_does_not_ask_for_them():
    """Without a history no penalty is kept, and without a repetition penalty no history."""
    g, x, ok, h = make(F32)
    rho = 0.5 + torch.rand(x.shape[0], generator=g, device="cuda")
    phi = rho.clone()
    leaf = x.clone().requires_grad_()
    y = O.constrain_logits(leaf, repetition=rho, allowed=bits_of(ok))
    z = O.constrain_logits(leaf, history=h, frequency=phi)
    rho.fill_(2.0)
    phi.fill_(2.0)
    h.fill_(0)
    (y[ok].sum() + z.sum()).backward()
    assert torch.equal(leaf.grad, 1.0 + ok.float())
