"""GPU parity of ``lucid_amd.model_ops.rotary`` with its definition in float64, and of ``rope_frequencies`` with closed forms.

Tolerance of a value y = s (a cos x - b sin x), elementwise: the angle's argument is left to 32 bits with at most 2^-25 of a
radian, cos and sin by two units of 2^-24 and the factor by one, the two products and their sum by one each: together
below 2^-21 s (|a| + |b|); the angle itself is worked out in 64 bits, on either side off by at most 2^-51 |x|; and half
a step of the type, finfo.eps / 2 |y|.  Copied columns are equal.
"""
import math

import pytest
import torch

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def ref(x, pos, freq, inter, scale, inverse=False):
    """(turned, tolerance without the rounding to the type) in float64 on the CPU."""
    x = x.detach().cpu().double()
    B, H, T, d = x.shape
    n = freq.numel()
    pos = pos.cpu().double()
    pos = pos[None] if pos.dim() == 1 else pos
    ang = (pos[:, None, :, None] * freq.cpu().double()).expand(B, 1, T, n)
    c, s = ang.cos(), ang.sin() * (-1 if inverse else 1)
    y, tol = x.clone(), torch.zeros_like(x)
    ia = torch.arange(n) * 2 if inter else torch.arange(n)
    ib = ia + 1 if inter else ia + n
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = scale * (a * c - b * s), scale * (b * c + a * s)
    e = abs(scale) * (a.abs() + b.abs()) * (2.0 ** -21 + 2.0 ** -51 * ang.abs())
    tol[..., ia] = e
    tol[..., ib] = e
    return y, tol


def close(got, want, what):
    y, tol = want
    g = got.detach().cpu().double()
    off = (g - y).abs() - tol - torch.where(tol > 0, torch.finfo(got.dtype).eps / 2 * y.abs(), 0.0)
    assert off.max().item() <= 0, f"{what}: off by {off.max().item():.3e} more than its tolerance"


def make(B, T, Hq, Hkv, d, dtype, seed=0, order="bthd"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(h):
        if order == "bthd":
            return torch.randn(B, T, h, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
        if order == "bhtd":
            return torch.randn(B, h, T, d, generator=g, device="cuda").to(dtype)
        if order == "odd":  # a view at an odd offset with odd strides
            return torch.randn(B, T, h, d + 3, generator=g, device="cuda").to(dtype)[..., 1:d + 1].transpose(1, 2)
        return torch.randn(B, d, T, h, generator=g, device="cuda").to(dtype).permute(0, 3, 2, 1)  # last axis strided
    return one(Hq), one(Hkv)


def check(q, k, pos, freq, inter=False, scale=1.0):
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    a, b = O.rotary(q, k, pos, freq, inter, scale)
    assert a.dtype == q.dtype and a.shape == q.shape and b.shape == k.shape
    da, db = torch.autograd.grad((a, b), (q, k), (gq, gk))
    torch.cuda.synchronize()
    for got, x, inv, what in ((a, q, False, "q"), (b, k, False, "k"), (da, gq, True, "dq"), (db, gk, True, "dk")):
        close(got, ref(x, pos, freq, inter, scale, inv), what)
    with torch.no_grad():  # the same values without a graph
        c, e = O.rotary(q, k, pos, freq, inter, scale)
    assert torch.equal(a, c) and torch.equal(b, e)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,part", [(64, 64), (68, 68), (128, 128), (128, 64), (96, 24), (68, 34), (68, 16), (80, 80), (65, 64),
                                    (33, 2), (1, 0), (2, 2), (256, 256), (64, 0)])
def test_dims(d, part, inter, dtype):
    print(f"case d={d} part={part} inter={inter} {dtype}", flush=True)
    q, k = make(2, 37, 5, 2, d, dtype)
    pos = torch.randint(0, 131072, (2, 37), device="cuda")
    check(q, k, pos, O.rope_frequencies(part)[0].cuda(), inter, 1.25)


@pytest.mark.parametrize("order", ["bthd", "bhtd", "odd", "strided"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("inter", [False, True])
def test_layouts(order, dtype, inter):
    for d, part in ((64, 64), (68, 68), (67, 34)):
        print(f"case {order} {dtype} inter={inter} d={d}", flush=True)
        q, k = make(3, 11, 4, 1, d, dtype, order=order)
        check(q, k, torch.arange(11, device="cuda") + 5, O.rope_frequencies(part)[0].cuda(), inter)


@pytest.mark.parametrize("B,T", [(1, 1), (32, 1), (1, 4095), (2, 2048), (1, 4097), (5, 1000)])
def test_tokens(B, T):
    print(f"case B={B} T={T}", flush=True)
    q, k = make(B, T, 3, 1, 68, BF)
    check(q, k, torch.randint(0, 200000, (B, T), device="cuda", dtype=torch.int32), O.rope_frequencies(68)[0].cuda())


def test_positions_far_negative_and_broadcast():
    q, k = make(2, 9, 2, 1, 64, F32)
    freq = O.rope_frequencies(64)[0].cuda()
    base = torch.tensor([0, 1, -1, 131071, 10 ** 6, 2 ** 31 - 1, -(2 ** 31), 12345678, 7], device="cuda")
    for pos in (base, base[None], base.int().expand(2, 9), torch.stack((base, base.flip(0)))):
        print(f"case {tuple(pos.shape)} {pos.dtype}", flush=True)
        check(q, k, pos, freq)
    check(q, k, torch.arange(18, device="cuda").view(9, 2).t(), freq)  # strided positions
    check(q, k, base, freq.float())  # frequencies in 32 bits are taken as they are


def test_only_one_of_both_and_empty():
    q, k = make(2, 9, 2, 1, 64, BF)
    freq, pos = O.rope_frequencies(64)[0].cuda(), torch.arange(9, device="cuda")
    a, none = O.rotary(q, None, pos, freq)
    assert none is None and torch.equal(a, O.rotary(q, k, pos, freq)[0])
    for leaf in (0, 1):  # a gradient of one, and through one
        x = [q.detach(), k.detach()]
        x[leaf] = x[leaf].clone().requires_grad_()
        y = O.rotary(*x, pos, freq)
        g, = torch.autograd.grad(y[leaf], x[leaf], torch.ones_like(y[leaf]))
        close(g, ref(torch.ones_like(x[leaf]), pos, freq, False, 1.0, True), "gradient")
    for shape in ((0, 2, 9, 64), (2, 2, 0, 64)):
        e = torch.empty(shape, dtype=BF, device="cuda")
        out = O.rotary(e, e, torch.zeros(shape[2], dtype=torch.int64, device="cuda"), freq)
        assert out[0].shape == shape


def test_gradient_by_differences():
    q, k = make(1, 6, 2, 1, 20, F32)
    pos, freq = torch.arange(6, device="cuda") * 1000, O.rope_frequencies(12)[0].cuda()
    q = q.detach().contiguous().requires_grad_()
    g = torch.randn(q.shape, device="cuda")
    dq, = torch.autograd.grad(O.rotary(q, k, pos, freq, True, 0.7)[0], q, g)
    h = 0.5
    for i in range(0, q.numel(), 7):
        e = torch.zeros_like(q).view(-1)
        e[i] = h
        e = e.view_as(q)
        with torch.no_grad():
            up, down = (O.rotary(q + x, k, pos, freq, True, 0.7)[0].double() for x in (e, -e))
        want = ((up - down) * g.double()).sum().item() / (2 * h)
        # two rows differ; each value by 2^-20 of its operands (4 at most here), two products with g
        assert abs(dq.reshape(-1)[i].item() - want) <= 4 * 2.0 ** -20 * 4 * g.abs().max().item() / h


def test_a_captured_call_follows_its_positions():
    q, k = make(2, 8, 4, 2, 68, BF)
    pos = torch.arange(8, device="cuda").expand(2, 8).contiguous()
    freq = O.rope_frequencies(68)[0].cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        O.rotary(q, k, pos, freq)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = O.rotary(q, k, pos, freq)
    for step in range(3):
        pos += 1000 * step
        graph.replay()
        torch.cuda.synchronize()
        c, e = O.rotary(q, k, pos, freq)
        assert torch.equal(a, c) and torch.equal(b, e)


def test_refusals():
    q, k = make(2, 9, 2, 1, 64, BF)
    pos, freq = torch.arange(9, device="cuda"), O.rope_frequencies(64)[0].cuda()
    with pytest.raises(RuntimeError, match="GPU"):
        O.rotary(q.cpu(), k, pos, freq)
    for bad in (q.half(), q.float()):
        with pytest.raises(TypeError, match="one dtype"):
            O.rotary(bad, k, pos, freq)
    for p in (pos[:8], pos.float(), pos.cpu(), pos.expand(3, 9)):
        with pytest.raises(ValueError, match="positions"):
            O.rotary(q, k, p, freq)
    for f in (torch.ones(33, device="cuda"), freq.half(), freq.cpu(), freq[::2], freq[None]):
        with pytest.raises(ValueError, match="inv_freq"):
            O.rotary(q, k, pos, f)
    with pytest.raises(ValueError, match="q .B, Hq"):
        O.rotary(q, k[:, :, :8], pos, freq)
    with pytest.raises(NotImplementedError, match="frequencies"):
        O.rotary(q, k, pos, freq.clone().requires_grad_())
    with pytest.raises(ValueError, match="finite"):
        O.rotary(q, k, pos, freq, scale=math.inf)
    with pytest.raises(ValueError, match="256"):
        O.rotary(*make(1, 9, 1, 1, 257, BF), pos, freq)


def test_tangents_and_second_derivatives_are_refused():
    from torch.autograd import forward_ad
    q, k = make(1, 4, 2, 1, 64, F32)
    pos, freq = torch.arange(4, device="cuda"), O.rope_frequencies(64)[0].cuda()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            O.rotary(forward_ad.make_dual(q, torch.ones_like(q)), k, pos, freq)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            O.rotary(q, forward_ad.make_dual(k, torch.ones_like(k)), pos, freq)
    x = q.clone().requires_grad_()
    g, = torch.autograd.grad(O.rotary(x, k, pos, freq)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_a_large_pass_and_its_gradient():
    """Results of 100 MB and more pass the caches by; a gradient that comes in as one value for all."""
    q, k = make(1, 14000, 24, 8, 128, BF)
    pos = torch.arange(14000, device="cuda")
    freq = O.rope_frequencies(128)[0].cuda()
    a, b = O.rotary(q, k, pos, freq)
    for t in (0, 1, 4095, 13999):
        close(a[:, :, t:t + 1], ref(q[:, :, t:t + 1], pos[t:t + 1], freq, False, 1.0), f"q at {t}")
        close(b[:, :, t:t + 1], ref(k[:, :, t:t + 1], pos[t:t + 1], freq, False, 1.0), f"k at {t}")
    x = q.clone().requires_grad_()
    O.rotary(x, k, pos, freq)[0].sum().backward()
    close(x.grad[:, :, -1:], ref(torch.ones_like(q[:, :, -1:]), pos[-1:], freq, False, 1.0, True), "dq")


def test_captured_backward():
    """A captured turn and its gradient on static leaves follow new values, while no eager graph of theirs lives."""
    q, k = make(2, 16, 4, 2, 68, BF)
    q, k = (x.detach().contiguous().requires_grad_() for x in (q, k))
    pos = torch.arange(16, device="cuda") * 100
    freq = O.rope_frequencies(68)[0].cuda()
    g = torch.randn(2, 4, 16, 68, device="cuda").to(BF)

    def step():
        a, b = O.rotary(q, k, pos, freq)
        return torch.autograd.grad((a, b), (q, k), (g, g[:, :2]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, dk = step()
    for _ in range(3):
        g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        close(dq, ref(g, pos, freq, False, 1.0, True), "dq")
        close(dk, ref(g[:, :2], pos, freq, False, 1.0, True), "dk")
