"""GPU parity of ``lucid_amd.model_ops.constrain_logits`` with its definition in float64.

Tolerance, elementwise: the quotient or product with the penalty and the penalty itself are off by 2^-24 relatively, each
of the three sums by 2^-24 of its magnitude: together at most 6 2^-24 (|x| max(rho, 1 / rho) + |presence| + n |frequency| + |bias|),
and half a step of the type, finfo.eps / 2 |y|.  Infinities and NaN are equal.
"""
import pytest
import torch

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def bits_of(ok):
    """A bool [..., V] as the packed int32 words."""
    V = ok.shape[-1]
    ok = torch.nn.functional.pad(ok, (0, -V % 32)).unflatten(-1, (-1, 32))
    return (ok.long() << torch.arange(32, device=ok.device)).sum(-1).to(torch.int32)


def ref(x, history=None, prompt_lens=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
    """(y, tolerance without the rounding to the type, slope) in float64; x [R, V], allowed as bool."""
    R, V = x.shape

    def per_row(p):
        p = p.double() if torch.is_tensor(p) else torch.full((R,), p, dtype=torch.float64, device=x.device)
        return p[:, None]

    rho, pi, phi = per_row(repetition), per_row(presence), per_row(frequency)
    x = x.double()
    seen = torch.zeros(R, V, dtype=torch.bool, device=x.device)
    count = torch.zeros(R, V, dtype=torch.float64, device=x.device)
    if history is not None:
        for r in range(R):
            h = history[r]
            fine = (h >= 0) & (h < V)
            seen[r, h[fine]] = True
            after = torch.arange(h.numel(), device=x.device) >= (0 if prompt_lens is None else prompt_lens[r])
            count[r] = torch.bincount(h[fine & after], minlength=V).double()
    slope = torch.where(seen, torch.where(x > 0, 1 / rho, rho), 1.0)
    y = x * slope - pi * (count > 0) - phi * count
    mag = x.abs() * torch.maximum(rho, 1 / rho) + pi.abs() + count * phi.abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if allowed is not None:
        y, slope = y.masked_fill(~allowed, -torch.inf), slope.masked_fill(~allowed, 0.0)
    return y, 6 * 2.0 ** -24 * mag, slope


def close(got, want, tol, what):
    g, eps = got.double(), torch.finfo(got.dtype).eps / 2
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.nan_to_num(g[odd], nan=7.0), torch.nan_to_num(want[odd], nan=7.0)), f"{what}: infinities or NaN"
    off = ((g - want).abs() - tol - eps * want.abs())[~odd]
    assert off.numel() == 0 or off.max().item() <= 0, f"{what}: off by {off.max().item():.3e} more than its tolerance"


def history_of(g, R, N, V, pad=True):
    h = (V ** torch.rand(R, N, generator=g, device="cuda")).long().clamp_(max=V) - 1
    if pad and N:
        n = torch.randint(0, N + 1, (R, 1), generator=g, device="cuda")
        h = torch.where(torch.arange(N, device="cuda") < n, h, -1)
    return h


def check(x, ok=None, **kw):
    grad = torch.randn(x.shape, device="cuda").to(x.dtype)
    x = x.detach().requires_grad_()
    args = dict(kw, allowed=None if ok is None else bits_of(ok))
    y = O.constrain_logits(x, **args)
    d, = torch.autograd.grad(y, x, grad)
    want, tol, slope = ref(x.detach(), allowed=ok, **kw)
    close(y.detach(), want, tol, "logits")
    close(d, slope * grad.double(), 2 * 2.0 ** -24 * (slope * grad.double()).abs(), "dlogits")
    with torch.no_grad():
        assert torch.equal(O.constrain_logits(x, **args).view(torch.int8), y.detach().view(torch.int8))


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("R,V", [(1, 1), (3, 7), (2, 31), (5, 33), (4, 8185), (3, 8192), (3, 8193), (2, 32003), (1, 131072), (65, 500)])
def test_sizes(R, V, dtype):
    print(f"case R={R} V={V} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (3 * torch.randn(R, V, generator=g, device="cuda")).to(dtype)
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.6
    bias = torch.randn(V, generator=g, device="cuda")
    prompt = torch.randint(0, 40, (R,), generator=g, device="cuda", dtype=torch.int32)
    h = history_of(g, R, 60, V)
    check(x)
    check(x, ok)
    check(x, history=h, repetition=1.3)
    check(x, history=h, prompt_lens=prompt, presence=0.5, frequency=0.25)
    check(x, ok, history=h, prompt_lens=prompt, repetition=0.8, presence=-0.5, frequency=0.1, bias=bias)
    check(x, bias=torch.randn(R, V, generator=g, device="cuda"))


@pytest.mark.parametrize("N", [0, 1, 511, 513, 5000, 70000])
def test_histories(N):
    print(f"case N={N}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn(3, 20000, generator=g, device="cuda")
    h = history_of(g, 3, N, 20000, pad=False)
    check(x, history=h, repetition=1.1, presence=0.3, frequency=0.01)
    if N:
        h[0] = 17  # one token alone
        h[1, ::2] = -100
        h[2, 0] = 20000  # outside the vocabulary
        h[2, -1] = 2 ** 40
        check(x, history=h, prompt_lens=torch.tensor([N // 2, N, 10 ** 6], dtype=torch.int32, device="cuda"), repetition=1.1,
              presence=0.3, frequency=0.01)
        check(x, history=h[:, :, None].expand(3, N, 2)[..., 0], presence=0.3)  # strided rows


def test_penalties_of_each_row():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(5, 1000, generator=g, device="cuda")
    h = history_of(g, 5, 300, 1000)
    p = {n: 0.5 + torch.rand(5, generator=g, device="cuda") for n in ("repetition", "presence", "frequency")}
    check(x, history=h, **p)
    check(x, history=h, repetition=p["repetition"])


def test_shapes_strides_and_shared_rows():
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(2, 6, 1003, generator=g, device="cuda").to(BF)
    ok = torch.rand(1000, generator=g, device="cuda") < 0.5
    h = history_of(g, 12, 40, 1000).view(2, 6, 40)
    for x in (base[..., :1000], base[..., 3:], base[:, ::2, 1:1001], base.transpose(0, 1)[..., 2:1002], base[0, 0, :1000]):
        V, lead = x.shape[-1], x.shape[:-1]
        hh = h.transpose(0, 1) if lead == (6, 2) else h[:, ::2] if lead == (2, 3) else h if len(lead) else h[0, 0]
        print(f"case {tuple(x.shape)} {x.stride()}", flush=True)
        y = O.constrain_logits(x, history=hh, repetition=1.2, allowed=bits_of(ok[:V]))
        assert y.shape == x.shape and y.is_contiguous()
        want, tol, _ = ref(x.reshape(-1, V), history=hh.reshape(-1, 40), repetition=1.2, allowed=ok[:V].expand(lead.numel(), V))
        close(y.reshape(-1, V), want, tol, "logits")
        leaf = x.detach().requires_grad_()
        d, = torch.autograd.grad(O.constrain_logits(leaf, history=hh, repetition=1.2, allowed=bits_of(ok[:V])).float().sum(), leaf)
        assert bool((d.reshape(-1, V)[:, ~ok[:V]] == 0).all()) and bool((d.reshape(-1, V)[:, ok[:V]] != 0).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_values_at_the_border(dtype):
    """Masked places may hold anything; a row may have nothing left; infinities and the type's ends go through."""
    V = 200
    ends = torch.finfo(dtype)
    x = torch.zeros(4, V, dtype=dtype, device="cuda")
    x[0, :6] = torch.tensor([float("nan"), float("inf"), float("-inf"), ends.max, ends.min, -0.0], dtype=dtype)
    x[1] = float("nan")
    x[2] = float("-inf")
    ok = torch.ones(4, V, dtype=torch.bool, device="cuda")
    ok[1] = False                # nothing left, and NaN under the mask
    ok[3, 1:] = False            # one token left
    h = torch.arange(6, device="cuda").expand(4, 6)
    y = O.constrain_logits(x, history=h, repetition=1.5, presence=1.0, allowed=bits_of(ok))
    want, tol, _ = ref(x, history=h, repetition=1.5, presence=1.0, allowed=ok)
    want[0, 4] = -float("inf")   # the lowest value, made lower, is out of the type's range
    close(y, want, tol, "logits")
    leaf = x.clone().requires_grad_()
    d, = torch.autograd.grad(O.constrain_logits(leaf, history=h, repetition=1.5, allowed=bits_of(ok)), leaf, torch.ones_like(x))
    assert bool((d[1] == 0).all()) and bool((d[3, 1:] == 0).all()) and d[3, 0] != 0 and bool(torch.isfinite(d).all())
    empty = O.constrain_logits(x[:0], history=h[:0], repetition=1.5)
    assert empty.shape == (0, V)


def test_gradient_by_differences():
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(2, 50, generator=g, device="cuda")
    x = torch.where(x.abs() < 0.3, 0.5, x).requires_grad_()  # away from the kink at 0
    h = history_of(g, 2, 30, 50)
    ok = torch.rand(2, 50, generator=g, device="cuda") < 0.7
    kw = dict(history=h, repetition=1.7, presence=0.4, frequency=0.2, allowed=bits_of(ok))
    w = torch.randn(2, 50, generator=g, device="cuda")
    d, = torch.autograd.grad(O.constrain_logits(x, **kw), x, w)
    step = 0.125
    with torch.no_grad():
        up, down = (torch.where(ok, O.constrain_logits(x + e, **kw), 0.0).double() for e in (step, -step))
    want = (up - down) / (2 * step) * w.double()  # every output hangs on its own input alone
    # each side is off by 8 2^-24 of values below 16
    assert ((d.double() - want).abs() <= 2 * 8 * 2.0 ** -24 * 16 / (2 * step) * w.abs().double() + 1e-6).all()


def test_with_log_probabilities_and_captured():
    """Log probabilities of the constrained rows; a captured call follows its history and mask."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(4, 3000, generator=g, device="cuda").to(BF)
    h = history_of(g, 4, 50, 3000)
    ok = torch.rand(4, 3000, generator=g, device="cuda") < 0.5
    ok[:, 5] = True
    tok = torch.full((4,), 5, device="cuda")
    words = bits_of(ok)
    r = O.token_logprobs(O.constrain_logits(x, history=h, repetition=1.3, allowed=words), tok, top=4)
    want = torch.log_softmax(O.constrain_logits(x, history=h, repetition=1.3, allowed=words).double(), -1)
    assert (r.logprobs.double() - want[:, 5]).abs().max().item() <= 1e-5 and bool(ok.gather(1, r.top_indices).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.no_grad():
        O.constrain_logits(x, history=h, repetition=1.3, allowed=words)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        y = O.constrain_logits(x, history=h, repetition=1.3, allowed=words)
    for _ in range(3):
        h.random_(0, 3000, generator=g)
        words.copy_(bits_of(torch.rand(4, 3000, generator=g, device="cuda") < 0.5))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, O.constrain_logits(x, history=h, repetition=1.3, allowed=words))


def test_refusals():
    x = torch.randn(2, 100, device="cuda")
    h = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="GPU"):
        O.constrain_logits(x.cpu())
    with pytest.raises(TypeError, match="logits"):
        O.constrain_logits(x.half())
    for kw, err, text in (
            (dict(history=h.int()), TypeError, "history"), (dict(history=h[:1]), ValueError, "history"),
            (dict(history=h.cpu()), TypeError, "history"), (dict(prompt_lens=h[:, 0].int()), ValueError, "without"),
            (dict(history=h, prompt_lens=h[:, 0]), ValueError, "prompt_lens"), (dict(bias=x[:, :99]), ValueError, "bias"),
            (dict(bias=x.double()), TypeError, "bias"), (dict(bias=x.clone().requires_grad_()), NotImplementedError, "gradient"),
            (dict(allowed=torch.zeros(3, dtype=torch.int32, device="cuda")), ValueError, "allowed"),
            (dict(allowed=torch.zeros(2, 100, dtype=torch.bool, device="cuda")), TypeError, "allowed"),
            (dict(repetition=0.0), ValueError, "positive"), (dict(repetition=float("nan")), ValueError, "positive"),
            (dict(presence=float("inf")), ValueError, "finite"), (dict(frequency=torch.ones(3, device="cuda")), ValueError, "frequency"),
            (dict(presence=torch.ones(2, device="cuda", requires_grad=True)), NotImplementedError, "gradient")):
        with pytest.raises(err, match=text):
            O.constrain_logits(x, **kw)


def test_tangents_and_second_derivatives_are_refused():
    from torch.autograd import forward_ad
    x = torch.randn(2, 100, device="cuda")
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        O.constrain_logits(forward_ad.make_dual(x, torch.ones_like(x)), bias=torch.zeros(100, device="cuda"))
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(O.constrain_logits(leaf).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("N", [300, 5000])
def test_large_rows_and_their_gradient(N):
    """Results of 100 MB and more pass the caches by; both ways of finding what has occurred."""
    g = torch.Generator(device="cuda").manual_seed(8)
    R, V = 1700, 32000
    x = torch.randn(R, V, generator=g, device="cuda").to(BF)
    h = history_of(g, R, N, V)
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.8
    grad = torch.randn(R, V, generator=g, device="cuda").to(BF)
    leaf = x.clone().requires_grad_()
    y = O.constrain_logits(leaf, history=h, repetition=1.25, presence=0.5, frequency=0.125, allowed=bits_of(ok))
    d, = torch.autograd.grad(y, leaf, grad)
    for rows in (slice(0, 40), slice(R - 40, R)):
        want, tol, slope = ref(x[rows], history=h[rows], repetition=1.25, presence=0.5, frequency=0.125, allowed=ok[rows])
        close(y[rows].detach(), want, tol, "logits")
        close(d[rows], slope * grad[rows].double(), 2 * 2.0 ** -24 * (slope * grad[rows].double()).abs(), "dlogits")


def test_gradient_of_log_probabilities_through_the_constraints():
    """d logprob / d logits = slope ([v = token] - p), against float64 autograd of the definition."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(6, 500, generator=g, device="cuda")
    h = history_of(g, 6, 40, 500)
    ok = torch.rand(6, 500, generator=g, device="cuda") < 0.5
    tok = torch.randint(0, 500, (6,), generator=g, device="cuda")
    ok[torch.arange(6), tok] = True
    leaf = x.clone().requires_grad_()
    lp = O.token_logprobs(O.constrain_logits(leaf, history=h, repetition=1.3, presence=0.2, allowed=bits_of(ok)), tok).logprobs
    d, = torch.autograd.grad(lp.sum(), leaf)
    y, _, slope = ref(x, history=h, repetition=1.3, presence=0.2, allowed=ok)
    p = torch.softmax(y, -1)
    want = slope * (torch.nn.functional.one_hot(tok, 500) - p)
    # p in 32 bits from exponents of at most 16 in size: 2^-19 of it, and the product's rounding
    assert ((d.double() - want).abs() <= 2.0 ** -18 * slope * p + 2.0 ** -22 * want.abs()).all()


def test_two_streams_and_expanded_rows():
    g = torch.Generator(device="cuda").manual_seed(10)
    x = torch.randn(1, 9000, generator=g, device="cuda").expand(4, 9000)
    h = history_of(g, 1, 50, 9000, pad=False).expand(4, 50)
    want, tol, _ = ref(x, history=h, repetition=1.4)
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs.append(O.constrain_logits(x, history=h, repetition=1.4))
    torch.cuda.synchronize()
    for y in outs:
        close(y, want, tol, "logits")


def test_histories_beyond_32_bits_are_refused():
    logits = torch.zeros(1, 10, device="cuda")
    with pytest.raises(ValueError, match="fewer than"):
        O.constrain_logits(logits, history=torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(1, 1 << 30))
