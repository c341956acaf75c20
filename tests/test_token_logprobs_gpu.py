"""GPU parity of ``lucid_amd.model_ops.token_logprobs`` against its definition in float64:

    x = logits / temperature, lse = log sum exp x, logprob = x_tok - lse, entropy = lse - sum p x,
    alternatives by (logit descending, index ascending) with x_i - lse,
    dx_j = [j = tok] g_lp + sum_i [j = top_i] g_i - p_j (g_lp + sum_i g_i + g_H (log p_j + H)).

Tolerances.  A term exp2(a), a = (x - m) log2 e, carries a relative error of at most 2^-22 (exp2) plus
|a| 2^-22 (its argument's two roundings); terms with |a| > 24 together weigh less than V 2^-24, so the sums are
relatively exact to 2^-17, their logarithm to 2^-17 absolutely; x_tok - m adds |x_tok - m| 2^-23.  The
entropy t / s adds the same relative error of t.  p_j: |log p_j| 2^-22 + 2^-17 relatively.  A bf16 result adds
half a step, 2^-8 relatively.
"""
import pytest
import torch

from lucid_amd.model_ops import token_logprobs

pytestmark = pytest.mark.gpu

D17, D22 = 2.0 ** -17, 2.0 ** -22


def _ref(logits, tokens, top, temperature):
    x = logits.double() / temperature
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    safe = torch.where(p > 0, logp, 0.0)
    ent = -(p * safe).sum(-1)
    given = (tokens >= 0) & (tokens < logits.shape[-1])
    lp = logp.gather(-1, tokens.clamp(0, logits.shape[-1] - 1)[..., None])[..., 0]
    lp = torch.where(tokens == -100, 0.0, torch.where(given, lp, float("nan")))
    idx = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[..., :top]
    return {"lp": lp, "ent": ent, "idx": idx, "top": logp.gather(-1, idx), "p": p, "logp": safe, "x": x}


def _check_forward(r, ref):
    def close(name, got, want):
        tol = D17 + want.abs() * (D17 if name == "entropy" else D22 * 2)
        ok = torch.where(torch.isfinite(want), (got.double() - want).abs() <= tol,
                         (got.double() == want) | (torch.isnan(got) & torch.isnan(want)))
        bad = (~ok).nonzero()
        assert bool(ok.all()), (name, bad[:3].tolist(), got[tuple(bad[0])].item(), want[tuple(bad[0])].item())

    close("logprobs", r.logprobs, ref["lp"])
    close("entropy", r.entropy, ref["ent"])
    close("top_logprobs", r.top_logprobs, ref["top"])
    assert torch.equal(r.top_indices, ref["idx"])


def _check_grad(got, ref, tokens, top, temperature, grads):
    glp, gh, gtop = (g.double() for g in grads)
    glp = torch.where(tokens >= 0, glp, 0.0)
    p, logp, H = ref["p"], ref["logp"], ref["ent"][..., None]
    every = glp + gtop.sum(-1)
    d = -p * (every[..., None] + gh[..., None] * (logp + H))
    size = p * (every.abs()[..., None] + gh.abs()[..., None] * (logp.abs() + H))
    # half of log p's own error enters through the entropy's factor too
    tol = size * (D17 * 2 + logp.abs() * D22) + p * gh.abs()[..., None] * (D17 * 2 + logp.abs() * D22)
    at = tokens.clamp(min=0)[..., None]
    d.scatter_add_(-1, at, glp[..., None])
    tol.scatter_add_(-1, at, glp.abs()[..., None] * D22)
    if top:
        d.scatter_add_(-1, ref["idx"], gtop)
        tol.scatter_add_(-1, ref["idx"], gtop.abs() * D22 * 2)
    d, tol = d / temperature, tol / temperature + 1e-35
    if got.dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + d.abs() * 2.0 ** -8
    else:
        tol = tol + d.abs() * D22
    bad = ((got.double() - d).abs() > tol).nonzero()
    assert bad.numel() == 0, (bad[:3].tolist(), got[tuple(bad[0])].item(), d[tuple(bad[0])].item(), tol[tuple(bad[0])].item())


def _run(logits, tokens, top, temperature, seed=0):
    logits = logits.detach().requires_grad_()
    r = token_logprobs(logits, tokens, top=top, temperature=temperature)
    ref = _ref(logits.detach(), tokens, top, temperature)
    torch.cuda.synchronize()
    assert r.logprobs.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32
    _check_forward(r, ref)
    g = torch.Generator(device="cuda").manual_seed(seed)
    grads = [torch.randn(t.shape, generator=g, device="cuda") for t in (r.logprobs, r.entropy, r.top_logprobs)]
    outs, gs = (r.logprobs, r.entropy), grads[:2]
    if top:
        outs, gs = outs + (r.top_logprobs,), grads
    dx, = torch.autograd.grad(outs, logits, gs)
    torch.cuda.synchronize()
    assert dx.dtype == logits.dtype and dx.shape == logits.shape
    _check_grad(dx, ref, tokens, top, temperature, grads)
    return r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,R,top,temperature", [
    (1, 3, 1, 1.0), (2, 1, 2, 0.5), (7, 5, 7, 1.0), (8, 4, 3, 2.0), (64, 2, 64, 1.0), (500, 33, 5, 1.0),
    (8184, 3, 20, 0.7), (8185, 3, 20, 1.0), (8192, 2, 1, 1.0), (8193, 5, 64, 1.0), (32000, 4, 20, 1.0),
    (32003, 5, 8, 0.7), (32761, 3, 50, 1.0), (32768, 3, 64, 1.0), (32769, 3, 33, 1.0), (70001, 3, 64, 1.3),
    (131072, 2, 5, 1.0), (300007, 2, 0, 1.0)])
def test_forward_and_gradient(V, R, top, temperature, dtype):
    print(f"case V={V} R={R} top={top} T={temperature} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V + R)
    logits = (2.5 * torch.randn(R, V, generator=g, device="cuda")).to(dtype)
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    tokens[R // 2] = -100
    _run(logits, tokens, top, temperature)


@pytest.mark.parametrize("dtype,R", [(torch.bfloat16, 1600), (torch.float32, 801)])
def test_gradients_of_100_megabytes(dtype, R):
    """Gradients from the size on that passes the caches by, the named values among them (written a second time)."""
    print(f"case large gradient R={R} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(R)
    logits = (2.5 * torch.randn(R, 32003, generator=g, device="cuda")).to(dtype)
    _run(logits, torch.randint(0, 32003, (R,), generator=g, device="cuda"), 8, 1.0)


@pytest.mark.parametrize("V", [40, 9000, 32003, 40000])
@pytest.mark.parametrize("kind", ["inf", "lowest", "few", "const", "steps", "ramp", "fall", "zeros"])
def test_masked_tied_and_ordered_rows(kind, V):
    """Masks of -inf and of the lowest value (a few allowed tokens among them, fewer than the alternatives), rows of
    one value, of a few values and in order: ties go to the lower index."""
    print(f"case {kind} V={V}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V)
    R, top = 4, 20
    logits = 2 * torch.randn(R, V, generator=g, device="cuda")
    if kind == "inf":
        logits[torch.rand(R, V, generator=g, device="cuda") < 0.5] = float("-inf")
    elif kind == "lowest":
        logits[torch.rand(R, V, generator=g, device="cuda") < 0.5] = torch.finfo(torch.bfloat16).min
    elif kind == "few":
        keep = torch.randint(0, V, (R, 6), generator=g, device="cuda")
        logits = torch.full_like(logits, float("-inf")).scatter(1, keep, logits.gather(1, keep))
    elif kind == "const":
        logits = torch.arange(R, device="cuda")[:, None].float().expand(R, V).contiguous() - 1
    elif kind == "steps":
        logits = torch.randint(-2, 3, (R, V), generator=g, device="cuda").float()
    elif kind == "zeros":
        logits = torch.where(torch.rand(R, V, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    else:
        logits = torch.linspace(-8, 8, V, device="cuda").expand(R, V).contiguous()
        if kind == "fall":
            logits = logits.flip(1).contiguous()
    tokens = logits.argmax(-1)
    for dtype in (torch.bfloat16, torch.float32):
        r = _run(logits.to(dtype), tokens, top, 1.0)
        if kind == "const":
            assert torch.equal(r.top_indices, torch.arange(top, device="cuda").expand(R, top))


def test_rows_without_a_distribution():
    """Rows of -inf alone, with a NaN, with +inf: NaN as log_softmax gives; the rows beside them are not affected.
    NaN logits come first among the alternatives."""
    for V in (50, 9001, 40000):
        logits = torch.randn(5, V, device="cuda")
        logits[0] = float("-inf")
        logits[1, V // 2] = float("nan")
        logits[2, V - 1] = float("inf")
        logits[4, 3:] = float("-inf")
        tokens = torch.tensor([1, 2, V - 1, 4, 1], device="cuda")
        for dtype in (torch.bfloat16, torch.float32):
            x = logits.to(dtype).requires_grad_()
            r = token_logprobs(x, tokens, top=4)
            for t in (r.logprobs, r.entropy, r.top_logprobs):
                assert bool(torch.isnan(t[:3]).all())
            ref = _ref(x.detach()[3:], tokens[3:], 4, 1.0)
            _check_forward(type(r)(*(t[3:] for t in r)), ref)
            assert torch.equal(r.top_indices, torch.sort(x.detach().float(), dim=-1, descending=True, stable=True).indices[:, :4])
            dx, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
            assert bool(torch.isnan(dx[:3]).any(-1).all()) and bool(torch.isfinite(dx[3:]).all())
            assert bool((dx[4, 3:] == 0).all())


def test_tokens_outside_the_vocabulary_and_ignored_ones():
    V = 1000
    x = torch.randn(4, V, device="cuda").requires_grad_()
    tokens = torch.tensor([V, -1, -100, 5], device="cuda")
    r = token_logprobs(x, tokens)
    assert bool(torch.isnan(r.logprobs[:2]).all()) and r.logprobs[2].item() == 0.0
    assert bool(torch.isfinite(r.entropy).all())
    dx, = torch.autograd.grad(r.logprobs, x, torch.ones(4, device="cuda"))
    assert bool(torch.isnan(dx[:2]).all()) and bool((dx[2] == 0).all()) and bool(torch.isfinite(dx[3]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1001, 32000, 32771])
def test_layouts(V, dtype):
    """[B, T - 1, V] slices, rows apart, a misaligned base, a column stride, one row, leading axes: the results of the
    contiguous copy."""
    g = torch.Generator(device="cuda").manual_seed(V)
    B, T, top = 2, 4, 5
    full = (2 * torch.randn(B, T, V + 3, generator=g, device="cuda")).to(dtype)
    flat = full.reshape(-1)
    views = {"slice": full[:, :-1, :V], "offset": flat[1:1 + 3 * V].view(3, V), "apart": full[:, 1, 2:2 + V],
             "columns": full.transpose(1, 2)[:, :T, :], "row": full[1, 2, 1:1 + V], "axes": full[..., :V].reshape(B, 2, 2, V),
             "expand": full[:1, :1, :V].expand(2, 3, V)}
    for name, x in views.items():
        print(f"case layout {name} V={V} {dtype}", flush=True)
        Vx = x.shape[-1]
        k = min(top, Vx)
        tokens = torch.randint(0, Vx, x.shape[:-1], generator=g, device="cuda")
        a = x.detach().requires_grad_()
        b = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        ra, rb = token_logprobs(a, tokens, top=k), token_logprobs(b, tokens, top=k)
        outs = [torch.randn(ra[i].shape, generator=g, device="cuda") for i in range(3)]
        da, = torch.autograd.grad(ra[:3], a, outs)
        db, = torch.autograd.grad(rb[:3], b, outs)
        # another alignment deals the values to other lanes, so the sums may round differently
        for s, t in zip(ra[:3], rb[:3]):
            assert (s - t).abs().max().item() <= 2 * D17 * (1 + t.abs().max().item())
        assert torch.equal(ra.top_indices, rb.top_indices)
        # the softmax part -p (a + g_H (log p + H)) cancels in some places, so its error is measured against the
        # magnitude of its terms, as in every other case
        for dx in (da, db):
            _check_grad(dx, _ref(x.detach(), tokens, k, 1.0), tokens, k, 1.0, outs)


def test_gradients_of_some_outputs_and_shared_ones():
    """Gradients of one output alone; a token that is also an alternative; the same logits used twice."""
    V, R, top = 3001, 6, 9
    g = torch.Generator(device="cuda").manual_seed(3)
    x0 = torch.randn(R, V, generator=g, device="cuda")
    tokens = x0.argmax(-1)  # the first alternative is the given token
    zeros = [torch.zeros(R, device="cuda"), torch.zeros(R, device="cuda"), torch.zeros(R, top, device="cuda")]
    for i in range(3):
        x = x0.clone().requires_grad_()
        r = token_logprobs(x, tokens, top=top)
        go = torch.randn(r[i].shape, generator=g, device="cuda")
        dx, = torch.autograd.grad(r[i], x, go)
        grads = list(zeros)
        grads[i] = go
        _check_grad(dx, _ref(x0, tokens, top, 1.0), tokens, top, 1.0, grads)
    x = x0.clone().requires_grad_()
    twice = token_logprobs(x, tokens).logprobs.sum() + token_logprobs(x, tokens).logprobs.sum()
    d2, = torch.autograd.grad(twice, x)
    y = x0.clone().requires_grad_()
    d1, = torch.autograd.grad(token_logprobs(y, tokens).logprobs.sum(), y)
    assert torch.equal(d2, 2 * d1)
    assert token_logprobs(x0, tokens).logprobs.grad_fn is None


def test_gradient_against_differences():
    """Central differences of the forward at fp32 logits.  With a step of 2^-6 the truncation is h^2 / 6 times a third
    derivative (at most 8 for these weights), the forward's error 2^-16 / h."""
    V, h = 37, 2.0 ** -6
    g = torch.Generator(device="cuda").manual_seed(5)
    x0 = torch.randn(1, V, generator=g, device="cuda")
    tokens = torch.tensor([4], device="cuda")
    w = torch.randn(3, generator=g, device="cuda")

    def f(x):
        r = token_logprobs(x, tokens.expand(x.shape[0]), temperature=0.8)
        return w[0] * r.logprobs + w[1] * r.entropy

    x = x0.clone().requires_grad_()
    dx, = torch.autograd.grad(f(x).sum(), x)
    e = h * torch.eye(V, device="cuda")
    num = (f(x0 + e) - f(x0 - e)) / (2 * h)
    assert (num - dx[0]).abs().max().item() <= w[:2].abs().sum().item() * (h * h / 6 * 8 / 0.8 ** 3 + 4 * 2.0 ** -16 / h)


def test_empty_batches_and_side_streams():
    r = token_logprobs(torch.empty(0, 7, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert r.logprobs.shape == (0,) and r.top_indices.shape == (0, 3)
    x = torch.empty(2, 0, 7, device="cuda", requires_grad=True)
    y = token_logprobs(x, torch.empty(2, 0, dtype=torch.int64, device="cuda")).logprobs.sum()
    assert torch.autograd.grad(y, x)[0].shape == (2, 0, 7)
    logits = torch.randn(64, 32000, device="cuda")
    tokens = torch.randint(0, 32000, (64,), device="cuda")
    want = token_logprobs(logits, tokens, top=5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = token_logprobs(logits, tokens, top=5)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("V", [32000, 40000])
def test_captured_forward_and_backward(V):
    """A captured forward and backward replayed on new logits gives the eager results each time."""
    R, top = 9, 6
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(R, V, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    go = [torch.randn(R, generator=g, device="cuda"), torch.randn(R, generator=g, device="cuda"),
          torch.randn(R, top, generator=g, device="cuda")]

    def step(t):
        r = token_logprobs(t, tokens, top=top, temperature=0.9)
        dx, = torch.autograd.grad(r[:3], t, go)
        return [*(y.detach() for y in r), dx]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(R, V, generator=g, device="cuda"))
            tokens.copy_(torch.randint(0, V, (R,), generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(x.detach().clone().requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
