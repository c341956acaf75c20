"""A captured pass through ``constrain_logits`` and its gradient follows new logits, histories, masks and penalties."""
import pytest
import torch

from test_constrain_logits_gpu import BF, F32, bits_of, close, history_of, ref

from lucid_amd import model_ops as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("N", [0, 200, 5000])
def test_captured_backward(N, dtype):
    """On static leaves, while no eager graph of theirs lives; without a history, with tokens held, with tokens counted."""
    print(f"case N={N} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(N)
    R, V = 6, 9001
    x = torch.randn(R, V, generator=g, device="cuda").to(dtype).requires_grad_()
    h = history_of(g, R, N, V, pad=False)
    ok = torch.rand(R, V, generator=g, device="cuda") < 0.6
    words = bits_of(ok)
    rho = 0.5 + torch.rand(R, generator=g, device="cuda")
    grad = torch.randn(R, V, generator=g, device="cuda").to(dtype)

    def step():
        y = O.constrain_logits(x, history=h, repetition=rho, presence=0.25, allowed=words)
        return y.detach(), torch.autograd.grad(y, x, grad)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, d = step()
    for _ in range(3):
        with torch.no_grad():
            x.normal_(generator=g)
        if N:
            h.random_(0, V, generator=g)
        ok = torch.rand(R, V, generator=g, device="cuda") < 0.6
        words.copy_(bits_of(ok))
        rho.uniform_(0.5, 1.5, generator=g)
        grad.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        want, tol, slope = ref(x.detach(), history=h if N else None, repetition=rho, presence=0.25, allowed=ok)
        close(y, want, tol, "logits")
        gd = slope * grad.double()
        close(d, gd, 2 * 2.0 ** -24 * gd.abs(), "dlogits")
        torch.cuda.synchronize()
