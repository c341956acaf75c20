"""A decoder with scaled rotary frequencies: generating in inference mode before training, and a first pass that is captured."""
import pytest
import torch

from lucid_amd import modeling_lucid as M

pytestmark = pytest.mark.gpu


def _model(**kw):
    torch.manual_seed(2)
    cfg = M.LucidConfig(vocab_size=200, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=4,
                        num_key_value_heads=2, head_dim=64, initializer_range=0.06, partial_rotary_factor=0.5,
                        rope_scaling={"rope_type": "linear", "factor": 4.0})
    return M.LlamaForCausalLM(cfg).to("cuda", torch.bfloat16)


def test_inference_mode_before_training():
    """A forward in inference mode, then a training step: its gradients are those of a model that only trains, up to the
    rounding to bf16 of sums in another order, 2^-8 on either side."""
    ids = torch.randint(0, 200, (2, 70), generator=torch.Generator().manual_seed(1)).cuda()

    def grads(model):
        model(ids, labels=ids)[0].backward()
        torch.cuda.synchronize()
        return [p.grad.clone() for p in model.parameters()]

    want = grads(_model())
    model = _model()
    with torch.inference_mode():
        first = model(ids)[1].clone()
    got = grads(model)
    for a, b in zip(got, want):
        assert (a.float() - b.float()).norm().item() <= 2.0 ** -7 * b.float().norm().item()
    with torch.no_grad():
        again = model(ids)[1]
    assert (again.float() - first.float()).abs().max().item() <= 3e-2 * first.float().abs().max().item()


@torch.no_grad()
def test_the_first_pass_may_be_captured():
    model = _model()
    emb, attn = model.model.rotary_emb, M._turn
    q = torch.randn(2, 4, 9, 64, device="cuda").to(torch.bfloat16)
    pos = torch.arange(9, device="cuda").expand(2, 9).contiguous()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = attn(q, q[:, :2], emb(q, pos))
    for step in range(3):
        pos += 100 * step
        graph.replay()
        torch.cuda.synchronize()
        c, d = attn(q, q[:, :2], emb(q, pos))
        assert torch.equal(a, c) and torch.equal(b, d)
        torch.cuda.synchronize()
