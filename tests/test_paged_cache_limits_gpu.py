"""Calls at the edges of ``LucidPagedCache`` on the GPU."""
import pytest
import torch

from lucid_amd import modeling_lucid as M
from lucid_amd.paged import LucidPagedCache

pytestmark = pytest.mark.gpu


def _model():
    torch.manual_seed(5)
    cfg = M.LucidConfig(vocab_size=128, hidden_size=512, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                        num_key_value_heads=2, head_dim=64, initializer_range=0.06)
    return M.LlamaForCausalLM(cfg).to("cuda", torch.bfloat16).eval()


@torch.no_grad()
def test_a_captured_pass_is_refused_and_the_next_one_runs():
    """Capturing a decoding pass, a fork or a compaction raises; the same passes run eagerly afterwards give what they
    give in a cache of which nothing was captured."""
    model = _model()
    ids = torch.randint(0, 128, (1, 20), generator=torch.Generator().manual_seed(1)).cuda()
    token = torch.tensor([[7]], device="cuda")
    outs = []
    for capture in (True, False):
        cache = LucidPagedCache(10, 16)
        (a,) = cache.new()
        cache.select([a])
        model(ids, past_key_values=cache)
        model(token, past_key_values=cache)
        if capture:
            for call in (lambda: model(token, past_key_values=cache), lambda: cache.fork(a), cache.compact):
                graph = torch.cuda.CUDAGraph()
                with pytest.raises(RuntimeError, match="captured"):
                    with torch.cuda.graph(graph):
                        call()
            assert cache.length(a) == 21 and cache.free_pages == 8
        out = [model(token, past_key_values=cache)[1]]
        cache.select([cache.fork(a)])
        out.append(model(token, past_key_values=cache)[1])
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(*outs))
