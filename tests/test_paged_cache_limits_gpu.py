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


def test_tables_of_one_page():
    """A table of one column is contiguous whatever its strides say, and its rows may be any distance apart."""
    from lucid_amd.paged import lucid_decode_paged, write_pages
    g = torch.Generator(device="cuda").manual_seed(2)
    kp, vp = (torch.randn(6, 2, 16, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q, k, v = (torch.randn(3, h, 1, 64, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2))
    lens = torch.tensor([3, 0, 15], dtype=torch.int32, device="cuda")
    ids = torch.tensor([[4, 0, 2]], dtype=torch.int32, device="cuda")
    wide = torch.full((3, 7), 5, dtype=torch.int32, device="cuda")
    wide[:, 3] = ids[0]
    outs = []
    for table in (ids[0][:, None].clone(), ids.t(), wide[:, 3:4], torch.as_strided(ids, (3, 1), (1, 3))):
        assert table.shape == (3, 1)
        a, b = kp.clone(), vp.clone()
        outs.append([*lucid_decode_paged(q, k, v, a, b, table, lens), a, b])
        a, b = kp.clone(), vp.clone()
        write_pages(k, v, a, b, table, lens)
        outs[-1] += [a, b]
    assert ids.t().stride() == (1, 3)
    for other in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(outs[0], other))
