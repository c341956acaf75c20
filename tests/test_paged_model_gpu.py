"""A decoder served from pages: a ragged prefill, decoding steps, forks, idle slots, freeing and compaction in one run,
against the same sequences one by one in the contiguous ``LucidCache``, and ``token_logprobs`` against the prefill.

Both runs are bf16 models on the same weights; the logits of a tiny decoder of unit scale differ by bf16 rounding at
several places (projections, norms, attention: about ten roundings of 2^-9 relatively, in root mean square), so the bar
is 3e-2 of the largest logit.  A cache that mixes up a row, a page or a position is off by the logits' own size.
"""
import pytest
import torch

from lucid_amd import modeling_lucid as M
from lucid_amd.paged import LucidPagedCache, OutOfPages

pytestmark = pytest.mark.gpu

BAR = 3e-2


def _model(heads=8, kv=2, d=64, layers=3):
    torch.manual_seed(11)
    cfg = M.LucidConfig(vocab_size=320, hidden_size=512, intermediate_size=768, num_hidden_layers=layers,
                        num_attention_heads=heads, num_key_value_heads=kv, head_dim=d, initializer_range=0.06)
    return M.LlamaForCausalLM(cfg).to("cuda", torch.bfloat16).eval()


class _Alone:
    """The same sequence by itself in a contiguous cache."""

    def __init__(self, model, tokens):
        self.model, self.tokens = model, list(tokens)

    def logits(self):
        """The logits after the last token, by one prefill of the whole sequence."""
        ids = torch.tensor([self.tokens], device="cuda")
        return self.model(ids, past_key_values=M.LucidCache())[1][0, -1].float()


def _close(got, want):
    assert (got.float() - want).abs().max().item() <= BAR * want.abs().max().item()


@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 64, 16), (8, 1, 68, 7), (4, 4, 128, 64)])
@torch.no_grad()
def test_serving_run(heads, kv, d, page):
    print(f"case serving heads={heads} kv={kv} d={d} page={page}", flush=True)
    model = _model(heads, kv, d)
    g = torch.Generator().manual_seed(d)
    prompts = [torch.randint(0, 320, (n,), generator=g).tolist() for n in (37, 5, 64, 1)]
    cache = LucidPagedCache(max(24, 400 // page), page)
    seqs = cache.new(4)
    alone = {s: _Alone(model, p) for s, p in zip(seqs, prompts)}
    T = max(map(len, prompts))
    # a right-padded prefill, one slot idle
    ids = torch.zeros(5, T, dtype=torch.int64)
    rows = [seqs[0], None, seqs[1], seqs[2], seqs[3]]
    lengths = [len(alone[s].tokens) if s is not None else 0 for s in rows]
    for i, s in enumerate(rows):
        if s is not None:
            ids[i, :lengths[i]] = torch.tensor(alone[s].tokens)
    cache.select(rows, lengths)
    logits = model(ids.cuda(), past_key_values=cache)[1]
    for i, s in enumerate(rows):
        if s is not None:
            _close(logits[i, lengths[i] - 1], alone[s].logits())
            assert cache.length(s) == lengths[i]

    def step(order, L=1):
        new = torch.randint(0, 320, (len(order), L), generator=g)
        out = model(new.cuda(), past_key_values=cache)[1]
        for i, s in enumerate(order):
            if s is not None:
                alone[s].tokens += new[i].tolist()
                _close(out[i, -1], alone[s].logits())

    cache.select([seqs[0], seqs[1], None, seqs[2], seqs[3]])
    for _ in range(3):
        step([seqs[0], seqs[1], None, seqs[2], seqs[3]])
    # two samples of the first sequence, one of the third
    kids = [cache.fork(seqs[0]), cache.fork(seqs[0]), cache.fork(seqs[2])]
    for k, s in zip(kids, (seqs[0], seqs[0], seqs[2])):
        alone[k] = _Alone(model, alone[s].tokens)
    order = [kids[2], seqs[0], kids[0], kids[1], seqs[3]]
    cache.select(order)
    step(order)
    step(order, L=3)
    # the parents end; what is left moves to the front
    cache.free(seqs[0], seqs[1], seqs[2])
    cache.compact()
    assert cache.free_pages == cache.num_pages - len({p for s in order[2:4] + order[:1] + order[4:] for p in cache.pages(s)})
    order = [kids[1], kids[2], seqs[3], None, kids[0]]
    cache.select(order)
    for _ in range(2):
        step(order)
    # a new sequence beside the old ones: its first tokens go through the decoding path
    (late,) = cache.new()
    alone[late] = _Alone(model, [])
    order = [late, kids[0]]
    cache.select(order)
    step(order, L=4)
    # the cache holds what the contiguous one holds
    ref = M.LucidCache()
    model(torch.tensor([alone[kids[1]].tokens], device="cuda"), past_key_values=ref)
    for layer in range(3):
        k, v = cache.gather(kids[1], layer)
        for a, b in ((k[..., :d], ref.key_cache[layer][0]), (v[..., :d], ref.value_cache[layer][0])):
            assert (a.float() - b.float()).abs().max().item() <= 5e-2 * b.float().abs().max().item()
        assert bool((k[..., d:] == 0).all()) and bool((v[..., d:] == 0).all())
    with pytest.raises(OutOfPages):
        model(torch.zeros(2, page * cache.num_pages, dtype=torch.int64, device="cuda"), past_key_values=cache)


@torch.no_grad()
def test_logprobs_of_a_decoding_step_match_those_of_the_sequence():
    """Tokens picked from the alternatives of each step, scored as they are picked and again all at once by
    ``LlamaForCausalLM.token_logprobs``."""
    model = _model()
    cache = LucidPagedCache(20, 16)
    (seq,) = cache.new()
    cache.select([seq])
    prompt = torch.randint(0, 320, (1, 21), generator=torch.Generator().manual_seed(2)).cuda()
    tokens, picked, entropies = prompt, [], []
    logits = model(prompt, past_key_values=cache)[1][:, -1]
    for i in range(6):
        top = M.token_logprobs(logits, torch.full((1,), -100, device="cuda"), top=3).top_indices[:, i % 3]
        r = M.token_logprobs(logits, top, top=3)
        assert torch.equal(r.logprobs, r.top_logprobs[:, i % 3])
        picked.append(r.logprobs.item())
        entropies.append(r.entropy.item())
        tokens = torch.cat([tokens, top[:, None]], 1)
        logits = model(top[:, None], past_key_values=cache)[1][:, -1]
    r = model.token_logprobs(tokens, top=2)
    assert r.logprobs.shape == tokens.shape and r.logprobs[0, -1].item() == 0.0
    scale = model(tokens)[1].float().abs().max().item()
    for i in range(6):
        assert abs(r.logprobs[0, 20 + i].item() - picked[i]) <= 2 * BAR * scale
        assert abs(r.entropy[0, 20 + i].item() - entropies[i]) <= 2 * BAR * scale


def test_scores_train_the_model():
    """Gradients of a weighted sum of log probabilities and entropies reach the parameters, equal to those of the same
    sum in float32 torch on the model's own logits: the logits' gradients agree to half a step of bf16 (and the error
    of p, 2^-16), the parameters' to the rounding of the backward products of bf16."""
    model = _model(layers=1)
    ids = torch.randint(0, 320, (2, 40), generator=torch.Generator().manual_seed(5)).cuda()
    w = torch.randn(2, 40, generator=torch.Generator().manual_seed(6)).cuda()

    def run(score):
        model.zero_grad(set_to_none=True)
        score().backward()
        torch.cuda.synchronize()
        return {n: p.grad.float().clone() for n, p in model.named_parameters()}

    def ours():
        r = model.token_logprobs(ids)
        return (w * (r.logprobs + 0.1 * r.entropy)).sum()

    def plain():
        lp = torch.log_softmax(model(ids)[1].float(), -1)
        given = torch.nn.functional.pad(lp[:, :-1].gather(-1, ids[:, 1:, None])[..., 0], (0, 1))
        return (w * (given - 0.1 * (lp.exp() * lp).sum(-1))).sum()

    a, b = run(ours), run(plain)
    for n in a:
        assert ((a[n] - b[n]).norm() / b[n].norm().clamp_min(1e-20)).item() <= 2e-2, n


def test_training_step_captured_beside_eager_scores():
    """The captured score and its gradient on static logits follow new values at each replay while an eager graph of
    other leaves lives."""
    from lucid_amd.model_ops import token_logprobs
    x = torch.randn(6, 1000, device="cuda", requires_grad=True)
    y = torch.randn(6, 1000, device="cuda", requires_grad=True)
    tok = torch.arange(6, device="cuda")
    alive = token_logprobs(y, tok).logprobs.sum()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(token_logprobs(x, tok).logprobs.sum(), x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(token_logprobs(x, tok).logprobs.sum(), x)
    for i in range(3):
        with torch.no_grad():
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        z = x.detach().clone().requires_grad_()
        want, = torch.autograd.grad(token_logprobs(z, tok).logprobs.sum(), z)
        assert torch.equal(dx, want), i
    assert torch.isfinite(torch.autograd.grad(alive, y)[0]).all()
