"""A decoder that reads prompts in chunks behind cached rows, at rotary positions scaled for a long context, and constrains its
next tokens, in one run, against the same sequences read at once.

bf16 models on the same weights; the logits of a tiny decoder of unit scale differ by bf16 rounding at several
places (projections, norms, attention: about ten roundings of 2^-9 relatively, in root mean square), so the bar is 3e-2 of
the largest logit.  A cache that mixes up a row, a page or a position is off by the logits' own size.
"""
import pytest
import torch

from lucid_amd import modeling_lucid as M
from lucid_amd.model_ops import constrain_logits, rope_frequencies, rotary, token_logprobs
from lucid_amd.paged import LucidPagedCache

pytestmark = pytest.mark.gpu

BAR = 3e-2
YARN = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 256}


def _model(heads=8, kv=2, d=64, layers=2, **kw):
    torch.manual_seed(11)
    cfg = M.LucidConfig(vocab_size=320, hidden_size=512, intermediate_size=768, num_hidden_layers=layers,
                        num_attention_heads=heads, num_key_value_heads=kv, head_dim=d, initializer_range=0.06, **kw)
    return M.LlamaForCausalLM(cfg).to("cuda", torch.bfloat16).eval()


def _close(got, want):
    assert (got.float() - want.float()).abs().max().item() <= BAR * want.float().abs().max().item()


@pytest.mark.parametrize("kw", [dict(), dict(d=68, kv=1, rope_scaling=YARN), dict(rope_scaling=YARN, partial_rotary_factor=0.5,
                                                                                  rope_interleaved=True),
                                dict(d=128, heads=4, rope_scaling={"rope_type": "linear", "factor": 4.0})], ids=str)
@torch.no_grad()
def test_chunks_of_prompts_beside_decoding(kw):
    """Three prompts of different lengths in chunks (a chunk beside single tokens, an idle slot, a fork in between), then the
    next token of each under constraints."""
    print(f"case {kw}", flush=True)
    model = _model(**kw)
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(0, 320, (n,), generator=g).tolist() for n in (300, 70, 33)]
    cache = LucidPagedCache(80, 16)
    seqs = cache.new(3)
    done = [0, 0, 0]

    def whole(tokens):
        return model(torch.tensor([tokens], device="cuda"), past_key_values=M.LucidCache())[1][0]

    def chunk(lengths, order=(0, 1, None, 2)):
        rows = [None if i is None else seqs[i] for i in order]
        T = max(lengths)
        ids = torch.randint(0, 320, (len(order), T), generator=g)  # padding holds any token
        for r, i in enumerate(order):
            if i is not None:
                ids[r, :lengths[r]] = torch.tensor(texts[i][done[i]:done[i] + lengths[r]], dtype=torch.int64)
        cache.select(rows, lengths, chunk=True)
        logits = model(ids.cuda(), past_key_values=cache)[1]
        for r, i in enumerate(order):
            if i is not None and lengths[r]:
                want = whole(texts[i][:done[i] + lengths[r]])
                _close(logits[r, :lengths[r]], want[done[i]:])
                done[i] += lengths[r]
                assert cache.length(seqs[i]) == done[i]
        return logits

    chunk([100, 5, 0, 33])      # all empty: the fused prefill
    chunk([150, 64, 0, 0])      # behind cached rows
    child = cache.fork(seqs[0])
    chunk([50, 1, 7, 0], order=(0, 1, None, 2))
    # the fork holds what its parent held then
    cache.select([child], chunk=True)
    _close(model(torch.tensor([texts[0][250:270]], device="cuda"), past_key_values=cache)[1][0], whole(texts[0][:270])[250:])
    # decoding goes on behind the chunks, its tokens under constraints
    history = torch.full((3, 310), -1, device="cuda")
    prompt = torch.tensor([len(t) for t in texts], dtype=torch.int32, device="cuda")
    cache.select(seqs)
    logits = torch.stack([whole(t)[-1] for t in texts])
    words = torch.full((10,), -2, dtype=torch.int32, device="cuda")  # token 0 is not allowed, nor 32, 64, ...
    for step in range(3):
        for i, t in enumerate(texts):
            history[i, :len(t)] = torch.tensor(t)
        bound = constrain_logits(logits, history=history, prompt_lens=prompt, repetition=1.2, presence=0.5, frequency=0.1, allowed=words)
        r = token_logprobs(bound, torch.full((3,), -100, device="cuda"), top=4)
        assert bool((r.top_indices % 32 != 0).all())
        new = r.top_indices[:, 0]
        for i, t in enumerate(texts):
            t.append(int(new[i]))
        logits = model(new[:, None], past_key_values=cache)[1][:, -1]
        for i, t in enumerate(texts):
            _close(logits[i], whole(t)[-1])


def test_scaled_positions_train():
    """Gradients through the rotary operator of a model with scaled, partial, interleaved positions equal those of the same
    model with the rotation in float32 torch, to the rounding of the backward products of bf16."""
    ids = torch.randint(0, 320, (2, 200), generator=torch.Generator().manual_seed(5)).cuda()
    model = _model(rope_scaling=YARN, partial_rotary_factor=0.5, rope_interleaved=True)

    def grads():
        model.zero_grad(set_to_none=True)
        model(ids, labels=ids)[0].backward()
        torch.cuda.synchronize()
        return {n: p.grad.float().clone() for n, p in model.named_parameters()}

    def plain(q, k, p):
        ang = p.positions[:, None, :, None].double() * p.inv_freq
        c, s = (p.scale * ang.cos()).float(), (p.scale * ang.sin()).float()

        def one(x):
            a, b = x[..., 0:32:2].float(), x[..., 1:32:2].float()
            return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2).to(x.dtype), x[..., 32:]), -1)
        return one(q), one(k)

    got = grads()
    ours, M._turn = M._turn, plain
    try:
        want = grads()
    finally:
        M._turn = ours
    for n in got:
        assert ((got[n] - want[n]).norm() / want[n].norm().clamp_min(1e-20)).item() <= 2e-2, n


@torch.no_grad()
def test_default_positions_are_what_they_were():
    """Without the new options the model's rotation is the reference's; the operator at the same frequencies is its unrounded
    form: tables in bf16 and two roundings, 3 2^-8 of the operands."""
    emb = _model().model.rotary_emb
    x = torch.randn(2, 4, 50, 64, device="cuda").to(torch.bfloat16)
    pos = torch.arange(50, device="cuda").expand(2, -1)
    emb.inv_freq = M.LlamaRotaryEmbedding(M.LucidConfig(head_dim=64)).inv_freq.cuda()  # (bf16 with the module otherwise)
    cos, sin = emb(x, pos)
    assert torch.is_tensor(cos) and cos.dtype == x.dtype
    old, _ = M.apply_rotary_pos_emb(x, x, cos, sin)
    new, _ = rotary(x, None, pos, rope_frequencies(64)[0].cuda())
    size = x.float().abs() + torch.cat((x[..., 32:], x[..., :32]), -1).float().abs()
    # (an angle of the tables is off by up to 50 2^-23: nothing beside these)
    assert ((old.float() - new.float()).abs() <= 4 * 2.0 ** -8 * size).all()
