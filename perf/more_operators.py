"""Prompts in chunks behind a paged (K, V') cache, rotary positions for long contexts and constraints on the next
token: the operators as cases that can be timed and compared.

Three operators, each through the entry point that a program calls:

* ``prefill``   -- :func:`lucid_amd.paged.lucid_prefill_paged`: a chunk of new tokens of every sequence of a batch
  (right-padded, each sequence with its own number of them) against its pages: their V' rows solved, K and V'
  appended, attention over what is cached and the chunk itself;
* ``rotary``    -- :func:`lucid_amd.model_ops.rotary`: queries and keys turned by their positions, in half or
  interleaved layout, the whole head or a part, with scaled frequencies, and the gradient;
* ``constrain`` -- :func:`lucid_amd.model_ops.constrain_logits`: penalties of tokens that have occurred, biases and
  bit masks of allowed tokens (grammars) on logit rows, and the gradient.

``own`` says whether ``run`` calls those entry points or computes the same in elementary torch operations in
float32 (angles in float64); ``exact`` evaluates the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the next turn of a short chat: the smallest call, latency alone
        {"name": "prefill_turn", "op": "prefill", "B": 1, "idle": 0, "Hq": 16, "Hkv": 16, "d": 64, "page": 64,
         "lo": 300, "hi": 300, "new": 37, "least": 37},
        # a pass of a busy server at the reference model's heads: some sequences bring a turn, some a single token
        {"name": "prefill_mixed", "op": "prefill", "B": 16, "idle": 2, "Hq": 32, "Hkv": 4, "d": 68, "page": 16,
         "lo": 50, "hi": 3500, "new": 256, "least": 1},
        # questions behind long documents that are cached
        {"name": "prefill_documents", "op": "prefill", "B": 4, "idle": 0, "Hq": 32, "Hkv": 4, "d": 64, "page": 64,
         "lo": 8192, "hi": 8192, "new": 512, "least": 300},
        # a chunk in the middle of a long prompt, grouped heads
        {"name": "prefill_chunk", "op": "prefill", "B": 1, "idle": 0, "Hq": 32, "Hkv": 8, "d": 128, "page": 64,
         "lo": 32768, "hi": 32768, "new": 2048, "least": 2048},
        # the last chunk of a 128K context
        {"name": "prefill_long", "op": "prefill", "B": 1, "idle": 0, "Hq": 32, "Hkv": 8, "d": 128, "page": 256,
         "lo": 130560, "hi": 130560, "new": 512, "least": 512},
        # one token of each of 32 sequences at the reference model's heads
        {"name": "rotary_step", "op": "rotary", "B": 32, "T": 1, "Hq": 32, "Hkv": 4, "d": 68, "part": 68, "dtype": "bf16",
         "interleaved": False, "scaling": "none", "grad": False},
        # a training pass of the reference model's heads in fp32
        {"name": "rotary_train", "op": "rotary", "B": 8, "T": 2048, "Hq": 32, "Hkv": 4, "d": 68, "part": 68, "dtype": "f32",
         "interleaved": False, "scaling": "none", "grad": True},
        # a 128K prompt: interleaved pairs in half of the head, frequencies scaled by parts
        {"name": "rotary_long", "op": "rotary", "B": 1, "T": 131072, "Hq": 32, "Hkv": 8, "d": 128, "part": 64, "dtype": "bf16",
         "interleaved": True, "scaling": "yarn", "grad": False},
        # the rows of one sampling step: all penalties, a bias, a grammar's mask
        {"name": "constrain_step", "op": "constrain", "R": 8, "V": 32000, "dtype": "bf16", "N": 700, "masked": 0.7,
         "bias": True, "penalties": True, "grad": False},
        # fp32 logits of an odd vocabulary behind very long contexts
        {"name": "constrain_history", "op": "constrain", "R": 4, "V": 32003, "dtype": "f32", "N": 100000, "masked": 0.0,
         "bias": False, "penalties": True, "grad": False},
        # many sequences of a wide vocabulary
        {"name": "constrain_wide", "op": "constrain", "R": 64, "V": 131072, "dtype": "bf16", "N": 4000, "masked": 0.95,
         "bias": False, "penalties": True, "grad": False},
        # a policy-gradient step: the constraints under which its tokens were sampled, and their gradient
        {"name": "constrain_train", "op": "constrain", "R": 8192, "V": 32000, "dtype": "bf16", "N": 500, "masked": 0.3,
         "bias": False, "penalties": True, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "prefill", "rotary", "rotary", "constrain", "constrain"])
    if op == "prefill":
        hq, hkv = rng.choice([(16, 16), (32, 8), (32, 4), (12, 4), (64, 2)])
        B = _log(rng, 1, 32)
        new = min(_log(rng, 1, 2048), max(1, 2 ** 17 // (B * hq)))
        hi = min(_log(rng, 16, 131072), max(1, 2 ** 31 // (B * hq * new)), 2 ** 20 // (B * hkv))
        return {"op": op, "B": B, "idle": rng.choice([0, 0, B // 8]), "Hq": hq, "Hkv": hkv,
                "d": rng.choice([64, 64, 68, 96, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "lo": int(hi * rng.choice([0.0, 0.05, 0.5, 1.0])), "hi": hi, "new": new,
                "least": max(1, int(new * rng.choice([0.0, 0.3, 1.0])))}
    if op == "rotary":
        hq, hkv = rng.choice([(16, 16), (32, 8), (32, 4), (12, 4), (64, 2)])
        d = rng.choice([64, 68, 96, 128, 128])
        B, dtype, grad = _log(rng, 1, 64), rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.5
        T = min(_log(rng, 1, 131072), int(2.6e9 / (B * (hq + hkv) * d * (4 if dtype == "bf16" else 8) * (2 if grad else 1))))
        return {"op": op, "B": B, "T": T, "Hq": hq, "Hkv": hkv, "d": d, "part": rng.choice([d, d, d // 2, 2 * (d // 8)]),
                "dtype": dtype, "interleaved": rng.random() < 0.4, "scaling": rng.choice(["none", "linear", "yarn"]), "grad": grad}
    V = rng.choice([_log(rng, 500, 200000), 8 * _log(rng, 64, 25000), 32000])
    R = min(_log(rng, 1, 8192), max(1, 2 ** 27 // V))
    return {"op": op, "R": R, "V": V, "dtype": rng.choice(["bf16", "bf16", "f32"]),
            "N": min(rng.choice([0, _log(rng, 10, 100000), _log(rng, 10, 2000)]), 2 ** 23 // R),
            "masked": rng.choice([0.0, 0.3, 0.95]), "bias": rng.random() < 0.4, "penalties": rng.random() < 0.8,
            "grad": rng.random() < 0.4}


# --------------------------------------------------------------------------------------------
# inputs, from the seed alone
# --------------------------------------------------------------------------------------------

def _spread(n, lo, hi):
    """n numbers from lo to hi, evenly over their logarithm, the large ones among the small."""
    if n == 1:
        return [hi]
    at = sorted(range(n), key=lambda i: (i * 7919) % 104729 % (2 * n + 1))
    out = [0] * n
    for rank, i in enumerate(at):
        out[i] = int(round(math.exp(math.log(max(lo, 1)) + (math.log(max(hi, 1)) - math.log(max(lo, 1))) * rank / (n - 1))))
        if rank == 0:
            out[i] = lo
    return out


def _lengths(case):
    """(rows cached, new tokens) of every slot of a prefill; a cached length of -1: an idle slot."""
    live = case["B"] - case["idle"]
    counts = _spread(live, case["least"], case["new"])
    return [(n, c) for n, c in zip(_spread(live, case["lo"], case["hi"]), counts[::-1])] + [(-1, 0)] * case["idle"]


def _width(d):
    return next(w for w in (64, 80, 96, 128) if w >= d)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _table(g, rows, page, spare):
    """Page tables of sequences that need `rows` rows each: ids in no order, -1 where there is none.
    Returns the table [B, M] and the number of pages of the pool."""
    need = [-(-max(n, 0) // page) for n in rows]
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(rows), max(max(need), 1) + 3), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pages


def _pool(g, pages, Hkv, page, d):
    """A pool's pages as they are after long use: every row holds something, columns from d on zeros."""
    p = torch.zeros(pages, Hkv, page, _width(d), dtype=torch.bfloat16, device=DEV)
    p[..., :d] = _randn(g, pages, Hkv, page, d, dtype=torch.bfloat16)
    return p


def _frequencies(part, scaling):
    """Inverse frequencies [part / 2] in float64 and the factor of the rotated values: base 10000, as it is; for
    positions eight times as dense ("linear"); or scaled by parts ("yarn": a frequency that turns 32 times or more in 4096
    positions stays, one that turns once or less is divided by 32, those between are interpolated)."""
    i = torch.arange(0, part, 2, dtype=torch.float64)
    f = 10000.0 ** (-i / max(part, 1))
    if scaling == "linear":
        return f / 8, 1.0
    if scaling == "yarn":
        lo, hi = (part * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(10000.0)) for n in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), part - 1)
        keep = 1 - ((torch.arange(part // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * keep + f / 32 * (1 - keep), 0.1 * math.log(32) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op == "prefill":
        B, Hq, Hkv, d, L = (case[n] for n in ("B", "Hq", "Hkv", "d", "new"))
        lens = _lengths(case)
        table, pages = _table(g, [n + c if n >= 0 else 0 for n, c in lens], case["page"], 5)
        # projections of unit variance, [B, L, H, d] seen as [B, H, L, d]; rows behind a sequence's tokens hold padding
        q, k, v = (_randn(g, B, L, h, d).to(torch.bfloat16).transpose(1, 2) for h in (Hq, Hkv, Hkv))
        state.update(table=table, k_pages=_pool(g, pages, Hkv, case["page"], d), v_pages=_pool(g, pages, Hkv, case["page"], d),
                     lens=torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV),
                     counts=torch.tensor([c for _, c in lens], dtype=torch.int32, device=DEV), q=q, k=k, v=v)
    elif op == "rotary":
        B, T, dt = case["B"], case["T"], _DTYPES[case["dtype"]]
        # each row's tokens in order, rows at any place of a long context
        start = torch.randint(0, max(131072 - T, 0) + 1, (B, 1), generator=g, device=DEV)
        f, scale = _frequencies(case["part"], case["scaling"])
        state.update(positions=start + torch.arange(T, device=DEV), inv_freq=f.to(DEV), scale=scale)
        for name, h in (("q", case["Hq"]), ("k", case["Hkv"])):
            state[name] = _randn(g, B, T, h, case["d"], dtype=dt).transpose(1, 2)
            if case["grad"]:
                state["d" + name] = _randn(g, B, T, h, case["d"], dtype=dt).transpose(1, 2)
                state[name].requires_grad_()
    else:
        R, V, N, dt = case["R"], case["V"], case["N"], _DTYPES[case["dtype"]]
        state["logits"] = (2.5 * _randn(g, R, V)).to(dt)
        state.update(history=None, prompt_lens=None, bias=None, allowed=None)
        if N:
            # tokens of a text: a few are frequent, most are rare; rows of different lengths, padded with -1
            rank = (V ** torch.rand(R, N, generator=g, device=DEV)).long().clamp_(max=V) - 1
            rank = (rank * 7919) % V
            length = torch.randint(N // 2, N + 1, (R, 1), generator=g, device=DEV)
            state["history"] = torch.where(torch.arange(N, device=DEV) < length, rank, -1)
            state["prompt_lens"] = (length[:, 0] * torch.rand(R, generator=g, device=DEV)).to(torch.int32)
        if case["bias"]:
            bias = torch.zeros(V, device=DEV)
            some = torch.randperm(V, generator=g, device=DEV)[:300]
            bias[some] = 4 * _randn(g, some.numel())
            state["bias"] = bias
        if case["masked"]:
            words = -(-V // 32)
            ok = torch.rand(R, words * 32, generator=g, device=DEV) >= case["masked"]
            ok[:, 0] = True  # something is allowed in every row
            bits = ok.view(R, words, 32).long() << torch.arange(32, device=DEV)
            state["allowed"] = bits.sum(-1).to(torch.int32)  # (the low 32 bits)
        if case["grad"]:
            state["g"] = _randn(g, R, V, dtype=dt)
            state["logits"].requires_grad_()
    return state


# --------------------------------------------------------------------------------------------
# one pass: the framework's operators, or their plain forms
# --------------------------------------------------------------------------------------------

# penalties of a case that has them: of tokens that occur in the prompt or the answer, and of those in the answer
_REPETITION, _PRESENCE, _FREQUENCY = 1.2, 0.4, 0.1


def _plain_prefill(s):
    case = s["case"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, Hq, L, d = q.shape
    Hkv, page = case["Hkv"], case["page"]
    G, scale = Hq // Hkv, d ** -0.5
    table, lens, counts = s["table"].long(), s["lens"].long(), s["counts"].long()

    def rows(pool):  # [B, Hkv, M page, d]
        return pool[table.clamp(min=0)].transpose(1, 2).reshape(B, Hkv, -1, pool.shape[-1])[..., :d].float()

    def hat(x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)

    real = (torch.arange(L, device=DEV) < counts[:, None])[:, None, :, None]  # [B, 1, L, 1]
    q, k, v = (torch.where(real, x, 0.0) for x in (q, k, v))
    kc, vc = rows(s["k_pages"]), rows(s["v_pages"])
    seen = (torch.arange(kc.shape[2], device=DEV) < lens[:, None])[:, None, None]  # [B, 1, 1, M page]
    kh = hat(k)
    p = torch.where(seen, torch.exp(scale * (kh @ hat(kc).transpose(2, 3)) - 1 / scale), 0.0)
    held = v - p @ vc  # minus the cached rows' part; row by row what the cache will hold
    del p
    among = torch.exp(scale * (kh @ kh.transpose(2, 3)) - 1 / scale)
    for t in range(L):
        part = (among[:, :, t:t + 1, :t] @ held[:, :, :t])[:, :, 0]
        held[:, :, t] = ((held[:, :, t] - part) / among[:, :, t, t, None]).to(torch.bfloat16).float()
    ask = q.reshape(B, Hkv, G * L, d)
    sc = (scale * (ask @ kc.transpose(2, 3))).masked_fill_(~seen, -math.inf)
    later = torch.arange(L, device=DEV)[None] > torch.arange(L, device=DEV)[:, None]
    sn = (scale * (ask @ k.transpose(2, 3))).view(B, Hkv, G, L, L).masked_fill_(later, -math.inf).view(B, Hkv, G * L, L)
    m = torch.maximum(sc.amax(-1, keepdim=True), sn.amax(-1, keepdim=True))
    ec, en = sc.sub_(m).exp_(), sn.sub_(m).exp_()
    o = (ec @ vc + en @ held) / (ec.sum(-1, keepdim=True) + en.sum(-1, keepdim=True))
    o = torch.where(real & (lens >= 0)[:, None, None, None], o.reshape(B, Hq, L, d), 0.0).transpose(1, 2).to(torch.bfloat16)
    # the new rows appended
    b, t = ((torch.arange(L, device=DEV) < counts[:, None]) & (lens >= 0)[:, None]).nonzero(as_tuple=True)
    at = lens[b] + t
    ids = table[b, at // page]
    s["k_pages"][ids, :, at % page, :d] = s["k"][b, :, t]
    s["v_pages"][ids, :, at % page, :d] = held[b, :, t].to(torch.bfloat16)
    return {"o": o, "k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}


def _turned(x, cos, sin, part, interleaved):
    """x [B, H, T, d] with its first `part` columns turned by the angles whose cos and sin [B, 1, T, part / 2] are given."""
    y = x.float().clone()
    if interleaved:
        a, b = x[..., 0:part:2].float(), x[..., 1:part:2].float()
        y[..., 0:part:2], y[..., 1:part:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :part // 2].float(), x[..., part // 2:part].float()
        y[..., :part // 2], y[..., part // 2:part] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    angle = s["positions"][:, None, :, None].double() * s["inv_freq"]
    cos, sin = (s["scale"] * angle.cos()).float(), (s["scale"] * angle.sin()).float()
    out = {n: _turned(s[n].detach(), cos, sin, case["part"], case["interleaved"]) for n in ("q", "k")}
    if case["grad"]:
        for n in ("q", "k"):
            out["d" + n] = _turned(s["d" + n], cos, -sin, case["part"], case["interleaved"])
    return out


def _plain_constrain(s):
    case = s["case"]
    x = s["logits"].detach().float()
    slope = torch.ones_like(x) if case["grad"] else None
    if s["history"] is not None and case["penalties"]:
        h = s["history"]
        there = (h >= 0).int()
        answer = there * (torch.arange(h.shape[1], device=DEV) >= s["prompt_lens"][:, None]).int()
        count = torch.zeros(x.shape, dtype=torch.int32, device=DEV)
        occurs = count.scatter_add(1, h.clamp(min=0), there) > 0
        count = count.scatter_add(1, h.clamp(min=0), answer)
        if case["grad"]:
            slope = torch.where(occurs, torch.where(x > 0, 1 / _REPETITION, _REPETITION), slope)
        x = torch.where(occurs, torch.where(x > 0, x / _REPETITION, x * _REPETITION), x)
        x = x - _PRESENCE * (count > 0).float() - _FREQUENCY * count.float()
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        v = torch.arange(case["V"], device=DEV)
        ok = (s["allowed"][:, v // 32] >> (v % 32)) & 1
        x = torch.where(ok > 0, x, -math.inf)
        if case["grad"]:
            slope = slope * ok.float()
    out = {"logits": x.to(s["logits"].dtype)}
    if case["grad"]:
        out["dlogits"] = (s["g"].float() * slope).to(s["logits"].dtype)
    return out


def _own(s):
    case = s["case"]
    if case["op"] == "prefill":
        from lucid_amd.paged import lucid_prefill_paged

        with torch.no_grad():
            o = lucid_prefill_paged(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["counts"])
        return {"o": o, "k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}
    if case["op"] == "rotary":
        from lucid_amd.model_ops import rotary

        q, k = rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"], scale=s["scale"])
        out = {"q": q.detach(), "k": k.detach()}
        if case["grad"]:
            out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return out
    from lucid_amd.model_ops import constrain_logits

    kw = {"repetition": _REPETITION, "presence": _PRESENCE, "frequency": _FREQUENCY} if case["penalties"] else {}
    y = constrain_logits(s["logits"], history=s["history"], prompt_lens=s["prompt_lens"], bias=s["bias"], allowed=s["allowed"],
                         **kw)
    out = {"logits": y.detach()}
    if case["grad"]:
        out["dlogits"], = torch.autograd.grad(y, s["logits"], s["g"])
    return out


def run(state):
    if own:
        return _own(state)
    plain = {"prefill": _plain_prefill, "rotary": _plain_rotary, "constrain": _plain_constrain}
    return plain[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "prefill":
        Hq, Hkv, d = (case[n] for n in ("Hq", "Hkv", "d"))
        lens = [(n, c) for n, c in _lengths(case) if n >= 0]
        # the cached rows of K and V'; q, k, v of the tokens, o of all slots' rows, and the appended rows
        moved = 4 * sum(n for n, _ in lens) * Hkv * d + sum(c for _, c in lens) * d * (2 * Hq + 8 * Hkv)
        moved += 2 * case["B"] * case["new"] * Hq * d
        return {"bytes": moved, "flops": 4 * (Hq + Hkv) * d * sum(c * n + c * (c + 1) // 2 for n, c in lens)}
    if op == "rotary":
        n = case["B"] * case["T"] * (case["Hq"] + case["Hkv"])
        passes = 2 if case["grad"] else 1
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": passes * 2 * n * case["d"] * size + 8 * case["B"] * case["T"], "flops": passes * 3 * n * case["part"]}
    R, V = case["R"], case["V"]
    size = 2 if case["dtype"] == "bf16" else 4
    words = R * -(-V // 32) if case["masked"] else 0
    moved = R * V * size * 2 + 4 * words + 8 * R * case["N"] + (4 * V if case["bias"] else 0)
    if case["grad"]:
        moved += R * V * size * 2
    return {"bytes": moved, "flops": R * V * (4 if case["grad"] else 2)}


# --------------------------------------------------------------------------------------------
# the definitions in float64
# --------------------------------------------------------------------------------------------

def _exact_prefill(s):
    case = s["case"]
    d, page, Hkv, L = case["d"], case["page"], case["Hkv"], case["new"]
    G, scale = case["Hq"] // Hkv, d ** -0.5
    o = torch.zeros(case["B"], L, case["Hq"], d, dtype=torch.float64, device=DEV)
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    for b, (n, c) in enumerate(_lengths(case)):
        if n < 0 or c == 0:
            continue
        row = torch.arange(n + c, device=DEV)
        ids = s["table"][b].long()[row // page]
        keys, vals = (x[ids, :, row % page, :d].transpose(0, 1).contiguous() for x in (kp, vp))  # [Hkv, n + c, d]
        keys[:, n:] = s["k"][b, :, :c].double()
        norm = (keys.square().sum(-1) / d + EPS).sqrt()
        new = s["v"][b, :, :c].double()
        unit = keys / norm[..., None]
        for h in range(Hkv):
            w = torch.exp(scale * (unit[h, n:] @ unit[h].T) - 1 / scale)  # [c, n + c]
            y = new[h] - w[:, :n] @ vals[h, :n]
            inner = w[:, n:].contiguous()
            x = torch.zeros_like(y)
            for t in range(c):
                x[t] = ((y[t] - inner[t, :t] @ x[:t]) / inner[t, t]).to(torch.bfloat16).double()
            vals[h, n:] = x
            a = scale * (s["q"][b, h * G:(h + 1) * G, :c].double().reshape(G * c, d) @ keys[h].T)
            a = a.view(G, c, n + c).masked_fill_(row > n + torch.arange(c, device=DEV)[:, None], -math.inf)
            a = torch.softmax(a, -1).view(G * c, n + c) @ vals[h]
            o[b, :c, h * G:(h + 1) * G] = a.view(G, c, d).transpose(0, 1)
        kp[ids[n:], :, row[n:] % page, :d] = keys[:, n:].transpose(0, 1)
        vp[ids[n:], :, row[n:] % page, :d] = vals[:, n:].transpose(0, 1)
    return {"o": o, "k_pages": kp, "vprime_pages": vp}


def _exact_rotary(s):
    case, part = s["case"], s["case"]["part"]
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device=DEV),
                       s["positions"][:, None, :, None].double() * s["inv_freq"])  # [B, 1, T, part / 2], complex

    def turned(x, by):
        y = x.detach().double()
        pairs = y[..., :part].unflatten(-1, (part // 2, 2) if case["interleaved"] else (2, part // 2))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return torch.cat((z, y[..., part:]), -1)

    out = {"q": turned(s["q"], turn), "k": turned(s["k"], turn)}
    if case["grad"]:
        out.update(dq=turned(s["dq"], turn.conj()), dk=turned(s["dk"], turn.conj()))
    return out


def _exact_constrain(s):
    case, V = s["case"], s["case"]["V"]
    parts = []
    for r0 in range(0, case["R"], 1024):
        cut = slice(r0, r0 + 1024)
        x = s["logits"].detach()[cut].double()
        R = x.shape[0]
        slope = torch.ones_like(x)
        if s["history"] is not None and case["penalties"]:
            h = s["history"][cut]
            place = torch.arange(R, device=DEV)[:, None] * V + h
            answer = torch.arange(h.shape[1], device=DEV) >= s["prompt_lens"][cut, None]
            everywhere = torch.bincount(place[h >= 0], minlength=R * V).view(R, V)
            answered = torch.bincount(place[(h >= 0) & answer], minlength=R * V).view(R, V)
            factor = torch.where(x > 0, torch.full_like(x, 1 / _REPETITION), torch.full_like(x, _REPETITION))
            slope = torch.where(everywhere > 0, factor, slope)
            x = x * slope - _PRESENCE * (answered > 0) - _FREQUENCY * answered
        if s["bias"] is not None:
            x = x + s["bias"].double()
        if s["allowed"] is not None:
            word = s["allowed"][cut].long() & 0xFFFFFFFF
            ok = ((word[..., None] // (1 << torch.arange(32, device=DEV))) % 2).flatten(1)[:, :V] == 1
            x, slope = x.masked_fill(~ok, -math.inf), slope.masked_fill(~ok, 0.0)
        out = {"logits": x}
        if case["grad"]:
            out["dlogits"] = s["g"][cut].double() * slope
        parts.append(out)
    return {n: torch.cat([q[n] for q in parts]) for n in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"prefill": _exact_prefill, "rotary": _exact_rotary, "constrain": _exact_constrain}[case["op"]](s)
