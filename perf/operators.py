"""Serving a LUCID decoder from a paged (K, V') cache: the operators as cases that can be timed and compared.

Four operators, each through the entry point that a program calls:

* ``decode`` -- :func:`lucid_amd.paged.lucid_decode_paged`: L new tokens of every sequence of a batch against
  its pages (row j of sequence b is row j % page of page ``table[b, j // page]``); each sequence has its own
  length, a negative length marks a batch slot that holds none;
* ``write``  -- :func:`lucid_amd.paged.write_pages`: a right-padded prefill's K and V' rows into their pages;
* ``copy``   -- :func:`lucid_amd.paged.copy_pages`: pages copied in every layer's pools at once, as forking a
  sequence (its partial last page) and compacting a pool do;
* ``logprobs`` -- :func:`lucid_amd.model_ops.token_logprobs`: log probabilities of given tokens, entropy and
  the top alternatives of logit rows, and the gradient of all three.

``own`` says whether ``run`` calls those entry points or computes the same in elementary torch operations in
float32; ``exact`` evaluates the definitions in float64.
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token of a session just begun: the smallest call, latency alone
        {"name": "decode_short", "op": "decode", "B": 1, "idle": 0, "Hq": 16, "Hkv": 16, "d": 64, "page": 64,
         "lo": 300, "hi": 300, "new": 1},
        # a step of a busy server at the reference model's heads: ragged chats, small pages, some idle slots
        {"name": "decode_batch", "op": "decode", "B": 32, "idle": 3, "Hq": 32, "Hkv": 4, "d": 68, "page": 16,
         "lo": 50, "hi": 3500, "new": 1},
        # one token at the end of a 128K context, grouped heads: the cache is read once
        {"name": "decode_long", "op": "decode", "B": 1, "idle": 0, "Hq": 32, "Hkv": 8, "d": 128, "page": 256,
         "lo": 131072, "hi": 131072, "new": 1},
        # drafted tokens checked five at a time, sequences of very different lengths
        {"name": "decode_draft", "op": "decode", "B": 8, "idle": 0, "Hq": 32, "Hkv": 8, "d": 128, "page": 64,
         "lo": 200, "hi": 16000, "new": 5},
        # a padded batch of prompts of the reference model's heads into small pages, V' as the prefill gives it
        {"name": "write_batch", "op": "write", "B": 4, "Hkv": 4, "d": 68, "page": 16, "T": 2048, "lo": 300,
         "vp": "f32"},
        # one long prompt, appended to a cached prefix
        {"name": "write_long", "op": "write", "B": 1, "Hkv": 8, "d": 128, "page": 64, "T": 30011, "lo": 30011,
         "vp": "f32"},
        # eight samples of one prompt: the partial last page of each, in every layer
        {"name": "copy_fork", "op": "copy", "layers": 16, "pages": 600, "Hkv": 4, "d": 68, "page": 16, "n": 8},
        # a pool compacted after many sequences have ended
        {"name": "copy_compact", "op": "copy", "layers": 16, "pages": 1000, "Hkv": 4, "d": 68, "page": 64, "n": 400},
        # the rows of one sampling step, a part of the vocabulary masked out, with the alternatives shown
        {"name": "logprobs_step", "op": "logprobs", "R": 8, "V": 32000, "dtype": "bf16", "top": 20, "grad": False,
         "masked": 0.3, "temperature": 0.7},
        # few rows of a wide vocabulary
        {"name": "logprobs_wide", "op": "logprobs", "R": 64, "V": 131072, "dtype": "bf16", "top": 50, "grad": False,
         "masked": 0.0, "temperature": 1.0},
        # fp32 logits of an odd vocabulary, a distillation step on the alternatives
        {"name": "logprobs_odd", "op": "logprobs", "R": 1021, "V": 32003, "dtype": "f32", "top": 8, "grad": True,
         "masked": 0.0, "temperature": 1.0},
        # a policy gradient step's log probabilities and entropy bonus, as long as a training sequence
        {"name": "logprobs_train", "op": "logprobs", "R": 8192, "V": 32000, "dtype": "bf16", "top": 0, "grad": True,
         "masked": 0.0, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "write", "copy", "logprobs", "logprobs"])
    if op == "decode":
        hq, hkv = rng.choice([(16, 16), (32, 8), (32, 4), (12, 4), (64, 2)])
        B = _log(rng, 1, 64)
        hi = min(_log(rng, 30, 131072), max(1, 2 ** 20 // (B * hkv)))
        return {"op": op, "B": B, "idle": rng.choice([0, 0, B // 8]), "Hq": hq, "Hkv": hkv,
                "d": rng.choice([64, 64, 68, 96, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "lo": max(0, int(hi * rng.choice([0.02, 0.5, 1.0]))), "hi": hi, "new": rng.choice([1, 1, 1, 2, 5, 8])}
    if op == "write":
        hkv, B = rng.choice([2, 4, 8, 16]), rng.choice([1, 2, 4, 8])
        T = min(_log(rng, 5, 32768), 2 ** 18 // (B * hkv))
        return {"op": op, "B": B, "Hkv": hkv, "d": rng.choice([64, 68, 96, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "T": T, "lo": max(1, int(T * rng.choice([0.1, 0.5, 1.0]))), "vp": rng.choice(["f32", "f32", "bf16"])}
    if op == "copy":
        pages = _log(rng, 32, 1000)
        return {"op": op, "layers": rng.choice([1, 2, 8, 16]), "pages": pages, "Hkv": rng.choice([2, 4]),
                "d": rng.choice([64, 68, 96]), "page": rng.choice([16, 32, 64]), "n": max(1, _log(rng, 1, 0.4 * pages))}
    V = rng.choice([_log(rng, 500, 200000), 8 * _log(rng, 64, 25000), 32000])
    top = rng.choice([0, 0, 1, 8, 20, 50])
    R = min(_log(rng, 1, 8192), max(1, (2 ** 27 if top == 0 else 2 ** 25) // V))
    return {"op": op, "R": R, "V": V, "dtype": rng.choice(["bf16", "bf16", "f32"]), "top": top,
            "grad": rng.random() < 0.5, "masked": rng.choice([0.0, 0.0, 0.3, 0.9]), "temperature": rng.choice([1.0, 1.0, 0.7])}


# --------------------------------------------------------------------------------------------
# inputs, from the seed alone
# --------------------------------------------------------------------------------------------

def _spread(n, lo, hi):
    """n lengths from lo to hi, evenly over their logarithm, the long ones among the short."""
    if n == 1:
        return [hi]
    at = sorted(range(n), key=lambda i: (i * 7919) % 104729 % (2 * n + 1))
    out = [0] * n
    for rank, i in enumerate(at):
        out[i] = int(round(math.exp(math.log(max(lo, 1)) + (math.log(max(hi, 1)) - math.log(max(lo, 1))) * rank / (n - 1))))
    return out


def _lengths(case):
    """The rows that each sequence of a decode has cached (-1: an idle slot), or that a prompt brings."""
    if case["op"] == "write":
        return _spread(case["B"], case["lo"], case["T"])
    live = case["B"] - case["idle"]
    return _spread(live, case["lo"], case["hi"]) + [-1] * case["idle"]


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


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op == "decode":
        B, Hq, Hkv, d, L = (case[n] for n in ("B", "Hq", "Hkv", "d", "new"))
        lens = _lengths(case)
        table, pages = _table(g, [n + L if n >= 0 else 0 for n in lens], case["page"], 5)
        state.update(table=table, k_pages=_pool(g, pages, Hkv, case["page"], d), v_pages=_pool(g, pages, Hkv, case["page"], d),
                     lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        # projections of unit variance, [B, L, H, d] seen as [B, H, L, d]
        q, k, v = (_randn(g, B, L, h, d).to(torch.bfloat16).transpose(1, 2) for h in (Hq, Hkv, Hkv))
        state.update(q=q, k=k, v=v)
    elif op == "write":
        B, Hkv, d, T = (case[n] for n in ("B", "Hkv", "d", "T"))
        counts = _lengths(case)
        before = [17 * b % 50 for b in range(B)]  # rows that are cached already (a shared system prompt, say)
        table, pages = _table(g, [n + m for n, m in zip(before, counts)], case["page"], 5)
        k = _randn(g, B, T, Hkv, d).to(torch.bfloat16).transpose(1, 2)
        # V' rows as the prefill returns them: d of the columns of its padded rows
        vp = _randn(g, B, Hkv, T, 64 if d <= 64 else 128).to(_DTYPES[case["vp"]])[..., :d]
        state.update(table=table, k_pages=_pool(g, pages, Hkv, case["page"], d), v_pages=_pool(g, pages, Hkv, case["page"], d),
                     k=k, vp=vp, lens=torch.tensor(before, dtype=torch.int32, device=DEV),
                     counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
    elif op == "copy":
        n, pages = case["n"], case["pages"]
        base = _randn(g, 2 * case["layers"], pages, case["Hkv"], case["page"], _width(case["d"]), dtype=torch.bfloat16)
        ids = torch.randperm(pages, generator=g, device=DEV).tolist()
        state.update(base=base, pools=list(base.unbind(0)), src=ids[:n], dst=ids[n:2 * n])
    else:
        R, V, dt = case["R"], case["V"], _DTYPES[case["dtype"]]
        logits = 2.5 * _randn(g, R, V)
        if case["masked"]:
            logits[torch.rand(R, V, generator=g, device=DEV) < case["masked"]] = float("-inf")
            logits[:, 0] = 1.0  # something is allowed in every row
        logits = logits.to(dt)
        # given tokens: sampled from the rows, one in twelve rows without one (padding)
        noise = torch.rand(R, V, generator=g, device=DEV).clamp_(1e-6, 1 - 1e-6).log_().neg_().log_().neg_()
        tokens = noise.add_(logits.float() / case["temperature"]).argmax(-1)
        tokens[torch.rand(R, generator=g, device=DEV) < 1 / 12] = -100
        state.update(logits=logits, tokens=tokens)
        if case["grad"]:
            state["g"] = (_randn(g, R), 0.1 * _randn(g, R), _randn(g, R, case["top"]))
            state["logits"].requires_grad_()
    return state


# --------------------------------------------------------------------------------------------
# one pass: the framework's operators, or their plain forms
# --------------------------------------------------------------------------------------------

def _plain_decode(s):
    case = s["case"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, Hq, L, d = q.shape
    Hkv, page = case["Hkv"], case["page"]
    G, scale = Hq // Hkv, d ** -0.5
    table, lens = s["table"].long(), s["lens"].long()

    def rows(pool):  # [B, Hkv, M page, d]
        return pool[table.clamp(min=0)].transpose(1, 2).reshape(B, Hkv, -1, pool.shape[-1])[..., :d].float()

    def hat(x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)

    kc, vc = rows(s["k_pages"]), rows(s["v_pages"])
    seen = (torch.arange(kc.shape[2], device=DEV) < lens[:, None])[:, None, None]  # [B, 1, 1, M page]
    kh, qg = hat(k), q.reshape(B, Hkv, G, L, d)
    p = torch.where(seen, torch.exp(scale * (kh @ hat(kc).transpose(2, 3)) - 1 / scale), 0.0)
    coupled = v - p @ vc  # minus the cached rows' part
    among = torch.exp(scale * (kh @ kh.transpose(2, 3)) - 1 / scale)
    vp = torch.empty_like(v)
    held = torch.zeros_like(v)  # the new rows as the cache holds them
    for t in range(L):
        vp[:, :, t] = (coupled[:, :, t] - (among[:, :, t:t + 1, :t] @ held[:, :, :t])[:, :, 0]) / among[:, :, t, t, None]
        held[:, :, t] = vp[:, :, t].to(torch.bfloat16).float()
    sc = torch.where(seen, scale * (qg.reshape(B, Hkv, G * L, d) @ kc.transpose(2, 3)), -math.inf)
    sn = scale * (qg.reshape(B, Hkv, G * L, d) @ k.transpose(2, 3))
    later = torch.arange(L, device=DEV)[None] > torch.arange(L, device=DEV)[:, None]
    sn = sn.view(B, Hkv, G, L, L).masked_fill(later, -math.inf).view(B, Hkv, G * L, L)
    m = torch.maximum(sc.amax(-1, keepdim=True), sn.amax(-1, keepdim=True))
    ec, en = torch.exp(sc - m), torch.exp(sn - m)
    o = (ec @ vc + en @ held) / (ec.sum(-1, keepdim=True) + en.sum(-1, keepdim=True))
    live = (lens >= 0)[:, None, None, None]
    o = torch.where(live, o.reshape(B, Hq, L, d).transpose(1, 2), 0.0).to(torch.bfloat16)
    vp = torch.where(live, vp, 0.0)
    # the new rows appended
    b = (lens >= 0).nonzero()[:, 0, None]
    at = lens[b] + torch.arange(L, device=DEV)
    ids = table[b, at // page]
    s["k_pages"][ids, :, at % page, :d] = s["k"].transpose(1, 2)[b[:, 0]]
    s["v_pages"][ids, :, at % page, :d] = held.to(torch.bfloat16).transpose(1, 2)[b[:, 0]]
    return {"o": o, "vprime": vp, "k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}


def _plain_write(s):
    case, d, page = s["case"], s["case"]["d"], s["case"]["page"]
    b, t = (torch.arange(case["T"], device=DEV) < s["counts"][:, None]).nonzero(as_tuple=True)
    at = s["lens"][b].long() + t
    ids = s["table"][b, at // page].long()
    s["k_pages"][ids, :, at % page, :d] = s["k"][b, :, t]
    s["v_pages"][ids, :, at % page, :d] = s["vp"][b, :, t].to(torch.bfloat16)
    return {"k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}


def _plain_copy(s):
    src, dst = (torch.tensor(s[n], device=DEV) for n in ("src", "dst"))
    s["base"][:, dst] = s["base"][:, src]
    return {"pools": s["base"]}


def _plain_logprobs(s):
    case, tokens = s["case"], s["tokens"]
    raw = s["logits"].detach()
    x = raw.float() / case["temperature"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    given = tokens != -100
    at = tokens.clamp(min=0)[:, None]
    out = {"logprobs": torch.where(given, (x.gather(1, at) - lse)[:, 0], 0.0)}
    p = e / z
    logp = x - lse
    out["entropy"] = H = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    if case["top"]:
        idx = torch.sort(raw.float(), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_indices"] = idx
        out["top_logprobs"] = x.gather(1, idx) - lse
    if case["grad"]:
        glp, gh, gtop = s["g"]
        glp = torch.where(given, glp, 0.0)
        dx = -p * (glp + gtop.sum(-1))[:, None] - torch.where(p > 0, p * (logp + H[:, None]), 0.0) * gh[:, None]
        dx.scatter_add_(1, at, glp[:, None])
        if case["top"]:
            dx.scatter_add_(1, idx, gtop)
        out["dlogits"] = (dx / case["temperature"]).to(raw.dtype)
    return out


def _own(s):
    case = s["case"]
    if case["op"] == "decode":
        from lucid_amd.paged import lucid_decode_paged

        with torch.no_grad():
            o, vp = lucid_decode_paged(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"])
        return {"o": o, "vprime": vp, "k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}
    if case["op"] == "write":
        from lucid_amd.paged import write_pages

        write_pages(s["k"], s["vp"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["counts"])
        return {"k_pages": s["k_pages"], "vprime_pages": s["v_pages"]}
    if case["op"] == "copy":
        from lucid_amd.paged import copy_pages

        copy_pages(s["pools"], s["src"], s["dst"])
        return {"pools": s["base"]}
    from lucid_amd.model_ops import token_logprobs

    r = token_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
    out = {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach()}
    if case["top"]:
        out.update(top_indices=r.top_indices, top_logprobs=r.top_logprobs.detach())
    if case["grad"]:
        glp, gh, gtop = s["g"]
        outs, grads = (r.logprobs, r.entropy), (glp, gh)
        if case["top"]:
            outs, grads = outs + (r.top_logprobs,), grads + (gtop,)
        out["dlogits"], = torch.autograd.grad(outs, s["logits"], grads)
    return out


def run(state):
    if own:
        return _own(state)
    plain = {"decode": _plain_decode, "write": _plain_write, "copy": _plain_copy, "logprobs": _plain_logprobs}
    return plain[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "decode":
        B, Hq, Hkv, d, L = (case[n] for n in ("B", "Hq", "Hkv", "d", "new"))
        lens = [n for n in _lengths(case) if n >= 0]
        rows = sum(lens)
        # the cached rows of K and V'; q, k, v, o and the appended rows, V' in fp32
        moved = 4 * rows * Hkv * d + len(lens) * L * d * (4 * Hq + 12 * Hkv)
        return {"bytes": moved, "flops": 4 * (Hq + Hkv) * d * sum(L * n + L * (L + 1) // 2 for n in lens)}
    if op == "write":
        rows = sum(_lengths(case)) * case["Hkv"]
        return {"bytes": rows * (case["d"] * (6 + (2 if case["vp"] == "bf16" else 4))), "flops": 0}
    if op == "copy":
        page = case["Hkv"] * case["page"] * _width(case["d"]) * 2
        return {"bytes": 2 * 2 * case["layers"] * case["n"] * page, "flops": 0}
    n = case["R"] * case["V"] * (2 if case["dtype"] == "bf16" else 4)
    return {"bytes": n * (2 if case["grad"] else 1) + case["R"] * (16 + 12 * case["top"]), "flops": case["R"] * case["V"] * (12 if case["grad"] else 6)}


# --------------------------------------------------------------------------------------------
# the definitions in float64
# --------------------------------------------------------------------------------------------

def _exact_decode(s):
    case = s["case"]
    d, page, L = case["d"], case["page"], case["new"]
    G, scale = case["Hq"] // case["Hkv"], case["d"] ** -0.5
    o = torch.zeros(case["B"], L, case["Hq"], d, dtype=torch.float64, device=DEV)
    vp = torch.zeros(case["B"], case["Hkv"], L, d, dtype=torch.float64, device=DEV)
    kp, vpp = s["k_pages"].double(), s["v_pages"].double()
    for b, n in enumerate(_lengths(case)):
        if n < 0:
            continue
        row = torch.arange(n + L, device=DEV)
        ids = s["table"][b].long()[row // page]
        keys, vals = (p[ids, :, row % page][..., :d].transpose(0, 1).double() for p in (s["k_pages"], s["v_pages"]))
        keys[:, n:] = s["k"][b].double()
        r = (keys.square().sum(-1) / d + EPS).rsqrt()  # [Hkv, n + L]
        for t in range(L):
            m = n + t
            dots = torch.linalg.vecdot(keys[:, m:m + 1], keys[:, :m + 1])
            w = torch.exp(scale * r[:, m:m + 1] * r[:, :m + 1] * dots - 1 / scale)
            new = (s["v"][b, :, t].double() - (w[:, None, :m] @ vals[:, :m])[:, 0]) / w[:, m:]
            vp[b, :, t] = new
            vals[:, m] = new.to(torch.bfloat16).double()
            ask = s["q"][b, :, t].double().reshape(case["Hkv"], G, d)
            a = torch.softmax(scale * (ask @ keys[:, :m + 1].transpose(1, 2).contiguous()), -1)
            o[b, t] = (a @ vals[:, :m + 1]).reshape(case["Hq"], d)
        new = row[n:]
        kp[ids[n:], :, new % page, :d] = keys[:, n:].transpose(0, 1)
        vpp[ids[n:], :, new % page, :d] = vals[:, n:].transpose(0, 1)
    return {"o": o, "vprime": vp, "k_pages": kp, "vprime_pages": vpp}


def _exact_logprobs(s):
    case, T = s["case"], s["case"]["temperature"]
    parts = []
    for r0 in range(0, case["R"], 1024):
        cut = slice(r0, r0 + 1024)
        x = s["logits"].detach()[cut].double() / T
        tok = s["tokens"][cut]
        row = torch.arange(x.shape[0], device=DEV)
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        safe = torch.where(logp == -math.inf, torch.zeros_like(logp), logp)
        out = {"logprobs": torch.where(tok >= 0, logp[row, tok.clamp(min=0)], torch.zeros_like(logp[:, 0])),
               "entropy": -(p * safe).sum(-1)}
        if case["top"]:
            # by (logit, lowest index): a stable descending sort
            best = x.sort(dim=-1, descending=True, stable=True)
            out["top_indices"] = best.indices[:, :case["top"]]
            out["top_logprobs"] = logp.gather(1, out["top_indices"])
        if case["grad"]:
            glp, gh, gtop = (t[cut].double() for t in s["g"])
            glp = glp * (tok >= 0)
            d = -p * ((glp + gtop.sum(-1))[:, None] + gh[:, None] * (safe + out["entropy"][:, None]))
            d[row, tok.clamp(min=0)] += glp
            for i in range(case["top"]):
                d[row, out["top_indices"][:, i]] += gtop[:, i]
            out["dlogits"] = d / T
        parts.append(out)
    return {n: torch.cat([q[n] for q in parts]) for n in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "decode":
        return _exact_decode(s)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "copy":
        out = s["base"].double()
        for i, j in zip(s["src"], s["dst"]):
            out[:, j] = s["base"][:, i].double()
        return {"pools": out}
    d, page = case["d"], case["page"]
    kp, vpp = s["k_pages"].double(), s["v_pages"].double()
    for b, n in enumerate(_lengths(case)):
        at = int(s["lens"][b]) + torch.arange(n, device=DEV)
        ids = s["table"][b].long()[at // page]
        kp[ids, :, at % page, :d] = s["k"][b, :, :n].transpose(0, 1).double()
        vpp[ids, :, at % page, :d] = s["vp"][b, :, :n].transpose(0, 1).double()
    return {"k_pages": kp, "vprime_pages": vpp}
