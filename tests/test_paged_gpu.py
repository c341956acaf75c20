"""GPU parity of the paged cache operators (``lucid_amd.paged``) against their definitions in float64.

A new token t of a sequence whose row j is row j % page of page table[j / page]:
    P_tj = exp(s r_t r_j k_t.k_j - 1/s), r = 1 / sqrt(mean k^2 + eps),
    v'_t = (v_t - sum_{j<t} P_tj w_j) / P_tt,   o_tg = softmax_{j<=t}(s q_tg.k_j) w_j,
w_j the V' rows as the cache holds them (bf16), the call's own earlier tokens among them.  The reference
takes those rows from the pages after the call (the appended ones are checked to be bf16(V') themselves),
so that a value that falls the other way in the rounding to bf16 does not count twice.

Tolerances, elementwise.  A score is a sum of d products in fp32: it is off by at most d 2^-24 sum |x_i k_i| s, and
a probability relatively by that, plus 2^-17 for its bf16 pair, 2^-21 for exp2 and the factors r.  Products
and sums of the second product add (n / 256 + 32) 2^-24 relatively to their magnitudes (chunks of rows summed
separately); so with delta the sum of these, |dV'| <= delta (sum_j P_tj |w_j| + |v_t|) / P_tt and, for numerator and
denominator, |dO| <= 2 delta sum_j p_j |w_j|, plus half a step of bf16, 2^-8 |O|.
"""
import pytest
import torch

from lucid_amd.paged import copy_pages, lucid_decode_paged, page_width, write_pages

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _pool(g, pages, Hkv, page, d, layout="dense", fill=None):
    W = page_width(d)
    if layout == "dense":
        p = torch.zeros(pages, Hkv, page, W, dtype=BF, device="cuda")
    elif layout == "rows":  # [pages, page, Hkv, W] seen as [pages, Hkv, page, W]
        p = torch.zeros(pages, page, Hkv, W, dtype=BF, device="cuda").transpose(1, 2)
    else:  # K and V' of a page beside each other
        p = torch.zeros(pages, 2, Hkv, page, W, dtype=BF, device="cuda")[:, 1]
    p[..., :d] = torch.randn(pages, Hkv, page, d, generator=g, device="cuda") if fill is None else fill
    return p


def _tables(g, lens, extra, page, spare=3, width=2):
    """Tables of sequences with room for extra[b] more rows; ids in no order, unused entries far outside the pool."""
    need = [-(-max(n + e, 0) // page) if n >= 0 else 0 for n, e in zip(lens, extra)]
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + width), -(1 << 30), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pages


def _gather(pool, row, page, n, d):
    """Rows 0 .. n-1 of a sequence as float64 [Hkv, n, d]."""
    j = torch.arange(n, device="cuda")
    return pool[row.long()[j // page], :, j % page][..., :d].transpose(0, 1).double()


def _case(lens, Hq, Hkv, L, d, page, seed=0, layout="dense", kscale=1.0, shared=False, stale=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lens)
    table, pages = _tables(g, lens, [L] * B, page)
    kp, vp = (_pool(g, pages, Hkv, page, d, layout) for _ in range(2))
    if shared:  # keys along one direction: every P_tj near 1
        kp[..., :d] = (torch.randn(1, Hkv, 1, d, generator=g, device="cuda") + 0.1 * kp[..., :d].float()).to(BF)
    q = (kscale * torch.randn(B, L, Hq, d, generator=g, device="cuda")).to(BF).transpose(1, 2)
    k = (torch.randn(B, L, Hkv, d, generator=g, device="cuda")).to(BF).transpose(1, 2)
    v = torch.randn(B, L, Hkv, d, generator=g, device="cuda").to(BF).transpose(1, 2)
    if shared:
        k = kp[table[:, 0].clamp(min=0).long(), :, :1, :d].expand(-1, -1, L, -1) + 0.1 * k
    if stale is not None:  # what no sequence holds: a stale row may hold anything
        live = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            if n > 0:
                j = torch.arange(n, device="cuda")
                live[table[b].long()[j // page], j % page] = True
        for p in (kp, vp):
            p.masked_fill_(~live[:, None, :, None], stale)
    return dict(q=q, k=k, v=v, kp=kp, vp=vp, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def _check(c, o, vnew, before, page, scale=None, eps=1e-5, skip=()):
    """Results and pools after a call against the definition; ``before``: the pools' clones."""
    q, k, v = (c[n].double() for n in ("q", "k", "v"))
    B, Hq, L, d = q.shape
    Hkv = k.shape[1]
    G, s = Hq // Hkv, d ** -0.5 if scale is None else scale
    want_k, want_v = before
    for b, n in enumerate(c["lens"].tolist()):
        if b in skip:
            continue
        if n < 0:
            assert bool((o[b] == 0).all()) and bool((vnew[b] == 0).all())
            continue
        j = torch.arange(n, n + L, device="cuda")
        ids = c["table"][b].long()[j // page]
        want_k[ids, :, j % page] = torch.nn.functional.pad(c["k"][b], (0, want_k.shape[3] - d)).transpose(0, 1)
        want_v[ids, :, j % page] = torch.nn.functional.pad(vnew[b].to(BF), (0, want_v.shape[3] - d)).transpose(0, 1)
        keys, w = _gather(c["kp"], c["table"][b], page, n + L, d), _gather(c["vp"], c["table"][b], page, n + L, d)
        r = (keys.square().mean(-1) + eps).rsqrt()
        mag = keys.abs()
        for t in range(L):
            m = n + t
            base = 2.0 ** -17 + 2.0 ** -20 + (n / 256 + 32) * 2.0 ** -24
            dots = (keys[:, m:m + 1] @ keys[:, :m + 1].transpose(1, 2).contiguous())[:, 0]  # [Hkv, m + 1]
            arg = s * r[:, m:m + 1] * r[:, :m + 1] * dots - 1 / s
            size = abs(s) * r[:, m:m + 1] * r[:, :m + 1] * (mag[:, m:m + 1] @ mag[:, :m + 1].transpose(1, 2).contiguous())[:, 0]
            P = arg.exp()
            delta = base + size * (d + 16) * 2.0 ** -24 + abs(1 / s) * 2.0 ** -22
            ref = (v[b, :, t] - (P[:, None, :m] @ w[:, :m])[:, 0]) / P[:, m:]
            tol = ((P * delta)[:, None, :m] @ w[:, :m].abs())[:, 0] + v[b, :, t].abs() * base
            tol = tol / P[:, m:] + ref.abs() * delta[:, m:]
            err = (vnew[b, :, t].double() - ref).abs()
            assert bool((err <= tol).all()), ("V'", b, t, err.max().item(), (err / tol).max().item())
            ask = q[b, :, t].reshape(Hkv, G, d)
            sc = s * (ask @ keys[:, :m + 1].transpose(1, 2).contiguous())
            size = abs(s) * (ask.abs() @ mag[:, :m + 1].transpose(1, 2).contiguous())
            p = torch.softmax(sc, -1)
            oref = p @ w[:, :m + 1]
            tol = 2 * ((p * (base + size * (d + 16) * 2.0 ** -24)) @ w[:, :m + 1].abs()) + oref.abs() * 2.0 ** -8
            err = (o[b, t].double().reshape(Hkv, G, d) - oref).abs()
            assert bool((err <= tol).all()), ("O", b, t, err.max().item(), (err / tol).max().item())
    # the appended rows, and nothing else (stale NaN compare as bits)
    for got, want in ((c["kp"], want_k), (c["vp"], want_v)):
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16))


def _go(c, page, **kw):
    before = c["kp"].clone(), c["vp"].clone()
    o, vnew = lucid_decode_paged(c["q"], c["k"], c["v"], c["kp"], c["vp"], c["table"], c["lens"], **kw)
    torch.cuda.synchronize()
    B, Hq, L, d = c["q"].shape
    assert o.shape == (B, L, Hq, d) and o.dtype == BF and vnew.shape == (B, c["k"].shape[1], L, d)
    _check(c, o, vnew, before, page, scale=kw.get("scaling"), eps=kw.get("eps", 1e-5))
    return o, vnew


@pytest.mark.parametrize("lens,Hq,Hkv,L,d,page", [
    ([0], 1, 1, 1, 64, 16), ([1], 2, 2, 1, 64, 16), ([300], 16, 16, 1, 64, 64), ([127, 128, 129], 4, 2, 1, 64, 64),
    ([5, -1, 300, 0], 4, 1, 1, 64, 16), ([31, 32, 33, 64], 8, 8, 1, 128, 32), ([1000], 8, 1, 1, 128, 256),
    ([70, 2000], 32, 4, 1, 68, 16), ([90], 5, 1, 1, 80, 48), ([257, 40], 6, 2, 1, 96, 7), ([33], 2, 1, 1, 20, 1),
    ([50, 90], 3, 3, 1, 1, 16), ([513], 4, 4, 1, 127, 64), ([100], 31, 1, 1, 64, 16), ([100, 3], 33, 1, 1, 64, 16),
    ([70], 64, 1, 1, 128, 16), ([4097], 4, 4, 1, 64, 4096),
    # several tokens a call: one tile, two tiles, several passes, two groups of query heads
    ([300, 0, -1], 4, 4, 5, 64, 16), ([130], 8, 2, 13, 64, 16), ([1000, 17], 8, 1, 7, 128, 64), ([0], 4, 2, 9, 64, 4),
    ([77], 2, 1, 20, 68, 16), ([200, 31], 12, 2, 5, 96, 64), ([129], 40, 1, 3, 64, 16), ([90, 1], 33, 1, 2, 80, 16),
    ([500], 1, 1, 16, 128, 128), ([15, 16, 17], 16, 4, 8, 128, 16)])
def test_decode_rows(lens, Hq, Hkv, L, d, page):
    print(f"case paged decode lens={lens} Hq={Hq} Hkv={Hkv} L={L} d={d} page={page}", flush=True)
    _go(_case(lens, Hq, Hkv, L, d, page, seed=sum(lens) + d), page)


@pytest.mark.parametrize("d", [64, 68, 128])
def test_decode_passes_of_unequal_tokens(d):
    """Eight tokens of eight query heads in a pass of two column tiles and one of one, in shares of their own."""
    print(f"case paged decode unequal passes d={d}", flush=True)
    _go(_case([3000, 40, -1, 700], 16, 2, 8, d, 64, seed=d), 64)


@pytest.mark.parametrize("d", [58, 68, 125, 127])
def test_first_token_divides_by_the_exact_diagonal(d):
    """V' of a sequence's first token is v / P_tt: an exponential (2^-23) and a product (2^-24), with no error from a scale
    d^-1/2 that fp32 does not hold (which alone makes 15 2^-24 at d = 127)."""
    print(f"case paged first token d={d}", flush=True)
    c = _case([0, 0, 0], 2, 2, 1, d, 16, seed=d)
    _, vnew = _go(c, 16)
    ms, s = c["k"].double().square().mean(-1, keepdim=True), d ** -0.5
    want = c["v"].double() / (s * d * ms / (ms + 1e-5) - 1 / s).exp()
    assert bool(((vnew.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("layout", ["rows", "pairs"])
@pytest.mark.parametrize("d", [64, 68, 128])
def test_decode_other_pool_layouts(layout, d):
    print(f"case paged layout {layout} d={d}", flush=True)
    _go(_case([200, 33, -1], 4, 2, 2, d, 16, layout=layout), 16)


def test_decode_operands_of_any_strides():
    """Query, key and value rows at odd offsets and row strides (no 8-byte boundaries), a strided table."""
    c = _case([100, 61], 4, 2, 3, 68, 16, seed=4)
    want = _case([100, 61], 4, 2, 3, 68, 16, seed=4)
    for n in ("q", "k", "v"):
        B, H, L, d = c[n].shape
        base = torch.full((B, L, H, d + 1), float("nan"), dtype=BF, device="cuda").reshape(-1)
        base = torch.cat([base, base])[1:1 + B * L * H * (d + 1)].view(B, L, H, d + 1)
        base[..., :d] = c[n].transpose(1, 2)
        c[n] = base[..., :d].transpose(1, 2)
        assert c[n].stride(3) == 1 and c[n].data_ptr() % 4
    wide = torch.full((2, c["table"].shape[1] + 5), 7, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = c["table"]
    c["table"] = wide[:, 2:-3]
    o, vn = _go(c, 16)
    o2, vn2 = lucid_decode_paged(*(want[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")))
    assert torch.equal(o, o2) and torch.equal(vn, vn2)


@pytest.mark.parametrize("stale", [float("nan"), float("inf")])
def test_stale_rows_and_columns_do_not_leak(stale):
    """Rows that no sequence holds -- behind the last row of a page, in free pages -- may hold anything."""
    for d, page in ((64, 64), (68, 16), (128, 48)):
        _go(_case([1, 47, 0, 130, -1], 4, 2, 2, d, page, stale=stale, seed=d), page)


def test_many_sequences_of_uneven_lengths():
    """More sequences than lanes; one far longer than the others."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(-1, 60, (150,), generator=g).tolist()
    lens[77] = 9000
    lens[149] = 700
    _go(_case(lens, 4, 2, 1, 64, 16, seed=2), 16)
    _go(_case(lens[60:90], 8, 2, 3, 128, 32, seed=3), 32)
    for d in (68, 96, 128):  # each row width's own number of lanes
        _go(_case(lens[:100], 2, 1, 2, d, 16, seed=d), 16)


def test_sharp_softmax_shared_keys_and_other_scales():
    """Scores up to several hundred (one key takes all), keys along one direction (P_tj near 1, V' many times V), a
    scale other than d^-1/2 and an epsilon of its own."""
    _go(_case([700, 65], 4, 2, 2, 64, 16, kscale=40.0), 16)
    _go(_case([300, 20], 4, 2, 1, 64, 16, shared=True), 16)
    _go(_case([300, 20], 4, 2, 3, 128, 16, shared=True), 16)
    _go(_case([150], 4, 4, 2, 64, 16), 16, scaling=0.3, eps=1e-2)


def test_tokens_in_one_call_equal_calls_of_one_token():
    """V' rows within the fp32 tolerance of the same tokens one a call, O within a step of bf16."""
    for Hq, Hkv, L, d in ((4, 2, 7, 64), (8, 1, 9, 68), (40, 1, 3, 128)):
        a, b = (_case([90, 0, 31], Hq, Hkv, L, d, 16, seed=8) for _ in range(2))
        oa, va = lucid_decode_paged(*(a[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")))
        outs = []
        for t in range(L):
            outs.append(lucid_decode_paged(*(b[n][:, :, t:t + 1] for n in ("q", "k", "v")), b["kp"], b["vp"], b["table"],
                                           b["lens"] + t))
        ob, vb = torch.cat([x[0] for x in outs], 1), torch.cat([x[1] for x in outs], 2)
        # (a value that rounds to the other bf16 neighbour in the cache changes later rows by P times its step)
        assert (va - vb).abs().max().item() <= 2.0 ** -7 * vb.abs().max().item()
        assert (oa.float() - ob.float()).abs().max().item() <= 2.0 ** -6 * ob.float().abs().max().item()
        assert torch.equal(a["kp"], b["kp"])


def test_matches_the_contiguous_cache():
    """Pages in order against lucid_decode on the same rows: that operator's own parity bar, 2e-2."""
    from lucid_amd import lucid_decode
    B, Hq, Hkv, n, d, page = 2, 8, 2, 640, 128, 64
    c = _case([n, n], Hq, Hkv, 2, d, page, seed=12)
    c["q"], c["k"], c["v"] = (x * 0.25 for x in (c["q"], c["k"], c["v"]))
    kc, vc = (torch.zeros(B, Hkv, n + page, d, dtype=BF, device="cuda") for _ in range(2))
    for b in range(B):
        for cache, pool in ((kc, c["kp"]), (vc, c["vp"])):
            cache[b, :, :n] = _gather(pool, c["table"][b], page, n, d).to(BF)
    o, vn = lucid_decode_paged(*(c[x] for x in ("q", "k", "v", "kp", "vp", "table", "lens")))
    o2, vn2 = lucid_decode(c["q"], c["k"], c["v"], kc, vc, n)
    assert (o.float() - o2.float()).abs().max().item() <= 2e-2
    assert (vn - vn2).abs().max().item() <= 2e-2 * vn2.abs().max().item()


def test_bad_tables_poison_their_own_sequence_only():
    """A page id outside the pool among those needed, and a table too short: NaN for that sequence, nothing written
    for it; the others as ever."""
    page, L = 16, 3
    lens = [40, 100, 70, 30, 60, 20]
    c = _case(lens, 4, 2, L, 64, page, seed=6)
    P = c["kp"].shape[0]
    c["table"][0, 1] = P               # a cached page, one past the last
    c["table"][2, 0] = -1              # a cached page, negative
    c["table"][4, 60 // page] = 1 << 30  # the page of the new rows
    full = c["table"].shape[1] * page
    c["lens"][5] = full - L + 1        # one row more than the table holds
    before = c["kp"].clone(), c["vp"].clone()
    o, vn = lucid_decode_paged(*(c[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")))
    torch.cuda.synchronize()
    for b in (0, 2, 4, 5):
        assert bool(torch.isnan(o[b].float()).all()) and bool(torch.isnan(vn[b]).all()), b
    _check(c, o, vn, before, page, skip=(0, 2, 4, 5))


def test_nan_and_infinity_in_live_rows_stay_in_their_sequence():
    """A NaN or an infinity in a cached row reaches the results of its own sequence, head and column as NaN: the
    probability is a sum of two bf16 numbers, hi + lo with lo of either sign or 0, and hi inf + lo inf is NaN (the
    definition's p inf would be inf; cached rows are documented to be finite)."""
    c = _case([50, 60, 70], 4, 2, 1, 64, 16, seed=7)
    ids = c["table"][1].long()
    c["kp"][ids[0], 1, 3, 5] = float("nan")
    c["vp"][ids[1], 0, 2, 9] = float("inf")
    before = c["kp"].clone(), c["vp"].clone()
    o, vn = lucid_decode_paged(*(c[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")))
    torch.cuda.synchronize()
    assert bool(torch.isnan(o[1, 0, 2:].float()).all()) and bool(torch.isnan(o[1, 0, :2, 9].float()).all())
    assert bool(torch.isfinite(o[1, 0, :2, :9].float()).all())
    before[0][ids[60 // 16], :, 60 % 16] = c["kp"][ids[60 // 16], :, 60 % 16]
    before[1][ids[60 // 16], :, 60 % 16] = c["vp"][ids[60 // 16], :, 60 % 16]
    _check(c, o, vn, before, 16, skip=(1,))


def test_offsets_beyond_32_bits():
    """Pages at the far end of pools of more than 2^32 elements."""
    Hkv, page, d, P = 2, 256, 128, 70000
    assert P * Hkv * page * d > 2 ** 32
    kp, vp = (torch.empty(P, Hkv, page, d, dtype=BF, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.tensor([[P - 1, 0, P - 2, 65535]], dtype=torch.int32, device="cuda")
    small = torch.randn(2, 4, Hkv, page, d, generator=g, device="cuda").to(BF)
    kp[ids[0].long()], vp[ids[0].long()] = small[0], small[1]
    q, k, v = (torch.randn(1, h, 1, d, generator=g, device="cuda").to(BF) for h in (4, Hkv, Hkv))
    lens = torch.tensor([3 * page + 7], dtype=torch.int32, device="cuda")
    o, vn = lucid_decode_paged(q, k, v, kp, vp, ids, lens)
    sk, sv = small[0].clone(), small[1].clone()
    o2, vn2 = lucid_decode_paged(q, k, v, sk, sv, torch.arange(4, dtype=torch.int32, device="cuda")[None], lens)
    assert torch.equal(o, o2) and torch.equal(vn, vn2)
    assert torch.equal(kp[65535], sk[3]) and torch.equal(vp[65535], sv[3])
    write_pages(k, v, kp, vp, ids, torch.tensor([2 * page - 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(kp[0, :, page - 1], k[0, :, 0]) and torch.equal(vp[0, :, page - 1], v[0, :, 0])
    copy_pages([kp, vp], [P - 1], [P - 3])
    assert torch.equal(kp[P - 3], kp[P - 1]) and torch.equal(vp[P - 3], vp[P - 1])


def test_captured_decoding_follows_lengths_and_tables():
    """A captured step (decode, lengths advanced) replayed: each replay is the eager step at the lengths and tables of
    that moment.  Two captured steps share no workspace."""
    page, d = 16, 64
    a, b = (_case([30, 5, -1, 47], 4, 2, 1, d, page, seed=21) for _ in range(2))
    room = torch.full((4, 4), 0, dtype=torch.int32, device="cuda")
    free = torch.arange(a["kp"].shape[0], a["kp"].shape[0] + 16, dtype=torch.int32, device="cuda").view(4, 4)
    for c in (a, b):
        c["kp"] = torch.cat([c["kp"], torch.zeros(16, *c["kp"].shape[1:], dtype=BF, device="cuda")])
        c["vp"] = torch.cat([c["vp"], torch.zeros(16, *c["vp"].shape[1:], dtype=BF, device="cuda")])
        t = torch.cat([c["table"], room], 1)
        for i, n in enumerate(c["lens"].tolist()):
            used = -(-max(n + 1, 0) // page) if n >= 0 else 0
            t[i, used:used + 4] = free[i]
        c["table"] = t.contiguous()
    step = torch.tensor([1, 1, 0, 1], dtype=torch.int32, device="cuda")

    def one(c, q, k, v):
        r = lucid_decode_paged(q, k, v, c["kp"], c["vp"], c["table"], c["lens"])
        c["lens"].add_(step)
        return r

    keep = [t.clone() for t in (a["kp"], a["vp"], a["lens"])]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one(a, a["q"], a["k"], a["v"])
    torch.cuda.current_stream().wait_stream(s)
    for t, x in zip((a["kp"], a["vp"], a["lens"]), keep):
        t.copy_(x)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = one(a, a["q"], a["k"], a["v"])
        graphs.append((graph, out))
    for t, x in zip((a["kp"], a["vp"], a["lens"]), keep):
        t.copy_(x)
    g = torch.Generator(device="cuda").manual_seed(5)
    for i in range(20):
        for n in ("q", "k", "v"):
            x = torch.randn(a[n].shape, generator=g, device="cuda").to(BF)
            a[n].copy_(x)
            b[n].copy_(x)
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = one(b, b["q"], b["k"], b["v"])
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i
        assert torch.equal(a["kp"], b["kp"]) and torch.equal(a["vp"], b["vp"]) and torch.equal(a["lens"], b["lens"]), i


def test_side_stream_and_repeated_calls_give_the_same_bits():
    c = _case([400, 33], 8, 2, 3, 128, 16, seed=9)
    args = [c[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")]
    o, vn = lucid_decode_paged(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o2, vn2 = lucid_decode_paged(*args)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(o, o2) and torch.equal(vn, vn2)


def test_empty_calls():
    c = _case([40], 4, 2, 1, 64, 16)
    keep = c["kp"].clone()
    o, vn = lucid_decode_paged(c["q"][:, :, :0], c["k"][:, :, :0], c["v"][:, :, :0], c["kp"], c["vp"], c["table"], c["lens"])
    assert o.shape == (1, 0, 4, 64) and vn.shape == (1, 2, 0, 64)
    o, vn = lucid_decode_paged(c["q"][:0], c["k"][:0], c["v"][:0], c["kp"], c["vp"], c["table"][:0], c["lens"][:0])
    assert o.shape == (0, 1, 4, 64)
    write_pages(c["k"][:0], c["v"][:0], c["kp"], c["vp"], c["table"][:0], c["lens"][:0])
    write_pages(c["k"][:, :, :0], c["v"][:, :, :0], c["kp"], c["vp"], c["table"], c["lens"])
    copy_pages([c["kp"]], [], [])
    copy_pages([torch.empty(0, 4, device="cuda")], [], [])
    assert torch.equal(c["kp"], keep)


def test_refusals_of_shapes_and_types():
    c = _case([40, 3], 4, 2, 1, 64, 16)
    names = ("q", "k", "v", "kp", "vp", "table", "lens")

    def call(**kw):
        return lucid_decode_paged(*(kw.get(n, c[n]) for n in names))

    with pytest.raises(TypeError):
        call(q=c["q"].float())
    with pytest.raises(TypeError):
        call(kp=c["kp"].float())
    with pytest.raises(ValueError, match="disagree"):
        call(q=c["q"][:, :3])
    with pytest.raises(ValueError, match="must be \\[pages"):
        call(kp=c["kp"][:, :1], vp=c["vp"][:, :1])
    with pytest.raises(ValueError, match="must match"):
        call(vp=c["vp"][1:])
    with pytest.raises(ValueError, match="page_table"):
        call(table=c["table"].long())
    with pytest.raises(ValueError, match="page_table"):
        call(table=c["table"][:1])
    with pytest.raises(ValueError, match="cache_lens"):
        call(lens=c["lens"].long())
    with pytest.raises(ValueError, match="cache_lens"):
        call(lens=c["lens"][:1])
    with pytest.raises(ValueError, match="aligned"):
        call(kp=torch.zeros(*c["kp"].shape[:3], 68, dtype=BF, device="cuda")[..., :64],
             vp=torch.zeros(*c["kp"].shape[:3], 68, dtype=BF, device="cuda")[..., :64])
    with pytest.raises(ValueError, match="v_prime"):
        write_pages(c["k"], c["v"].half(), c["kp"], c["vp"], c["table"], c["lens"])
    with pytest.raises(ValueError, match="new_lens"):
        write_pages(c["k"], c["v"], c["kp"], c["vp"], c["table"], c["lens"], c["lens"].long())
    with pytest.raises(ValueError, match="outside"):
        copy_pages([c["kp"]], [0], [c["kp"].shape[0]])
    with pytest.raises(ValueError, match="both read and written"):
        copy_pages([c["kp"]], [0, 1], [1, 2])
    with pytest.raises(ValueError, match="contiguous"):
        copy_pages([c["kp"].transpose(1, 2)], [0], [1])
    with pytest.raises(ValueError, match="share"):
        copy_pages([c["kp"], c["kp"][1:]], [0], [1])


@pytest.mark.parametrize("vdtype", [torch.float32, BF])
@pytest.mark.parametrize("d,page,layout,odd", [(64, 16, "dense", False), (68, 16, "dense", False), (68, 7, "rows", True),
                                               (80, 32, "pairs", False), (96, 64, "dense", True), (128, 64, "rows", False),
                                               (33, 1, "dense", True)])
def test_write_pages(d, page, layout, odd, vdtype):
    """Ragged prompts appended to cached prefixes; idle slots, ids outside the pool, rows beyond the table; everything
    else in the pools as it was."""
    print(f"case write d={d} page={page} {layout} odd={odd} {vdtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(d)
    B, Hkv, T = 6, 3, 75
    lens, counts = [0, 5, -1, 130, 17, 0], [75, 40, 20, 1, 75, 0]
    table, pages = _tables(g, lens, counts, page)
    W = page_width(d)
    kp, vp = (_pool(g, pages, Hkv, page, d, layout, fill=7.0) for _ in range(2))
    pad = d + 1 if odd else 2 * W
    k = torch.randn(B, T, Hkv, pad, generator=g, device="cuda").to(BF)[..., :d].transpose(1, 2)
    v = torch.randn(B, Hkv, T, pad, generator=g, device="cuda").to(vdtype)[..., :d]
    if page > 1:
        table[4, 17 // page + 1] = pages  # one page of sequence 4 lies outside
    want_k, want_v = kp.clone(), vp.clone()
    for b in range(B):
        for t in range(counts[b]):
            j = lens[b] + t
            if lens[b] < 0 or not 0 <= int(table[b, j // page]) < pages:
                continue
            at = (int(table[b, j // page]), slice(None), j % page)
            for want, x in ((want_k, k), (want_v, v)):
                want[at] = 0
                want[at][..., :d] = x[b, :, t].to(BF)
    dl, dc = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, counts))
    write_pages(k, v, kp, vp, table, dl, dc)
    torch.cuda.synchronize()
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    # without counts every row is written; those beyond the table are left out
    M = table.shape[1]
    write_pages(k[:1], v[:1], kp, vp, table[:1], torch.tensor([M * page - 3], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,shape", [(BF, (2, 16, 64)), (torch.float32, (3, 7)), (torch.uint8, (13,)), (BF, (1,)),
                                         (BF, (8, 256, 128)), (torch.float64, ())])
def test_copy_pages(dtype, shape):
    print(f"case copy {dtype} {shape}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    P = 40
    pools = [(100 * torch.rand(P, *shape, generator=g, device="cuda")).to(dtype) for _ in range(3)]
    src, dst = [3, 3, 39, 0, 7], [1, 20, 8, 38, 9]  # a page may be read twice
    want = [p.clone() for p in pools]
    for p in want:
        p[dst] = p[src]
    copy_pages(pools, src, dst)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


def test_copy_pages_of_many_pools_pairs_and_strides():
    """More pools and pairs than one launch takes; pages that are not next to each other; a captured copy."""
    g = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(70, 900, 2, 12, generator=g, device="cuda")
    pools = [base[i][:, 1] for i in range(70)]
    ids = torch.randperm(900, generator=torch.Generator().manual_seed(3)).tolist()
    src, dst = ids[:300], ids[300:600]
    want = base.clone()
    want[:, dst, 1] = base[:, src, 1]
    copy_pages(pools, src, dst)
    torch.cuda.synchronize()
    assert torch.equal(base, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages(pools[:2], ids[600:610], ids[700:710])
    for i in range(3):
        base.normal_(generator=g)
        want = base.clone()
        want[:2, ids[700:710], 1] = base[:2, ids[600:610], 1]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(base, want)


def test_thousands_of_sequences_equal_smaller_batches():
    """3000 sequences (the line of 47 groups of 64), each shorter than a share's unit: the bits of batches of 60."""
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(-1, 100, (3000,), generator=g).tolist()
    for Hq, Hkv, L, d in ((2, 1, 1, 64), (4, 2, 2, 68)):
        c = _case(lens, Hq, Hkv, L, d, 16, seed=d)
        o, vn = lucid_decode_paged(*(c[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")))
        for i in range(0, 3000, 60):
            part = [c[n][i:i + 60] for n in ("q", "k", "v")] + [c["kp"], c["vp"], c["table"][i:i + 60], c["lens"][i:i + 60]]
            o2, vn2 = lucid_decode_paged(*part)
            assert torch.equal(o[i:i + 60], o2) and torch.equal(vn[i:i + 60], vn2), i


def test_calls_on_two_streams_at_once():
    """Two calls in flight (workspaces of their own), each writing its own pools, give what they give one by one."""
    cases = [_case([3000, 500], 8, 2, 2, 128, 16, seed=s) for s in (1, 2)]
    names = ("q", "k", "v", "kp", "vp", "table", "lens")
    want = [lucid_decode_paged(*(c[n].clone() for n in names)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(lucid_decode_paged(*(c[n] for n in names)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(a, b) for r in gs for a, b in zip(r, w))


def test_captured_writes_and_shared_pages():
    """A captured prefill write follows new rows and lengths; two sequences that share full pages (a forked prompt) read
    the same rows and append to pages of their own."""
    g = torch.Generator(device="cuda").manual_seed(4)
    B, Hkv, T, d, page = 2, 2, 20, 64, 16
    table, pages = _tables(g, [0, 0], [40, 40], page)
    kp, vp = (_pool(g, pages, Hkv, page, d) for _ in range(2))
    k = torch.randn(B, Hkv, T, d, generator=g, device="cuda").to(BF)
    v = torch.randn(B, Hkv, T, d, generator=g, device="cuda")
    lens, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [20, 7]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_pages(k, v, kp, vp, table, lens, counts)
    for i in range(3):
        k.normal_(generator=g)
        v.normal_(generator=g)
        lens.copy_(torch.tensor([i, 11 - i], dtype=torch.int32))
        want_k, want_v = kp.clone(), vp.clone()
        write_pages(k, v, want_k, want_v, table, lens, counts)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kp, want_k) and torch.equal(vp, want_v), i
    c = _case([33, 33], 4, 2, 1, d, page, seed=3)
    c["table"][1, :2] = c["table"][0, :2]  # rows 0 .. 31 shared, row 32 and the new one its own
    _go(c, page)
