"""GPU parity of chunks of new tokens behind paged rows (``lucid_amd.paged.lucid_prefill_paged``) with the definition in float64.

With a sequence's rows j = 0 .. n + c - 1, the last c of them new, and w_j the V' rows as the pages hold them (bf16):
    P_tj = exp(s r_t r_j k_t.k_j - 1/s), r = 1 / sqrt(mean k^2 + eps),
    v'_t = (v_t - sum_{j<t} P_tj w_j) / P_tt, w_t = bf16(v'_t),   o_tg = softmax_{j<=t}(s q_tg.k_j) w_j.
The reference takes all w_j from the pages after the call, so that a new row which falls the other way in the rounding to
bf16 does not count twice; the rows themselves are checked against their own v'_t.

Tolerances, elementwise.  A score is a sum of d products in fp32, off by at most d 2^-24 sum |x_i k_i| s, and its exponent's other
factors by 2^-22 of their size; P is off relatively by that and 2^-20 (exp2, r), and by 2^-17 as a bf16 pair; sums
of products add (n / 256 + 64) 2^-24 of their magnitudes.  With delta the sum of these, |dv'_t| <= delta (sum_j P_tj |w_j| +
|v_t|) / P_tt + delta_tt |v'_t|, and half a step of bf16 for the row in the pages, 2^-8 |v'_t|.  The softmax's weights are single
bf16 values, 2^-8, summed as such: |do| <= (2^-8 + 2 delta) (sum_j a_j |w_j| + |o|) + 2^-8 |o|.
"""
import pytest
import torch

from lucid_amd.paged import lucid_decode_paged, lucid_prefill_paged, page_width

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def make(lens, counts, Hq, Hkv, d, page, L=None, seed=0, layout="dense", shared=None, stale=None, pad=None, kscale=1.0):
    """A batch: rows cached and tokens brought of each slot.  stale: what fills rows that no sequence holds; pad: what
    fills the tokens behind a sequence's own; shared: keys along one direction with that spread."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, L, W = len(lens), max(counts) if L is None else L, page_width(d)
    need = [-(-(n + min(c, L)) // page) if n >= 0 else 0 for n, c in zip(lens, counts)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max(need + [1]) + 2), -(1 << 30), dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = ids[at:at + m]
        at += m

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def pool():
        if layout == "dense":
            p = torch.zeros(pages, Hkv, page, W, dtype=BF, device="cuda")
        elif layout == "rows":  # [pages, page, Hkv, W] seen as [pages, Hkv, page, W]
            p = torch.zeros(pages, page, Hkv, W, dtype=BF, device="cuda").transpose(1, 2)
        else:  # K and V' of a page beside each other
            p = torch.zeros(pages, 2, Hkv, page, W, dtype=BF, device="cuda")[:, 1]
        p[..., :d] = randn(pages, Hkv, page, d)
        return p

    kp, vp = pool(), pool()
    q, k, v = ((kscale if h == Hq else 1.0) * randn(B, L, h, d) for h in (Hq, Hkv, Hkv))
    if shared is not None:
        way = randn(1, Hkv, 1, d)
        kp[..., :d] = (way + shared * kp[..., :d].float()).to(BF)
        k = way.transpose(1, 2) + shared * k
    q, k, v = (x.to(BF).transpose(1, 2) for x in (q, k, v))
    if pad is not None:
        for b, c in enumerate(counts):
            for x in (q, k, v):
                x[b, :, max(c, 0):] = pad
    if stale is not None:
        live = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            if n > 0:
                j = torch.arange(n, device="cuda")
                live[table[b].long()[j // page], j % page] = True
        for p in (kp, vp):
            p.masked_fill_(~live[:, None, :, None], stale)

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    return dict(q=q, k=k, v=v, kp=kp, vp=vp, table=table, lens=i32(lens), counts=i32(counts), page=page)


def call(c, counts=True, **kw):
    return lucid_prefill_paged(c["q"], c["k"], c["v"], c["kp"], c["vp"], c["table"], c["lens"], c["counts"] if counts else None, **kw)


def check(c, o, before, scale=None, eps=1e-5, skip=()):
    """Results and pools after a call against the definition; ``before``: the pools' clones."""
    q, k, v = c["q"], c["k"], c["v"]
    B, Hq, L, d = q.shape
    Hkv, page = k.shape[1], c["page"]
    G, s = Hq // Hkv, d ** -0.5 if scale is None else scale
    want_k, want_v = before
    for b, (n, m) in enumerate(zip(c["lens"].tolist(), c["counts"].tolist())):
        m = 0 if n < 0 else min(max(m, 0), L)
        if b in skip:
            continue
        assert bool((o[b, m:] == 0).all()), f"slot {b}: padding"
        if m == 0:
            continue
        j = torch.arange(n + m, device="cuda")
        ids = c["table"][b].long()[j // page]
        new = j[n:]
        want_k[ids[n:], :, new % page] = torch.nn.functional.pad(k[b, :, :m], (0, want_k.shape[3] - d)).transpose(0, 1)
        keys, w = (p[ids, :, j % page][..., :d].transpose(0, 1).double() for p in (c["kp"], c["vp"]))
        want_v[ids[n:], :, new % page] = c["vp"][ids[n:], :, new % page]  # compared by value below
        assert bool((c["vp"][ids[n:], :, new % page][..., d:] == 0).all()), "columns beyond the head dim"
        r = (keys.square().mean(-1) + eps).rsqrt()  # [Hkv, n + m]
        base = 2.0 ** -17 + 2.0 ** -20 + ((n + m) / 256 + 64) * 2.0 ** -24
        rr = abs(s) * r[:, n:, None] * r[:, None, :]
        arg = (1 if s > 0 else -1) * rr * (keys[:, n:] @ keys.transpose(1, 2).contiguous()) - 1 / s
        size = rr * (keys[:, n:].abs() @ keys.abs().transpose(1, 2).contiguous())
        delta = base + size * (d + 16) * 2.0 ** -24 + abs(1 / s) * 2.0 ** -22
        P = arg.exp()
        diag = P[:, :, n:].diagonal(dim1=1, dim2=2)[..., None]  # [Hkv, m, 1]
        dd = delta[:, :, n:].diagonal(dim1=1, dim2=2)[..., None]
        low = j[None, :] < new[:, None]
        P = P.masked_fill(~low, 0.0)
        vd = v[b, :, :m].double()
        ref = (vd - P @ w) / diag
        tol = ((P * delta) @ w.abs() + vd.abs() * base) / diag + ref.abs() * (dd + 2.0 ** -8)
        off = (w[:, n:] - ref).abs() - tol
        assert off.max().item() <= 0, f"slot {b}: V' off by {off.max().item():.3e} more than its tolerance"
        qd = q[b, :, :m].double().reshape(Hkv, G * m, d)
        sc = s * (qd @ keys.transpose(1, 2).contiguous())
        ssize = abs(s) * (qd.abs() @ keys.abs().transpose(1, 2).contiguous())
        sc = sc.view(Hkv, G, m, n + m).masked_fill(j > new[:, None], -torch.inf).view(Hkv, G * m, n + m)
        a = torch.softmax(sc, -1)
        rel = base + ssize.amax(-1, keepdim=True) * (d + 16) * 2.0 ** -24
        want = a @ w
        tol = (2.0 ** -8 + 2 * rel) * (a @ w.abs() + want.abs()) + 2.0 ** -8 * want.abs()
        got = o[b, :m].double().transpose(0, 1).reshape(Hkv, G * m, d)
        off = (got - want).abs() - tol
        assert off.max().item() <= 0, f"slot {b}: O off by {off.max().item():.3e} more than its tolerance"
    assert torch.equal(c["kp"].view(torch.int16), want_k.view(torch.int16)), "key pages"
    assert torch.equal(c["vp"].view(torch.int16), want_v.view(torch.int16)), "V' pages: rows that are not the call's"


def run(c, skip=(), **kw):
    before = c["kp"].clone(), c["vp"].clone()
    o = call(c, **kw)
    torch.cuda.synchronize()
    check(c, o, before, kw.get("scaling"), kw.get("eps", 1e-5), skip)
    return o


@pytest.mark.parametrize("lens,counts", [
    ([0], [1]), ([0], [33]), ([5], [1]), ([300], [37]), ([127], [64]), ([128], [65]), ([129], [128]), ([1000], [129]),
    ([64], [256]), ([700], [257]), ([0], [600]), ([1500], [520]), ([31, -1, 0, 700, 256], [40, 7, 70, 0, 13]),
    ([0, 0, 10], [0, 0, 0])], ids=str)
@pytest.mark.parametrize("Hq,Hkv,d,page", [(4, 4, 64, 64), (8, 2, 128, 16), (8, 1, 68, 16), (6, 2, 96, 32)])
def test_lengths(lens, counts, Hq, Hkv, d, page):
    print(f"case {lens} {counts} {Hq}/{Hkv} d={d} page={page}", flush=True)
    run(make(lens, counts, Hq, Hkv, d, page, L=max(max(counts), 1)))


@pytest.mark.parametrize("d", [1, 7, 8, 17, 64, 65, 80, 81, 97, 127, 128])
@pytest.mark.parametrize("page", [1, 7, 100])
def test_head_dims_and_odd_pages(d, page):
    print(f"case d={d} page={page}", flush=True)
    run(make([150, 3], [70, 140], 3, 1, d, page, seed=d))


@pytest.mark.parametrize("layout", ["dense", "rows", "beside"])
@pytest.mark.parametrize("d", [64, 68, 128])
def test_layouts_stale_rows_and_padding(layout, d):
    """Rows that no sequence holds, and tokens behind a sequence's own, may hold anything."""
    print(f"case {layout} d={d}", flush=True)
    for fill in (float("nan"), float("inf")):
        run(make([40, 0, 333], [100, 37, 300], 4, 2, d, 16, layout=layout, stale=fill, pad=fill))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 1), (31, 1), (64, 2), (40, 8)])
def test_groups(Hq, Hkv):
    print(f"case {Hq}/{Hkv}", flush=True)
    run(make([90, 700], [77, 21], Hq, Hkv, 64, 32))


@pytest.mark.parametrize("spread", [0.02, 0.1, 0.4, 1.0])
@pytest.mark.parametrize("d", [64, 128])
def test_alike_keys(spread, d):
    """Keys along one direction: P near 1, V' solved through large cancelling sums."""
    print(f"case spread={spread} d={d}", flush=True)
    run(make([300, 0], [290, 130], 4, 2, d, 64, shared=spread))


@pytest.mark.parametrize("scale,kscale", [(0.05, 1.0), (0.4, 1.0), (None, 20.0)])
def test_scales(scale, kscale):
    """Other scales, and scores that reach into the hundreds."""
    print(f"case scale={scale} kscale={kscale}", flush=True)
    run(make([260], [150], 4, 2, 64, 64, kscale=kscale), scaling=scale)


def test_negative_scales_are_refused():
    """With s < 0 a key's own P is 1 and those of unlike keys are exp(1/|s|): V' overflows within a few rows."""
    c = make([260], [150], 4, 2, 64, 64)
    with pytest.raises(ValueError, match="positive"):
        call(c, scaling=-0.125)


def test_long_prefix_is_cut_along_the_keys():
    for counts in ([20], [100], [300]):
        print(f"case {counts}", flush=True)
        run(make([9000], counts, 4, 1, 64, 64))
    run(make([9000, 40, 5000], [33, 200, 5], 8, 2, 128, 32))


def test_without_counts_every_row_is_a_token():
    c = make([10, 300], [45, 45], 4, 2, 64, 16)
    before = c["kp"].clone(), c["vp"].clone()
    o = call(c, counts=False)
    check(c, o, before)


def test_counts_beyond_the_chunk_and_negative():
    c = make([10, 300, 7], [45, 45, 45], 4, 2, 64, 16)
    c["counts"] = torch.tensor([1000, -5, 45], dtype=torch.int32, device="cuda")
    run(c)


def test_chunks_give_what_single_tokens_give():
    """A prompt in chunks of any cutting, and token by token in decoding calls, leaves the same rows: up to the fp32
    rounding before the rounding to bf16, one step of it, 2^-7."""
    Hq, Hkv, d, page, n, m = 4, 2, 64, 16, 50, 300
    base = make([n], [m], Hq, Hkv, d, page, seed=3)
    want = None
    for cuts in ([300], [256, 44], [1, 255, 44], [100, 100, 100], [130, 170], None):
        c = {x: (t.clone() if torch.is_tensor(t) else t) for x, t in base.items()}
        outs, at = [], 0
        for step in cuts or [1] * m:
            part = [c[x][:, :, at:at + step] for x in "qkv"]
            lens = torch.tensor([n + at], dtype=torch.int32, device="cuda")
            if cuts:
                outs.append(lucid_prefill_paged(*part, c["kp"], c["vp"], c["table"], lens))
            else:
                outs.append(lucid_decode_paged(*part, c["kp"], c["vp"], c["table"], lens)[0])
            at += step
        got = torch.cat(outs, 1).double(), c["vp"].double()
        if want is None:
            want = got
            continue
        assert (got[1] - want[1]).abs().max().item() <= 2.0 ** -7 * want[1].abs().max().item()
        # O: the weights' rounding on both sides (2^-8 each of weights that sum to one) and its own
        assert (got[0] - want[0]).abs().max().item() <= 2.0 ** -6 * want[1].abs().max().item()


def test_bad_pages_and_short_tables_touch_nothing():
    """A sequence that needs a page outside the pool, or has no room for its rows, gets NaN; its neighbours their results."""
    c = make([100, 70, 64, 30], [40, 40, 40, 40], 4, 2, 64, 16)
    c["table"][0, 2] = c["kp"].shape[0]     # cached, one past the pool
    c["table"][1, 6] = -1                    # of the new rows (70 + 40 rows: 7 pages)
    c["lens"][2] = c["table"].shape[1] * 16 - 39  # one row more than the table has
    before = c["kp"].clone(), c["vp"].clone()
    o = call(c)
    torch.cuda.synchronize()
    assert bool(o[:3].isnan().all())
    check(c, o, before, skip=(0, 1, 2))


def test_lengths_beyond_32_bits_together_are_refused_by_the_sequence():
    c = make([10], [20], 2, 1, 64, 16)
    c["lens"][0] = 2 ** 31 - 5  # its sum with the tokens passes 32 bits
    before = c["kp"].clone(), c["vp"].clone()
    o = call(c)
    torch.cuda.synchronize()
    assert bool(o.isnan().all())
    check(c, o, before, skip=(0,))


def test_strided_operands_and_repeated_calls():
    """Projections as a stacked product leaves them, an odd offset among them; a call repeats itself to the bit."""
    c = make([400, 33], [70, 90], 8, 2, 68, 16)
    B, L, d = 2, 90, 68
    for off in (0, 1):
        buf = torch.zeros(B, L, 12 * d + off, dtype=BF, device="cuda")
        parts = []
        for x, h, at in (("q", 8, 0), ("k", 2, 8), ("v", 2, 10)):
            view = buf[..., off + at * d: off + (at + h) * d].view(B, L, h, d) if not off else \
                buf.as_strided((B, L, h, d), (buf.stride(0), buf.stride(1), d, 1), off + at * d)
            view.copy_(c[x].transpose(1, 2))
            parts.append(view.transpose(1, 2))
        s = dict(c, q=parts[0], k=parts[1], v=parts[2], kp=c["kp"].clone(), vp=c["vp"].clone())
        first = run(s)
        again = call(s)
        assert torch.equal(first, again)
