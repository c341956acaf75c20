"""``lucid_prefill_paged`` where its bookkeeping could go wrong: large batches, captured calls, two streams, shared prefixes, pools
beyond 4 GB, shares that end anywhere, whole rounds of sequences without tokens.  References and tolerances are those of
test_prefill_paged_gpu.py."""
import pytest
import torch

from test_prefill_paged_gpu import BF, call, check, make, run

from lucid_amd.paged import lucid_prefill_paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_batches_beyond_a_wave(B):
    print(f"case B={B}", flush=True)
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(-1, 90, (B,), generator=g).tolist()
    counts = torch.randint(0, 20, (B,), generator=g).tolist()
    run(make(lens, counts, 4, 2, 64, 16, L=20))


def test_most_slots_have_nothing_to_do():
    lens, counts = [-1] * 130, [5] * 130
    lens[129], counts[3], lens[3] = 700, 0, 12
    run(make(lens, counts, 2, 1, 64, 16))
    c = make([5, 9], [0, 0], 2, 1, 64, 16, L=7)
    assert bool((run(c) == 0).all())


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("lens,counts", [([4000, 200, 4000], [130, 3, 64]), ([2600] * 7, [33] * 7), ([130, 5000, 900], [270, 40, 300]),
                                         ([12000], [8]), ([1023, 1024, 1025], [128, 129, 1])], ids=str)
def test_shares_end_anywhere(d, lens, counts):
    """Row tiles cut into parts at many places of a ragged line, for workgroups of every kind."""
    print(f"case d={d} {lens} {counts}", flush=True)
    run(make(lens, counts, 8, 2, d, 32))
    run(make(lens, counts, 2, 2, d, 48, seed=1))


@pytest.mark.parametrize("page", [32, 64, 256, 96, 24])
def test_pages_of_whole_runs_and_others(page):
    """Runs of 32 rows are staged from one page at a time where pages hold whole runs; prefixes that end anywhere in one."""
    for n in (31, 64, 500, 512, 513):
        print(f"case page={page} n={n}", flush=True)
        run(make([n], [300], 4, 2, 64, page, stale=float("nan"), pad=float("nan")))


def test_captured_call_follows_lengths_counts_and_table():
    c = make([300, 40, 0], [60, 60, 60], 4, 2, 64, 16)
    pools = c["kp"].clone(), c["vp"].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(c)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call(c)
    for lens, counts in (([300, 40, 0], [60, 1, 33]), ([10, -1, 5], [3, 60, 0]), ([250, 30, 20], [60, 60, 40])):
        c["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["counts"].copy_(torch.tensor(counts, dtype=torch.int32))
        c["kp"].copy_(pools[0])
        c["vp"].copy_(pools[1])
        graph.replay()
        torch.cuda.synchronize()
        check(c, o, (pools[0].clone(), pools[1].clone()))
        again = dict(c, kp=pools[0].clone(), vp=pools[1].clone())
        assert torch.equal(o, call(again))
        torch.cuda.synchronize()


def test_two_streams_at_once():
    cases = [make([900, 100], [200, 50], 4, 2, 64, 16, seed=i) for i in range(2)]
    before = [(c["kp"].clone(), c["vp"].clone()) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = call(cases[i])
    torch.cuda.synchronize()
    for c, o, b in zip(cases, outs, before):
        check(c, o, b)


def test_shared_prefix():
    """Sequences that share their cached pages and have new ones of their own."""
    c = make([256, 256, 256], [100, 30, 77], 4, 2, 128, 64)
    c["table"][1:, :4] = c["table"][0, :4]
    run(c)


def test_table_of_one_column_and_expanded_operands():
    c = make([10], [50], 4, 2, 64, 64)
    c["table"] = c["table"][:, :1].expand(1, 1)
    run(c)
    c = make([20, 20], [40, 40], 4, 2, 64, 32)
    for n in ("q", "k", "v"):
        c[n] = c[n][:1].expand(2, -1, -1, -1)
    run(c)


def test_pools_beyond_4_gb():
    """Rows whose byte offsets in the pool pass 32 bits."""
    d, page, Hkv = 128, 256, 8
    pages = 9000  # 4.7 GB a pool
    c = make([700], [90], 16, Hkv, d, page)
    need = int((c["table"][0] >= 0).sum())
    kp, vp = (torch.empty(pages, Hkv, page, d, dtype=BF, device="cuda") for _ in range(2))
    new = torch.tensor([pages - 1 - 7 * i for i in range(need)], device="cuda")
    old = c["table"][0, :need].long()
    for big, small in ((kp, "kp"), (vp, "vp")):
        big[new] = c[small][old]
    table = c["table"].clone()
    table[0, :need] = new.int()
    want = lucid_prefill_paged(c["q"], c["k"], c["v"], c["kp"], c["vp"], c["table"], c["lens"], c["counts"])
    got = lucid_prefill_paged(c["q"], c["k"], c["v"], kp, vp, table, c["lens"], c["counts"])
    assert torch.equal(got, want) and torch.equal(kp[new], c["kp"][old]) and torch.equal(vp[new], c["vp"][old])


def test_python_refusals():
    c = make([10, 20], [5, 6], 4, 2, 64, 16)

    def bad(err, match, **kw):
        x = dict(c, **kw)
        with pytest.raises(err, match=match):
            call(x)

    bad(TypeError, "bfloat16", q=c["q"].float())
    bad(TypeError, "bfloat16", k=c["k"].float())
    bad(ValueError, "disagree", v=c["v"][:, :, :4])
    bad(ValueError, "disagree", q=c["q"][:, :3])
    bad(ValueError, "key_pages", kp=c["kp"][..., :32])
    bad(ValueError, "must match", vp=c["vp"][:-1])
    bad(TypeError, "vprime_pages", vp=c["vp"].float())
    bad(ValueError, "cache_lens", lens=c["lens"].long())
    bad(ValueError, "new_lens", counts=c["counts"].cpu())
    bad(ValueError, "new_lens", counts=c["counts"][:1])
    bad(ValueError, "page_table", table=c["table"][:1])
    assert call(dict(c, q=c["q"][:, :, :0], k=c["k"][:, :, :0], v=c["v"][:, :, :0])).shape == (2, 0, 4, 64)


@pytest.mark.parametrize("d", [64, 68, 96, 128])
@pytest.mark.parametrize("lens,counts", [([1500, 900, 2100], [256, 256, 256]), ([1500, 900, 2100, 40], [1, 130, 20, 64]),
                                         ([0, 3000], [500, 512]), ([0, 3000, 77, 1025, 2500], [3, 65, 512, 1, 129])], ids=str)
def test_full_and_ragged_chunks(d, lens, counts):
    """129 to 512 rows a kv head: full chunks take 256 rows to a row tile, ragged ones 64, and both are cut along the keys."""
    print(f"case d={d} {lens} {counts}", flush=True)
    run(make(lens, counts, 2, 2, d, 64))
    run(make(lens, [min(c, 170) for c in counts], 9, 3, d, 16, L=170, seed=1))


def test_captured_call_goes_from_full_to_ragged():
    """The same graph with chunks that fill their row tiles, and with ones that do not."""
    c = make([800, 800, 800], [256, 256, 256], 4, 4, 64, 64)
    pools = c["kp"].clone(), c["vp"].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(c)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call(c)
    for counts in ([256, 256, 256], [3, 70, 1], [256, 0, 200], [10, 10, 10]):
        c["counts"].copy_(torch.tensor(counts, dtype=torch.int32))
        c["kp"].copy_(pools[0])
        c["vp"].copy_(pools[1])
        graph.replay()
        torch.cuda.synchronize()
        check(c, o, (pools[0].clone(), pools[1].clone()))
