"""``lucid_amd.paged.write_pages`` where rows do not fit and where no counts are given: the whole of both pools against
rows written one by one."""
import pytest
import torch

from lucid_amd.paged import page_width, write_pages

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _want(pool, x, table, lens, page, M, d):
    """Every row of x [B, Hkv, T, d] written by itself; rows from M * page on left out."""
    pool = pool.clone()
    for b, n in enumerate(lens):
        if n < 0:
            continue
        for t in range(x.shape[2]):
            j = n + t
            if j < M * page:
                at = (int(table[b, j // page]), slice(None), j % page)
                pool[at] = 0
                pool[at][..., :d] = x[b, :, t].to(BF)
    return pool


@pytest.mark.parametrize("vdtype", [torch.float32, BF])
@pytest.mark.parametrize("d,page,T,odd", [(64, 16, 9, False), (68, 7, 20, True), (128, 64, 70, False), (96, 1, 6, True),
                                          (80, 48, 33, False)])
def test_rows_beyond_the_table_are_left_out(d, page, T, odd, vdtype):
    """No counts: every row of every live sequence, up to the end of its table and no further.  The table is a slice of a
    wider one whose next columns name valid pages of the same pools, so that a row written there would show; one
    sequence ends three rows into the call, one at its first row, one just fits, one is far within, one is idle."""
    print(f"case write limits d={d} page={page} T={T} odd={odd} {vdtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(d + T)
    Hkv, M, W = 2, -(-(T + 3) // page) + 1, page_width(d)
    full = M * page
    lens = [full - 3, full, full - T, 1, -1, full + 5]
    B, wide = len(lens), M + 3
    wide += -(-(T + 6) // page)
    ids = torch.randperm(B * wide + 2, generator=g, device="cuda")[:B * wide].to(torch.int32).view(B, wide)
    table = ids[:, :M]
    kp, vp = (torch.full((B * wide + 2, Hkv, page, W), 7.0, dtype=BF, device="cuda") for _ in range(2))
    pad = d + 1 if odd else W
    k = torch.randn(B, T, Hkv, pad, generator=g, device="cuda").to(BF)[..., :d].transpose(1, 2)
    v = torch.randn(B, Hkv, T, pad, generator=g, device="cuda").to(vdtype)[..., :d]
    host = table.tolist()
    want_k, want_v = (_want(p, x, table.cpu(), lens, page, M, d) for p, x in ((kp, k), (vp, v)))
    written = (want_k != 7.0).any(-1).any(1).sum().item()
    assert written == 3 + 0 + T + T + 0 + 0, written  # (in rows: no row of random values is 7 throughout)
    write_pages(k, v, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    assert table.tolist() == host


def test_decoding_past_the_table_writes_nothing():
    """The same for new rows of a decode: a sequence whose table ends among them gets NaN, and the pages that the wider
    table names next stay as they were."""
    from lucid_amd.paged import lucid_decode_paged
    g = torch.Generator(device="cuda").manual_seed(9)
    page, L = 16, 4
    wide = torch.randperm(24, generator=g, device="cuda").to(torch.int32).view(3, 8)
    kp, vp = (torch.randn(24, 2, page, 64, generator=g, device="cuda").to(BF) for _ in range(2))
    q, k, v = (torch.randn(3, h, L, 64, generator=g, device="cuda").to(BF) for h in (4, 2, 2))
    lens = torch.tensor([3 * page - 2, 3 * page, 3 * page - L], dtype=torch.int32, device="cuda")
    before = kp.clone(), vp.clone()
    o, vn = lucid_decode_paged(q, k, v, kp, vp, wide[:, :3], lens)
    torch.cuda.synchronize()
    assert bool(torch.isnan(o[:2].float()).all()) and bool(torch.isnan(vn[:2]).all())
    assert bool(torch.isfinite(o[2].float()).all())
    last = int(wide[2, 2])
    before[0][last, :, page - L:] = k[2]
    before[1][last, :, page - L:] = vn[2].to(BF)
    assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])
