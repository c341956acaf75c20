"""Paged decoding of sequences that share most of their pages (samples of one prompt) and of wide groups of query heads:
definition, tolerances and checks of ``test_paged_gpu``."""
import pytest
import torch

from test_paged_gpu import BF, _case, _go

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,L,d,page,n", [(8, 2, 1, 64, 16, 3000), (16, 4, 5, 128, 64, 4100), (32, 4, 8, 68, 16, 1500),
                                               (64, 2, 1, 128, 64, 2500)])
def test_samples_of_one_prompt(Hq, Hkv, L, d, page, n):
    """Eight sequences on the full pages of one prompt, each with a partial page and rows of its own: each gives what it
    gives with pages of its own, to the bit, and what the definition says."""
    print(f"case shared Hq={Hq} Hkv={Hkv} L={L} d={d} page={page} n={n}", flush=True)
    B = 8
    c = _case([n + 3 * b for b in range(B)], Hq, Hkv, L, d, page, seed=n)
    full = n // page
    own = {k: x.clone() for k, x in c.items()}
    for p in (own["kp"], own["vp"]):  # the prompt's rows copied into everyone's own pages
        for b in range(1, B):
            p[own["table"][b, :full].long()] = p[own["table"][0, :full].long()]
    c["table"][1:, :full] = c["table"][0, :full]
    o, vn = _go(c, page)
    o2, vn2 = _go(own, page)
    assert torch.equal(o, o2) and torch.equal(vn, vn2)


@pytest.mark.parametrize("lens,Hq,Hkv,L,d", [([4000, 9, 700], 32, 1, 1, 128), ([4000, 9, -1, 700], 64, 2, 1, 68),
                                             ([2000, 50], 64, 2, 8, 64), ([1500, 0], 96, 3, 2, 96), ([900, 33], 62, 1, 3, 128),
                                             ([900, 33], 63, 1, 1, 80)])
def test_wide_groups(lens, Hq, Hkv, L, d):
    """32 query heads a kv head and more: chunks of at most 31, of equal and unequal size."""
    print(f"case wide group lens={lens} Hq={Hq} Hkv={Hkv} L={L} d={d}", flush=True)
    _go(_case(lens, Hq, Hkv, L, d, 32, seed=Hq + d), 32)


@pytest.mark.parametrize("d", [64, 68, 128])
def test_calls_repeat_themselves(d):
    """The same call on the same pages gives the same bits each time, whatever order the workgroups run in."""
    c = _case([5000, 3, 900, -1, 17, 2600], 8, 2, 5, d, 16, seed=d)
    from lucid_amd.paged import lucid_decode_paged
    args = [c[n] for n in ("q", "k", "v", "kp", "vp", "table", "lens")]
    o, vn = lucid_decode_paged(*args)
    pools = c["kp"].clone(), c["vp"].clone()
    for _ in range(20):
        o2, vn2 = lucid_decode_paged(*args)
        assert torch.equal(o, o2) and torch.equal(vn, vn2)
        assert torch.equal(c["kp"], pools[0]) and torch.equal(c["vp"], pools[1])
    assert o.dtype == BF
