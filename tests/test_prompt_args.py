"""What the prompt operators (chunks behind a paged cache, rotary positions, constraints on logits) refuse, checked on the host
before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

from lucid_amd import _lib

PTR = ctypes.c_void_p(1 << 20)


@pytest.fixture(scope="module")
def lib():
    import os

    from lucid_amd import build
    if not all(os.path.exists(_lib.lib_path(n)) for n in build.TARGETS):
        build.build()
    return _lib.load()


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _err(lib, rc, text):
    assert rc == _lib.LUCID_EINVAL
    assert text in lib.lucid_last_error(), lib.lucid_last_error()


def test_entry_points_are_counted(lib):
    assert lib.lucid_abi_version() == 6 and lib.lucid_abi_minor() >= 2


def test_workspaces(lib):
    ws = lib.lucid_prefill_paged_workspace_bytes
    assert ws(1, 4, 2, 100, 64, 100, 64) > 0
    for bad in ((0, 4, 2, 9, 64, 100, 64), (1, 3, 2, 9, 64, 100, 64), (1, 4, 2, 0, 64, 100, 64), (1, 4, 2, 9, 0, 100, 64),
                (1, 4, 2, 9, 64, 0, 64), (1, 4, 2, 9, 64, 100, 129), (1, 4, 2, 9, 64, 100, 0), (70000, 4, 2, 9, 64, 100, 64),
                (1, 4, 2, 9, 1 << 20, 1 << 20, 64), (1, 8, 1, 1 << 22, 64, 100, 64), (65535, 64, 64, 2000, 64, 4, 64)):
        assert ws(*bad) == 0, bad
    # the workspace does not fall as the batch or the chunk grows
    for d in (64, 68, 96, 128):
        sizes = [[ws(b, 8, 2, L, 16, 50, d) for L in (1, 16, 17, 256, 257, 3000)] for b in (1, 7, 64, 300)]
        assert all(x <= y for row in sizes for x, y in zip(row, row[1:]))
        assert all(x <= y for a, b in zip(sizes, sizes[1:]) for x, y in zip(a, b))


def _prefill(lib, **kw):
    a = dict(k_pages=PTR, ks=_s(8192, 4096, 64), v_pages=PTR, vs=_s(8192, 4096, 64), table=PTR, tstride=8, lens=PTR, ws=PTR,
             o=PTR, q=PTR, B=1, Hq=4, Hkv=2, L=20, P=8, page=64, M=8, D=64, scale=0.125)
    a.update(kw)
    s = _s(256, 64, 64)
    return lib.lucid_prefill_paged(a["q"], s, PTR, s, PTR, s, a["k_pages"], a["ks"], a["v_pages"], a["vs"], a["table"],
                                   a["tstride"], a["lens"], None, a["o"], s, a["ws"], a["B"], a["Hq"], a["Hkv"], a["L"], a["P"],
                                   a["page"], a["M"], a["D"], a["scale"], 1e-5, None)


@pytest.mark.parametrize("kw,text", [
    (dict(D=129), b"head_dim"), (dict(D=0), b"head_dim"), (dict(Hq=3), b"multiple of Hkv"), (dict(B=0), b"positive"),
    (dict(L=0), b"positive"), (dict(P=0), b"no pages"), (dict(page=1 << 20, M=1 << 12), b"2^30"), (dict(table=None), b"null"),
    (dict(lens=None), b"null"), (dict(ws=None), b"null"), (dict(o=None), b"null"), (dict(q=None), b"null"),
    (dict(ws=ctypes.c_void_p((1 << 20) + 128)), b"256-byte"), (dict(k_pages=None), b"null"),
    (dict(k_pages=ctypes.c_void_p((1 << 20) + 8)), b"16-byte"), (dict(ks=_s(8192, 4096, 60)), b"multiples of 8"),
    (dict(vs=_s(8192, -4096, 64)), b"non-negative"), (dict(P=(1 << 22) + 1), b"64 GB"), (dict(ks=_s(1 << 40, 64, 64)), b"64 GB"),
    (dict(scale=0.0), b"positive and finite"), (dict(scale=-0.1), b"positive and finite"),
    (dict(scale=float("inf")), b"positive and finite"), (dict(scale=float("nan")), b"positive and finite"),
    (dict(tstride=-1), b"table stride"), (dict(B=70000), b"65535"), (dict(L=1 << 24), b"2^24"),
    (dict(B=60000, Hq=64, Hkv=64, L=2000, M=1), b"2^23"), (dict(B=30000, Hq=2, L=64, page=1024, M=1 << 14), b"2^30 pairs")])
def test_prefill_paged_refuses(lib, kw, text):
    _err(lib, _prefill(lib, **kw), text)


def _rotary(lib, **kw):
    a = dict(q=PTR, qs=_s(64, 64, 64), qo=PTR, Hq=2, k=PTR, ks=_s(64, 64, 64), ko=PTR, Hkv=1, pos=PTR, freq=PTR, B=1, T=4, D=64, part=64,
             scale=1.0, inter=0, dtype=0)
    a.update(kw)
    s = _s(64, 64, 64)
    return lib.lucid_rotary(a["q"], a["qs"], a["qo"], s, a["Hq"], a["k"], a["ks"], a["ko"], s, a["Hkv"], a["pos"], 1, 4, 1, a["freq"],
                            1, a["B"], a["T"], a["D"], a["part"], a["scale"], a["inter"], 0, a["dtype"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), b"dtype"), (dict(B=-1), b"negative"), (dict(Hq=-1), b"negative"), (dict(D=0), b"head_dim"),
    (dict(D=257), b"head_dim"), (dict(part=63), b"even part"), (dict(part=66), b"even part"), (dict(part=-2), b"even part"),
    (dict(Hq=2048), b"2048 heads"), (dict(scale=float("nan")), b"finite"), (dict(q=None), b"null"), (dict(qo=None), b"null"),
    (dict(qs=None), b"null"), (dict(k=None), b"null"), (dict(pos=None), b"null"), (dict(freq=None), b"null"),
    (dict(q=ctypes.c_void_p((1 << 20) + 1)), b"misaligned"), (dict(k=ctypes.c_void_p((1 << 20) + 2), dtype=1), b"misaligned"),
    (dict(B=1 << 20, T=1 << 10), b"too many tokens")])
def test_rotary_refuses(lib, kw, text):
    _err(lib, _rotary(lib, **kw), text)


def test_rotary_of_nothing(lib):
    for kw in (dict(B=0), dict(T=0), dict(Hq=0, Hkv=0)):
        assert _rotary(lib, pos=None, **kw) == 0


def _constrain(lib, bwd=False, **kw):
    a = dict(x=PTR, sb=0, st=100, R=2, T=2, V=100, dtype=0, hist=PTR, hs=8, N=8, rep=1.2, pres=0.0, freq=0.0, bs=0, ast=4, out=PTR)
    a.update(kw)
    if bwd:
        return lib.lucid_constrain_logits_bwd(a["x"], a["sb"], a["st"], a["R"], a["T"], a["V"], a["dtype"], a["hist"], a["hs"], a["N"],
                                              None, a["rep"], PTR, a["ast"], PTR, a["out"], None)
    return lib.lucid_constrain_logits(a["x"], a["sb"], a["st"], a["R"], a["T"], a["V"], a["dtype"], a["hist"], a["hs"], a["N"], None, None,
                                      a["rep"], None, a["pres"], None, a["freq"], PTR, a["bs"], PTR, a["ast"], a["out"], None)


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"dtype"), (dict(R=-1), b"multiple"), (dict(R=3), b"multiple"), (dict(T=0), b"multiple"), (dict(V=0), b"V from 1"),
    (dict(V=2000001), b"V from 1"), (dict(st=-1), b"negative strides"), (dict(hs=-1), b"negative strides"),
    (dict(ast=-4), b"negative strides"), (dict(N=-1), b"N >= 0"), (dict(hist=None), b"history"), (dict(rep=0.0), b"positive"),
    (dict(rep=-1.0), b"positive"), (dict(rep=float("inf")), b"positive"), (dict(x=None), b"null"), (dict(out=None), b"null"),
    (dict(x=ctypes.c_void_p((1 << 20) + 1)), b"misaligned"), (dict(R=1 << 26, T=1, V=2000), b"too many rows")])
def test_constrain_refuses(lib, kw, text, bwd):
    _err(lib, _constrain(lib, bwd, **kw), text)


def test_constrain_refuses_penalties(lib):
    _err(lib, _constrain(lib, pres=float("nan")), b"finite")
    _err(lib, _constrain(lib, freq=float("inf")), b"finite")
    _err(lib, _constrain(lib, bs=-1), b"negative strides")
    assert _constrain(lib, R=0, x=None, out=None) == 0 and _constrain(lib, True, R=0, x=None, out=None) == 0


def test_python_refuses_without_a_gpu():
    from lucid_amd import constrain_logits, lucid_prefill_paged, rotary
    x = torch.zeros(1, 1, 4, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(x, x, torch.arange(4), torch.ones(4))
    with pytest.raises(RuntimeError, match="GPU"):
        constrain_logits(torch.zeros(2, 5))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        lucid_prefill_paged(x, x, x, x, x, i[None], i)


def test_chunks_of_a_cache():
    """Lengths go with chunks of sequences that hold rows; the pass is described as one; a selection lasts one pass."""
    from lucid_amd.paged import LucidPagedCache, OutOfPages
    cache = LucidPagedCache(6, 4, device="cpu")
    a, b = cache.new(2)
    cache.select([a, None, b], [3, 0, 0], chunk=True)
    step = cache.begin(3, 3)
    assert step.prefill and step.chunk and step.counts.tolist() == [3, 0, 0]
    cache.commit()
    assert (cache.length(a), cache.length(b)) == (3, 0)
    cache.select([b, None, a], [4, 0, 6], chunk=True)
    step = cache.begin(3, 6)
    assert not step.prefill and step.chunk and step.lens.tolist() == [0, -1, 3] and step.counts.tolist() == [4, 0, 6]
    assert step.positions[2].tolist() == list(range(3, 9)) and len(cache.pages(a)) == 3 and len(cache.pages(b)) == 1
    cache.commit()
    assert (cache.length(a), cache.length(b)) == (9, 4)
    step = cache.begin(3, 1)  # the next pass is an ordinary one
    assert not step.chunk and step.counts is None
    cache.commit()
    cache.select([a], [1])
    with pytest.raises(ValueError, match="chunks"):
        cache.begin(1, 1)
    cache.select([a], [3], chunk=True)
    with pytest.raises(ValueError, match="at most its tokens"):
        cache.begin(1, 2)
    cache.select([a], chunk=True)
    with pytest.raises(OutOfPages):
        cache.begin(1, 40)
    assert cache.length(a) == 10 and cache.begin(1, 2).chunk  # a refused pass changes nothing


def test_workspaces_of_short_tables_and_few_rows(lib):
    """Parts of row tiles are kept only where one can be cut, and 64 rows of each where that is what a row tile has."""
    ws = lib.lucid_prefill_paged_workspace_bytes
    short, few, many = (ws(1, 16, 16, L, 64, pages, 64) for L, pages in ((37, 16), (37, 17), (200, 17)))
    assert short < 4 << 20  # 16 heads' panels (148 KB) and rows (64 KB)
    assert few - short == 2 * 256 * 64 * (64 + 2) * 4
    assert many - short == 2 * 256 * 256 * (64 + 2) * 4
