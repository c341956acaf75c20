"""What the serving operators refuse, checked on the host before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

from lucid_amd import _lib


@pytest.fixture(scope="module")
def lib():
    from lucid_amd import build
    import os
    if not all(os.path.exists(_lib.lib_path(n)) for n in build.TARGETS):
        build.build()
    return _lib.load()


PTR = ctypes.c_void_p(1 << 20)


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _err(lib, rc, text):
    assert rc == _lib.LUCID_EINVAL
    assert text in lib.lucid_last_error(), lib.lucid_last_error()


def test_page_width_and_workspaces(lib):
    from lucid_amd.paged import page_width
    for d, w in ((1, 64), (64, 64), (65, 80), (68, 80), (80, 80), (81, 96), (96, 96), (97, 128), (128, 128)):
        assert lib.lucid_page_width(d) == w == page_width(d)
    for d in (0, -1, 129):
        assert lib.lucid_page_width(d) == 0
        with pytest.raises(ValueError, match="head_dim"):
            page_width(d)
    ws = lib.lucid_decode_paged_workspace_bytes
    assert ws(1, 4, 2, 1, 64, 100, 64) > 0
    for bad in ((0, 4, 2, 1, 64, 100, 64), (1, 3, 2, 1, 64, 100, 64), (1, 4, 2, 0, 64, 100, 64), (1, 4, 2, 1, 0, 100, 64),
                (1, 4, 2, 1, 64, 0, 64), (1, 4, 2, 1, 64, 100, 129), (1, 4, 2, 1, 1 << 20, 1 << 20, 64)):
        assert ws(*bad) == 0
    # the workspace does not fall as the batch or the table grows
    for d in (64, 68, 96, 128):
        for L in (1, 5, 20):
            sizes = [ws(b, 8, 2, L, 16, m, d) for b in (1, 7, 64, 300) for m in (1, 50, 4000)]
            assert all(x <= y for x, y in zip(sizes[0::3], sizes[3::3])) and sizes[0] <= sizes[1] <= sizes[2]
    assert lib.lucid_token_logprobs_workspace_bytes(8, 32000, 20) == 0
    assert lib.lucid_token_logprobs_workspace_bytes(8, 131072, 20) > 0
    assert lib.lucid_abi_minor() >= 1


def _decode(lib, **kw):
    a = dict(k_pages=PTR, ks=_s(8192, 4096, 64), v_pages=PTR, vs=_s(8192, 4096, 64), table=PTR, tstride=8, lens=PTR, ws=PTR,
             B=1, Hq=4, Hkv=2, L=1, P=8, page=64, M=8, D=64, scale=0.125)
    a.update(kw)
    s = _s(256, 64, 64)
    return lib.lucid_decode_paged(PTR, s, PTR, s, PTR, s, a["k_pages"], a["ks"], a["v_pages"], a["vs"], a["table"],
                                  a["tstride"], a["lens"], PTR, s, PTR, a["ws"], a["B"], a["Hq"], a["Hkv"], a["L"], a["P"],
                                  a["page"], a["M"], a["D"], a["scale"], 1e-5, None)


@pytest.mark.parametrize("kw,text", [
    (dict(D=129), b"head_dim"), (dict(D=0), b"head_dim"), (dict(Hq=3), b"multiple of Hkv"), (dict(B=0), b"positive"),
    (dict(L=0), b"positive"), (dict(P=0), b"no pages"), (dict(page=1 << 20, M=1 << 12), b"2^30"), (dict(table=None), b"null"),
    (dict(lens=None), b"null"), (dict(ws=None), b"null"), (dict(ws=ctypes.c_void_p((1 << 20) + 128)), b"256-byte"),
    (dict(k_pages=None), b"null"), (dict(k_pages=ctypes.c_void_p((1 << 20) + 8)), b"16-byte"),
    (dict(ks=_s(8192, 4096, 60)), b"multiples of 8"), (dict(vs=_s(8192, -4096, 64)), b"non-negative"),
    (dict(P=(1 << 22) + 1), b"64 GB"), (dict(ks=_s(1 << 40, 64, 64)), b"64 GB"), (dict(scale=0.0), b"scale"),
    (dict(tstride=-1), b"table stride"), (dict(B=1 << 20, Hq=8, Hkv=8, M=1), b"2^22"),
    (dict(B=1 << 20, Hq=1, Hkv=1, M=1 << 24, page=64), b"2^38")])
def test_decode_paged_refuses(lib, kw, text):
    _err(lib, _decode(lib, **kw), text)


def test_write_pages_refuses(lib):
    s, p = _s(256, 64, 64), _s(8192, 4096, 64)

    def call(B=1, Hkv=2, T=4, P=8, page=64, M=8, D=64, k=PTR, ks=p, tstride=8):
        return lib.lucid_write_pages(k, s, PTR, s, 1, PTR, ks, PTR, p, PTR, tstride, PTR, None, B, Hkv, T, P, page, M, D, None)

    assert call(B=0) == 0 and call(T=0) == 0
    _err(lib, call(D=130), b"head_dim")
    _err(lib, call(B=-1), b"B in")
    _err(lib, call(B=70000), b"B in")
    _err(lib, call(P=0), b"no pages")
    _err(lib, call(k=None), b"null")
    _err(lib, call(ks=_s(8192, 4096, 68)), b"multiples of 8")
    _err(lib, call(tstride=-8), b"table stride")


def test_copy_pages_refuses(lib):
    def call(src, dst, pages=10, pools=(1 << 20,), stride=64, size=64):
        n, m = len(pools), len(src)
        return lib.lucid_copy_pages(n, (ctypes.c_void_p * n)(*pools), stride, size, pages, m, (ctypes.c_int * m)(*src),
                                    (ctypes.c_int * m)(*dst), None)

    assert call([], []) == 0 and call([1], [2], pools=()) == 0 and call([1], [2], stride=0, size=0) == 0
    _err(lib, call([1], [10]), b"outside")
    _err(lib, call([-1], [1]), b"outside")
    _err(lib, call([1, 2], [3, 3]), b"written twice")
    _err(lib, call([1, 2], [2, 3]), b"both read and written")
    _err(lib, call([1], [1]), b"both read and written")
    _err(lib, call([1], [2], stride=32), b"overlap")
    _err(lib, call([1], [2], pools=(None,)), b"null")
    _err(lib, lib.lucid_copy_pages(1, None, 64, 64, 4, 1, (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(1), None), b"null")


def test_token_logprobs_refuses(lib):
    def fwd(logits=PTR, R=4, T=4, V=1000, dtype=0, temp=1.0, top=3, out=PTR, ws=PTR, sb=0, st=1000):
        return lib.lucid_token_logprobs_fwd(logits, sb, st, PTR, R, T, V, dtype, temp, top, out, PTR, PTR, PTR, PTR, ws, None)

    assert fwd(R=0) == 0
    for kw, text in ((dict(dtype=2), b"dtype"), (dict(R=5), b"multiple"), (dict(V=0), b"V from 1"), (dict(V=3000000), b"V from 1"),
                     (dict(top=65), b"top"), (dict(top=4, V=3), b"top"), (dict(top=-1), b"top"), (dict(temp=0.0), b"temperature"),
                     (dict(temp=float("nan")), b"temperature"), (dict(temp=1e-39), b"temperature"), (dict(temp=float("inf")), b"temperature"),
                     (dict(logits=None), b"null"), (dict(logits=ctypes.c_void_p((1 << 20) + 1)), b"misaligned"),
                     (dict(out=None), b"null"), (dict(V=131072, ws=None), b"null"), (dict(st=-8), b"negative"),
                     (dict(V=131072, ws=ctypes.c_void_p((1 << 20) + 8)), b"256-byte"), (dict(R=1 << 30, T=1), b"too many")):
        _err(lib, fwd(**kw), text)
    rc = lib.lucid_token_logprobs_bwd(PTR, 0, 8, PTR, 4, 4, 8, 0, 1.0, 2, PTR, None, PTR, None, None, PTR, None)
    _err(lib, rc, b"null")
    rc = lib.lucid_token_logprobs_bwd(PTR, 0, 8, PTR, 4, 4, 8, 0, 1.0, 0, PTR, None, PTR, None, None,
                                      ctypes.c_void_p((1 << 20) + 1), None)
    _err(lib, rc, b"misaligned")


def test_python_layer_refuses_cpu_tensors():
    from lucid_amd.model_ops import token_logprobs
    from lucid_amd.paged import copy_pages, lucid_decode_paged, write_pages
    bf = torch.bfloat16
    q, pool = torch.zeros(1, 2, 1, 64, dtype=bf), torch.zeros(4, 2, 16, 64, dtype=bf)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        lucid_decode_paged(q, q, q, pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        write_pages(q, q, pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        copy_pages([pool], [0], [1])
    with pytest.raises(ValueError, match="source and"):
        copy_pages([pool], [0], [1, 2])
    copy_pages([], [0], [1])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
