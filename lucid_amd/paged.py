"""Serving a LUCID decoder from a paged (K, V') cache.

The reference keeps one cache buffer per layer with one length for the whole batch
(``modeling_lucid.py:475-496``); :func:`lucid_amd.lucid.lucid_decode` works on such a buffer.  Here a
layer's cache is two pools of pages that any number of sequences share out among themselves:

* :func:`lucid_decode_paged` -- new tokens of every sequence of a batch against its pages, each sequence at
  its own length (C ``lucid_decode_paged``);
* :func:`write_pages` -- the K and V' rows of a (right-padded) prefill into their pages;
* :func:`copy_pages` -- pages copied in every layer's pools at once.

A pool is bf16 ``[pages, Hkv, page_size, W]`` with ``W = page_width(d)``: the smallest of 64, 80, 96 and 128
columns that holds the head dim, columns from d on zero.  Row j of sequence b is row ``j % page_size`` of page
``page_table[b, j // page_size]``.  Everything runs on the HIP kernels of GPU tensors (there is no CPU path).
"""
from __future__ import annotations

import array
import ctypes
import functools
from typing import Sequence

import torch

from . import _lib


def page_width(d: int) -> int:
    """Columns of a page's rows for head dim ``d``: 64, 80, 96 or 128."""
    if not 1 <= d <= 128:
        raise ValueError(f"lucid_amd: head_dim {d} not supported (supported: 1 .. 128)")
    return 64 if d <= 64 else 80 if d <= 80 else 96 if d <= 96 else 128


@functools.lru_cache(maxsize=4096)
def _strides(stride: tuple):
    """The first three of a tensor's strides as the C entry points take them (they only read the array)."""
    return (ctypes.c_int64 * 3)(*stride[:3])


def _pools_ok(key_pages, vprime_pages, Hkv, W, device) -> bool:
    P, H, page, w = key_pages.shape
    a, b, c, e = s = key_pages.stride()
    if vprime_pages.stride() != s:
        x, y, z, f = vprime_pages.stride()
        a, b, c, e = a | x, b | y, c | z, e if f == 1 else 0
    return (H == Hkv and w == W and page > 0 and e == 1 and not (a | b | c) & 7
            and not (key_pages.data_ptr() | vprime_pages.data_ptr()) & 15 and vprime_pages.shape == key_pages.shape
            and key_pages.dtype is torch.bfloat16 and vprime_pages.dtype is torch.bfloat16
            and key_pages.device == device and vprime_pages.device == device)


def _refuse(what, device, dims, key_pages, vprime_pages, page_table, lens):
    """Says what is wrong with the pools, the table or the lengths of a call."""
    B, Hkv, d = dims
    W = page_width(d)
    for name, t in (("key_pages", key_pages), ("vprime_pages", vprime_pages)):
        if t.dtype != torch.bfloat16 or t.dim() != 4 or t.device != device:
            raise TypeError(f"lucid_amd.{what}: {name} must be a 4-D bfloat16 tensor on {device}")
        if t.shape[1] != Hkv or t.shape[3] != W or t.shape[2] < 1:
            raise ValueError(f"lucid_amd.{what}: {name} must be [pages, {Hkv}, page_size, {W}] for {Hkv} kv heads of "
                             f"head_dim {d}, got {tuple(t.shape)}")
        s = t.stride()
        if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16:
            raise ValueError(f"lucid_amd.{what}: {name} needs a contiguous last axis and 8-element aligned strides")
    if key_pages.shape != vprime_pages.shape:
        raise ValueError(f"lucid_amd.{what}: key_pages {tuple(key_pages.shape)} and vprime_pages "
                         f"{tuple(vprime_pages.shape)} must match")
    for name, t in lens:
        if t.dtype != torch.int32 or t.shape != (B,) or t.device != device or not t.is_contiguous():
            raise ValueError(f"lucid_amd.{what}: {name} must be contiguous int32 [{B}] on {device}")
    raise ValueError(f"lucid_amd.{what}: page_table must be int32 [{B}, max_pages] on {device}, rows contiguous")


def _table_ok(page_table, B, device) -> bool:
    return (page_table.dtype is torch.int32 and page_table.dim() == 2 and page_table.shape[0] == B
            and page_table.shape[1] > 0 and page_table.stride(1) == 1 and page_table.device == device)


def _lens_ok(t, B, device) -> bool:
    return t.dtype is torch.int32 and t.shape == (B,) and t.is_contiguous() and t.device == device


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 else t.contiguous()


def lucid_decode_paged(query, key, value, key_pages, vprime_pages, page_table, cache_lens, scaling=None, eps=1e-5):
    """L new tokens of every sequence of a batch against its pages: :func:`lucid_amd.lucid.lucid_decode` for
    sequences of different lengths in a paged cache.

    ``query [B, Hq, L, d]``, ``key/value [B, Hkv, L, d]`` (bf16, any strides with a contiguous last axis; keys
    with RoPE applied); ``key_pages`` / ``vprime_pages`` bf16 ``[pages, Hkv, page_size, page_width(d)]``;
    ``page_table`` int32 ``[B, max_pages]`` and ``cache_lens`` int32 ``[B]`` on the same device (read by the kernels:
    no synchronisation, and a captured call follows them).  The new rows are written at rows ``cache_lens[b] ..
    cache_lens[b] + L - 1``, whose pages have to be in the table and belong to that sequence alone;
    ``cache_lens`` is not advanced.  L tokens in one call give what L calls of one token give (each new token is
    coupled to, and attends to, the earlier ones' V' rows as the cache holds them, in bf16).

    Returns ``(O [B, L, Hq, d], V' fp32 [B, Hkv, L, d])``.  A slot with a negative length holds no sequence: its
    results are zeros.  A sequence that needs a page id outside the pool, or more rows than its table has, gets
    NaN results and nothing is written for it.  Cached rows have to be finite: a NaN or an infinity in one gives
    NaN in the results of its sequence and head that it enters.  Not differentiable.
    """
    device = query.device
    if not query.is_cuda:
        raise RuntimeError("lucid_amd: query must be a GPU tensor (no CPU path)")
    bf = torch.bfloat16
    if not (query.dtype is key.dtype is value.dtype is bf and query.dim() == key.dim() == 4 and key.device == device
            and value.device == device):
        raise TypeError(f"lucid_amd.lucid_decode_paged: query, key and value must be 4-D bfloat16 tensors on {device}")
    B, Hkv, L, d = key.shape
    Hq = query.shape[1]
    if value.shape != key.shape or query.shape != (B, Hq, L, d) or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("lucid_amd.lucid_decode_paged: query [B, Hq, L, d], key and value [B, Hkv, L, d] disagree")
    if not (key_pages.dim() == 4 and vprime_pages.dim() == 4
            and _pools_ok(key_pages, vprime_pages, Hkv, page_width(d), device)
            and _table_ok(page_table, B, device) and _lens_ok(cache_lens, B, device)):
        _refuse("lucid_decode_paged", device, (B, Hkv, d), key_pages, vprime_pages, page_table,
                (("cache_lens", cache_lens),))
    o = torch.empty((B, L, Hq, d), dtype=bf, device=device)
    vp_new = torch.empty((B, Hkv, L, d), dtype=torch.float32, device=device)
    if B == 0 or L == 0:
        return o, vp_new
    lib = _lib.load()
    P, _, page, _ = key_pages.shape
    M = page_table.shape[1]
    nbytes = lib.lucid_decode_paged_workspace_bytes(B, Hq, Hkv, L, page, M, d)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    q, k, v = _rows(query), _rows(key), _rows(value)
    with _lib.on(device):
        rc = lib.lucid_decode_paged(
            q.data_ptr(), _strides(q.stride()), k.data_ptr(), _strides(k.stride()), v.data_ptr(), _strides(v.stride()),
            key_pages.data_ptr(), _strides(key_pages.stride()), vprime_pages.data_ptr(), _strides(vprime_pages.stride()),
            page_table.data_ptr(), page_table.stride(0), cache_lens.data_ptr(), o.data_ptr(),
            _strides((L * Hq * d, d, Hq * d)), vp_new.data_ptr(), ws.data_ptr(), B, Hq, Hkv, L, P, page, M, d,
            d ** -0.5 if scaling is None else float(scaling), float(eps), _lib.stream_handle(device))
    _lib.check(lib, rc, "lucid_decode_paged")
    return o, vp_new


def write_pages(key, v_prime, key_pages, vprime_pages, page_table, cache_lens, new_lens=None) -> None:
    """The rows of a prefill into their pages: row t of ``key`` (bf16) and ``v_prime`` (bf16, or fp32 as the
    prefill returns it, rounded to bf16), both ``[B, Hkv, T, d]``, goes to row ``cache_lens[b] + t`` of sequence b,
    for ``t < new_lens[b]`` (int32 ``[B]``; None: all T, the batch is not padded).

    Pools and table as for :func:`lucid_decode_paged`.  Rows of a sequence with a negative length, beyond its
    table or on a page id outside the pool are left out."""
    device = key.device
    if not key.is_cuda:
        raise RuntimeError("lucid_amd: key must be a GPU tensor (no CPU path)")
    if key.dtype != torch.bfloat16 or key.dim() != 4:
        raise TypeError("lucid_amd.write_pages: key must be a 4-D bfloat16 tensor")
    if v_prime.dtype not in (torch.bfloat16, torch.float32) or v_prime.shape != key.shape or v_prime.device != device:
        raise ValueError("lucid_amd.write_pages: v_prime must be a bf16 or fp32 tensor shaped like key, on its device")
    B, Hkv, T, d = key.shape
    if not (key_pages.dim() == 4 and vprime_pages.dim() == 4
            and _pools_ok(key_pages, vprime_pages, Hkv, page_width(d), device)
            and _table_ok(page_table, B, device) and _lens_ok(cache_lens, B, device)
            and (new_lens is None or _lens_ok(new_lens, B, device))):
        lens = (("cache_lens", cache_lens),) if new_lens is None else (("cache_lens", cache_lens), ("new_lens", new_lens))
        _refuse("write_pages", device, (B, Hkv, d), key_pages, vprime_pages, page_table, lens)
    lib = _lib.load()
    P, _, page, _ = key_pages.shape
    k, v = _rows(key), _rows(v_prime)
    with _lib.on(device):
        rc = lib.lucid_write_pages(
            k.data_ptr(), _strides(k.stride()), v.data_ptr(), _strides(v.stride()), int(v.dtype == torch.float32),
            key_pages.data_ptr(), _strides(key_pages.stride()), vprime_pages.data_ptr(),
            _strides(vprime_pages.stride()), page_table.data_ptr(), page_table.stride(0), cache_lens.data_ptr(),
            None if new_lens is None else new_lens.data_ptr(), B, Hkv, T, P, page, page_table.shape[1], d,
            _lib.stream_handle(device))
    _lib.check(lib, rc, "lucid_write_pages")


def copy_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """``pool[dst[i]] = pool[src[i]]`` for every pool (all layers' key and V' pools, say: tensors ``[pages, ...]`` of
    one shape, dtype and layout on one device, each page contiguous), in one launch per 64 pools and 256 pages.

    ``src`` and ``dst`` are host integers (they travel in the kernels' arguments).  A page may be read any number
    of times, but is written once and not both read and written (ValueError)."""
    if len(src) != len(dst):
        raise ValueError(f"lucid_amd.copy_pages: {len(src)} source and {len(dst)} destination pages")
    if not pools:
        return
    first = pools[0]
    device, shape, stride = first.device, first.shape, first.stride()
    if not first.is_cuda:
        raise RuntimeError("lucid_amd: pools must be GPU tensors (no CPU path)")
    n, m = len(pools), len(src)
    tensor = torch.Tensor
    # (whole lists at a time: this is most of a small call's time)
    if (n > 1 and (list(map(tensor.size, pools)) != [shape] * n or list(map(tensor.stride, pools)) != [stride] * n
                   or list(map(tensor.get_device, pools)) != [device.index] * n
                   or any(t.dtype is not first.dtype for t in pools))):
        raise ValueError("lucid_amd.copy_pages: pools must share shape, strides, dtype and device")
    if first.dim() < 1 or (shape[0] > 0 and not first[0].is_contiguous()):
        raise ValueError("lucid_amd.copy_pages: a page must be contiguous")
    size = first.element_size()
    page_bytes = size * (first.numel() // shape[0] if shape[0] else 0)
    try:
        s, t = array.array("i", src), array.array("i", dst)
    except OverflowError:
        raise ValueError("lucid_amd.copy_pages: page outside the pool") from None
    lib = _lib.load()
    with _lib.on(device):
        rc = lib.lucid_copy_pages(n, (ctypes.c_void_p * n)(*map(tensor.data_ptr, pools)),
                                  max(stride[0] * size, page_bytes) if shape[0] < 2 else stride[0] * size, page_bytes,
                                  shape[0], m, (ctypes.c_int * m).from_buffer(s), (ctypes.c_int * m).from_buffer(t),
                                  _lib.stream_handle(device))
    _lib.check(lib, rc, "lucid_copy_pages")
