"""Serving a LUCID decoder from a paged (K, V') cache.

The reference keeps one cache buffer per layer with one length for the whole batch
(``modeling_lucid.py:475-496``); :func:`lucid_amd.lucid.lucid_decode` works on such a buffer.  Here a
layer's cache is two pools of pages that any number of sequences share out among themselves:

* :func:`lucid_decode_paged` -- new tokens of every sequence of a batch against its pages, each sequence at
  its own length (C ``lucid_decode_paged``);
* :func:`lucid_prefill_paged` -- chunks of prompts behind what is cached, each sequence with its own number of tokens (C
  ``lucid_prefill_paged``);
* :func:`write_pages` -- the K and V' rows of a (right-padded) prefill into their pages;
* :func:`copy_pages` -- pages copied in every layer's pools at once;
* :class:`LucidPagedCache` -- the pools, page tables and free pages of a model's sequences: forking (full
  pages are shared, the partial last one is copied), freeing and compacting.

A pool is bf16 ``[pages, Hkv, page_size, W]`` with ``W = page_width(d)``: the smallest of 64, 80, 96 and 128
columns that holds the head dim, columns from d on zero.  Row j of sequence b is row ``j % page_size`` of page
``page_table[b, j // page_size]``.  The operators run on GPU tensors only (there is no CPU path); the cache's
bookkeeping is host work.
"""
from __future__ import annotations

import array
import ctypes
import functools
import heapq
from typing import NamedTuple, Optional, Sequence

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
            and page_table.shape[1] > 0 and (page_table.stride(1) == 1 or page_table.shape[1] == 1)
            and page_table.device == device)


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
    ws = cache_lens.new_empty(max(nbytes, 256) // 4)  # (0.5 us less than torch.empty with a dtype and a device)
    q, k, v = _rows(query), _rows(key), _rows(value)
    with _lib.on(device):
        rc = lib.lucid_decode_paged(
            q.data_ptr(), _strides(q.stride()), k.data_ptr(), _strides(k.stride()), v.data_ptr(), _strides(v.stride()),
            key_pages.data_ptr(), _strides(key_pages.stride()), vprime_pages.data_ptr(),
            _strides(vprime_pages.stride()), page_table.data_ptr(), page_table.stride(0), cache_lens.data_ptr(),
            o.data_ptr(), _strides((L * Hq * d, d, Hq * d)), vp_new.data_ptr(), ws.data_ptr(), B, Hq, Hkv, L, P, page,
            M, d, d ** -0.5 if scaling is None else float(scaling), float(eps), _lib.stream_handle(device))
    _lib.check(lib, rc, "lucid_decode_paged")
    return o, vp_new


def lucid_prefill_paged(query, key, value, key_pages, vprime_pages, page_table, cache_lens, new_lens=None, scaling=None,
                        eps=1e-5):
    """A chunk of new tokens of every sequence of a batch behind its cached rows: a prompt that is read in parts, or that
    follows a cached prefix.

    ``query [B, Hq, L, d]``, ``key/value [B, Hkv, L, d]`` (bf16, any strides with a contiguous last axis; keys with RoPE
    applied), pages, table and lengths as for :func:`lucid_decode_paged`; ``new_lens`` int32 ``[B]``: the tokens that each
    sequence brings (rows behind them are padding and not used; a number beyond L counts as L, a negative one as 0;
    None: L each).  The chunk's K and V' rows are written at rows ``cache_lens[b] ..``, whose pages have to be in the table
    and belong to that sequence alone; ``cache_lens`` is not advanced.  Any cutting of a prompt into calls of this and of
    :func:`lucid_decode_paged` gives the same rows up to rounding: a token is coupled to, and attends to, the V' rows
    before it as the cache holds them.

    The rows are solved to the precision of :func:`lucid_decode_paged`; O's attention weights are single bf16 values, as in
    :func:`lucid_amd.lucid.lucid_attention`, where decoding has pairs: O is off by 0.0024 of its norm, there by 0.0017.

    Returns O ``[B, L, Hq, d]``, zeros in padding and in slots with a negative length.  A sequence that needs a page id
    outside the pool, or more rows than its table has, gets NaN results and nothing is written for it.  Cached rows and the
    tokens' own have to be finite, ``scaling`` positive.  Not differentiable."""
    device = query.device
    if not query.is_cuda:
        raise RuntimeError("lucid_amd: query must be a GPU tensor (no CPU path)")
    bf = torch.bfloat16
    if not (query.dtype is key.dtype is value.dtype is bf and query.dim() == key.dim() == 4 and key.device == device
            and value.device == device):
        raise TypeError(f"lucid_amd.lucid_prefill_paged: query, key and value must be 4-D bfloat16 tensors on {device}")
    B, Hkv, L, d = key.shape
    Hq = query.shape[1]
    if value.shape != key.shape or query.shape != (B, Hq, L, d) or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("lucid_amd.lucid_prefill_paged: query [B, Hq, L, d], key and value [B, Hkv, L, d] disagree")
    if not (key_pages.dim() == 4 and vprime_pages.dim() == 4
            and _pools_ok(key_pages, vprime_pages, Hkv, page_width(d), device)
            and _table_ok(page_table, B, device) and _lens_ok(cache_lens, B, device)
            and (new_lens is None or _lens_ok(new_lens, B, device))):
        lens = (("cache_lens", cache_lens), ("new_lens", new_lens))
        _refuse("lucid_prefill_paged", device, (B, Hkv, d), key_pages, vprime_pages, page_table,
                lens[:1] if new_lens is None else lens)
    o = torch.empty((B, L, Hq, d), dtype=bf, device=device)
    if B == 0 or L == 0:
        return o
    lib = _lib.load()
    P, _, page, _ = key_pages.shape
    M = page_table.shape[1]
    nbytes = lib.lucid_prefill_paged_workspace_bytes(B, Hq, Hkv, L, page, M, d)
    ws = cache_lens.new_empty(max(nbytes, 256) // 4)
    q, k, v = _rows(query), _rows(key), _rows(value)
    with _lib.on(device):
        rc = lib.lucid_prefill_paged(
            q.data_ptr(), _strides(q.stride()), k.data_ptr(), _strides(k.stride()), v.data_ptr(), _strides(v.stride()),
            key_pages.data_ptr(), _strides(key_pages.stride()), vprime_pages.data_ptr(),
            _strides(vprime_pages.stride()), page_table.data_ptr(), page_table.stride(0), cache_lens.data_ptr(),
            None if new_lens is None else new_lens.data_ptr(), o.data_ptr(), _strides((L * Hq * d, d, Hq * d)),
            ws.data_ptr(), B, Hq, Hkv, L, P, page, M, d, d ** -0.5 if scaling is None else float(scaling), float(eps),
            _lib.stream_handle(device))
    _lib.check(lib, rc, "lucid_prefill_paged")
    return o


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
        lens = (("cache_lens", cache_lens), ("new_lens", new_lens))
        _refuse("write_pages", device, (B, Hkv, d), key_pages, vprime_pages, page_table,
                lens[:1] if new_lens is None else lens)
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


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a call needs; nothing was changed."""


class PagedStep(NamedTuple):
    """What the layers of a forward pass read of a :class:`LucidPagedCache` (device tensors of the batch)."""

    table: torch.Tensor             # int32 [B, max_pages] page ids
    lens: torch.Tensor              # int32 [B] rows cached before the pass, -1 for an idle slot
    counts: Optional[torch.Tensor]  # int32 [B] real tokens of each right-padded row (None: all)
    positions: torch.Tensor         # int64 [B, T] of the tokens
    prefill: bool                   # every sequence is empty: the pass is a prefill
    chunk: bool = False             # the rows are chunks of prompts behind what is cached


class LucidPagedCache:
    """The (K with RoPE applied, V') cache of many sequences in pages, for
    :class:`lucid_amd.modeling_lucid.LlamaForCausalLM` in place of its ``LucidCache``.

    Every layer has two pools of ``num_pages`` pages (made on its first pass); a page id is the same page in
    all of them.  :meth:`new` opens sequences, :meth:`select` says which sequence each row of the next forward
    passes belongs to (None: an idle slot), and the passes append to them.  :meth:`fork` gives a sequence that
    shares the full pages of another and has its own copy of the partial last one; :meth:`free` returns pages that no
    sequence uses any more, the lowest free id being given out first; :meth:`compact` moves the pages in use to the
    front of the pools.  The bookkeeping is host work on page ids; only rows and copied pages touch the GPU, on the
    current stream.  A graph would not replay the host's part, so passes, forks and compactions are refused while the
    current stream is being captured (the operators of this module, on tables and lengths of the caller's, are not).
    bf16, one device, not thread safe."""

    def __init__(self, num_pages: int, page_size: int = 64, device="cuda"):
        if num_pages < 1 or page_size < 1:
            raise ValueError("lucid_amd: num_pages and page_size must be positive")
        self.num_pages, self.page_size = num_pages, page_size
        self.device = torch.device(device)
        self._pools: list[tuple[torch.Tensor, torch.Tensor]] = []
        self._free = list(range(num_pages))  # a heap
        self._refs = [0] * num_pages
        self._pages: dict[int, list[int]] = {}
        self._lens: dict[int, int] = {}
        self._next = 0
        self._batch: tuple = ()
        self._lengths: Optional[list[int]] = None
        self._chunk = False
        self._dev: Optional[tuple] = None  # (table, lens, 1 in the live rows) of the selection, on the device
        self._step: Optional[PagedStep] = None

    def _not_captured(self, what: str) -> None:
        if self.device.type == "cuda" and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"lucid_amd: a LucidPagedCache's {what} cannot be captured into a graph: a replay would "
                               "not repeat its bookkeeping")

    # -- sequences -----------------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def new(self, n: int = 1) -> list[int]:
        """``n`` empty sequences; their ids (never used again)."""
        ids = list(range(self._next, self._next + n))
        self._next += n
        for i in ids:
            self._pages[i], self._lens[i] = [], 0
        return ids

    def length(self, seq: int) -> int:
        return self._lens[seq]

    def pages(self, seq: int) -> list[int]:
        """The page ids of a sequence, in order."""
        return list(self._pages[seq])

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def fork(self, seq: int) -> int:
        """A sequence with the rows of ``seq``: its full pages shared, its partial last page copied (all layers in one
        launch).  Raises :class:`OutOfPages` where there is no page for the copy."""
        self._not_captured("fork")
        full, part = divmod(self._lens[seq], self.page_size)
        pages = self._pages[seq]
        if part and not self._free:
            raise OutOfPages("lucid_amd: no free page to fork the last one into")
        (child,) = self.new()
        for page in pages[:full]:
            self._refs[page] += 1
        self._pages[child] = pages[:full]
        self._lens[child] = self._lens[seq]
        if part:
            page = self._take()
            self._pages[child].append(page)
            copy_pages([p for kv in self._pools for p in kv], [pages[full]], [page])
        return child

    def free(self, *seqs: int) -> None:
        """Ends sequences; pages that no other sequence shares are free again."""
        if len(set(seqs)) != len(seqs):
            raise ValueError("lucid_amd: a sequence is freed twice")
        for seq in seqs:
            self._lens[seq]  # (KeyError before anything is changed)
        for seq in seqs:
            if seq in self._batch:
                self._batch, self._dev, self._step = (), None, None
            del self._lens[seq]
            for page in self._pages.pop(seq):
                self._drop(page)

    def compact(self) -> int:
        """Moves the pages in use to the ids 0 .. n - 1 (all layers in one launch); the number of pages moved.  Those
        beyond n go to the free ids below n, in order."""
        self._not_captured("compaction")
        n = self.num_pages - len(self._free)
        src = [p for p in range(n, self.num_pages) if self._refs[p]]
        dst = sorted(p for p in self._free if p < n)
        copy_pages([p for kv in self._pools for p in kv], src, dst)
        to = dict(zip(src, dst))
        for pages in self._pages.values():
            pages[:] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(n, self.num_pages))
        self._dev = self._step = None
        return len(src)

    # -- forward passes ------------------------------------------------------------------------

    def select(self, seqs: Sequence[Optional[int]], lengths: Optional[Sequence[int]] = None, chunk: bool = False) -> None:
        """The sequence of each row of the passes that follow, each at most once (None: an idle slot, whose row of the
        batch is ignored).  ``lengths``: the real tokens of each row of the next pass, a prefill that is padded on
        the right.  ``chunk``: the next pass brings chunks of prompts, behind what the sequences have cached or as their first
        tokens, padded on the right where ``lengths`` are given (:func:`lucid_prefill_paged`: any number of tokens at the
        rate of a prefill, at its precision; one token beside them is a chunk too)."""
        seqs = tuple(seqs)
        live = [s for s in seqs if s is not None]
        if len(set(live)) != len(live):
            raise ValueError("lucid_amd: a sequence is selected twice")
        for s in live:
            if s not in self._lens:
                raise ValueError(f"lucid_amd: no sequence {s}")
        if lengths is not None and (len(lengths) != len(seqs) or any(n < 0 for n in lengths)):
            raise ValueError("lucid_amd: one length per selected row, none negative")
        if seqs != self._batch:
            self._batch, self._dev = seqs, None
        self._lengths = None if lengths is None else [int(n) for n in lengths]
        self._chunk = bool(chunk)
        self._step = None

    def begin(self, B: int, T: int) -> PagedStep:
        """Makes room for a pass of T tokens a row and describes it to the layers (the model calls this).  Raises
        :class:`OutOfPages` before anything is changed."""
        self._not_captured("pass")
        self._step = None
        if len(self._batch) != B:
            raise ValueError(f"lucid_amd: {B} rows, but {len(self._batch)} selected sequences (LucidPagedCache.select)")
        counts = self._lengths
        live = [(i, s) for i, s in enumerate(self._batch) if s is not None]
        past = [self._lens[s] for _, s in live]
        prefill = not any(past)
        if counts is not None and (not (prefill or self._chunk) or max(counts, default=0) > T):
            raise ValueError("lucid_amd: lengths are for a prefill of empty sequences or for chunks, and at most its tokens")
        more = {s: -(-(n + (T if counts is None else counts[i])) // self.page_size) - len(self._pages[s])
                for (i, s), n in zip(live, past)}
        need = sum(m for m in more.values() if m > 0)
        if need > len(self._free):
            raise OutOfPages(f"lucid_amd: {need} pages needed, {len(self._free)} free")
        for s, m in more.items():
            if m > 0:
                self._pages[s].extend(self._take() for _ in range(m))
                self._dev = None
        if self._dev is None:
            width = max([len(self._pages[s]) for _, s in live], default=0)
            table = [self._pages[s] + [-1] * (width + 1 - len(self._pages[s])) if s is not None else [-1] * (width + 1)
                     for s in self._batch]
            lens = [-1 if s is None else self._lens[s] for s in self._batch]
            both = torch.tensor([r + [n, int(n >= 0)] for r, n in zip(table, lens)], dtype=torch.int32).to(self.device)
            self._dev = both[:, :-2], both[:, -2].contiguous(), both[:, -1].contiguous()
        table, lens, ones = self._dev
        positions = lens.clamp(min=0).long()[:, None] + torch.arange(T, device=self.device)
        self._step = PagedStep(table, lens, None if counts is None else
                               torch.tensor(counts, dtype=torch.int32).to(self.device), positions, prefill, self._chunk)
        return self._step

    @property
    def step(self) -> PagedStep:
        """The pass that :meth:`begin` described, until it is committed; a selection, a compaction or the end of one of
        its sequences ends it too, with nothing counted."""
        if self._step is None:
            raise RuntimeError("lucid_amd: no forward pass has begun (LucidPagedCache.begin), or its sequences or pages have "
                               "changed since")
        return self._step

    def commit(self) -> None:
        """Ends a pass: its tokens are part of their sequences (the model calls this)."""
        step, counts = self.step, self._lengths
        T = step.positions.shape[1]
        for i, s in enumerate(self._batch):
            if s is not None:
                self._lens[s] += T if counts is None else counts[i]
        # (out of place: the pass's own tensors stay as its layers saw them)
        table, lens, ones = self._dev
        self._dev = table, lens + (ones * T if step.counts is None else step.counts * ones), ones
        self._lengths = self._step = None
        self._chunk = False

    def pools(self, layer_idx: int, Hkv: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(key_pages, vprime_pages) of a layer."""
        shape = (self.num_pages, Hkv, self.page_size, page_width(d))
        if layer_idx == len(self._pools):
            self._pools.append((torch.zeros(shape, dtype=torch.bfloat16, device=self.device),
                                torch.zeros(shape, dtype=torch.bfloat16, device=self.device)))
        k, v = self._pools[layer_idx]
        if k.shape != shape:
            raise ValueError(f"lucid_amd: the cache holds pages {tuple(k.shape)}, not {shape}")
        return k, v

    def gather(self, seq: int, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Copies of a sequence's rows of a layer, (K, V') [Hkv, rows, page_width(d)]."""
        rows = torch.arange(self._lens[seq], device=self.device)
        ids = torch.tensor(self._pages[seq], dtype=torch.int64).to(self.device)[rows // self.page_size]
        k, v = self._pools[layer_idx]
        return tuple(p[ids, :, rows % self.page_size].transpose(0, 1) for p in (k, v))
