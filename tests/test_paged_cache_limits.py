"""Calls at the edges of ``LucidPagedCache``'s bookkeeping, on the CPU."""
import pytest
import torch

from lucid_amd import paged
from lucid_amd.paged import LucidPagedCache


def _state(cache):
    return (list(cache._free), list(cache._refs), {s: list(p) for s, p in cache._pages.items()}, dict(cache._lens),
            cache._next, cache._batch)


def test_a_captured_pass_fork_or_compaction_is_refused(monkeypatch):
    """While the current stream is being captured nothing of the bookkeeping runs, and nothing is changed."""
    monkeypatch.setattr(paged, "copy_pages", lambda pools, src, dst: None)
    cache = LucidPagedCache(8, 4, device="cpu")
    a, b = cache.new(2)
    cache.select([a, b])
    cache.begin(2, 5)
    cache.commit()
    cache.free(b)
    cache.select([a])
    before = _state(cache)
    cache.device = torch.device("cuda")  # (as a GPU's cache: only host work is done on it here)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for call in (lambda: cache.begin(1, 1), lambda: cache.fork(a), cache.compact):
        with pytest.raises(RuntimeError, match="captured"):
            call()
        assert _state(cache) == before
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    child = cache.fork(a)
    assert cache.length(child) == 5
