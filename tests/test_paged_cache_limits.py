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


def _two(monkeypatch):
    monkeypatch.setattr(paged, "copy_pages", lambda pools, src, dst: None)
    cache = LucidPagedCache(8, 4, device="cpu")
    a, b, c = cache.new(3)
    cache.select([c, a, b])
    cache.begin(3, 5)
    cache.commit()
    return cache, a, b, c


@pytest.mark.parametrize("what", ["select", "free", "compact"])
def test_a_pass_whose_sequences_or_pages_change_ends(monkeypatch, what):
    """Between begin and commit: another selection, the end of one of the pass's sequences, a compaction (the layers would
    go on in the old pages).  The pass is over, nothing is counted, and the next one goes on from the same lengths."""
    cache, a, b, c = _two(monkeypatch)
    cache.select([a])
    cache.begin(1, 2)
    if what == "select":
        cache.select([b])
    elif what == "free":
        cache.free(a)
    else:
        cache.free(c)
        assert cache.compact() > 0
    with pytest.raises(RuntimeError, match="no forward pass"):
        cache.step
    with pytest.raises(RuntimeError, match="no forward pass"):
        cache.commit()
    assert [cache._lens.get(s) for s in (a, b)] == [None if what == "free" else 5, 5]
    cache.select([b])
    step = cache.begin(1, 1)
    assert step.lens.tolist() == [5] and step.positions.tolist() == [[5]]
    assert step.table[0, :2].tolist() == cache.pages(b)
    cache.commit()
    assert cache.length(b) == 6


def test_a_refused_pass_leaves_none_to_commit(monkeypatch):
    """A pass that was begun and left (an error in a layer), then one that does not fit: commit counts neither.  Ending a
    sequence of no pass leaves the pass as it is."""
    cache, a, b, c = _two(monkeypatch)
    cache.select([a])
    cache.begin(1, 1)
    with pytest.raises(paged.OutOfPages):
        cache.begin(1, 100)
    with pytest.raises(RuntimeError, match="no forward pass"):
        cache.commit()
    assert cache.length(a) == 5
    cache.begin(1, 1)
    cache.free(c)
    cache.commit()
    assert cache.length(a) == 6
