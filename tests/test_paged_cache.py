"""Bookkeeping of ``LucidPagedCache``: pages, forks, frees and compaction against plain lists of rows, on the CPU
(the page copies in torch)."""
import random

import pytest
import torch

from lucid_amd import paged
from lucid_amd.paged import LucidPagedCache, OutOfPages


@pytest.fixture
def cpu_copies(monkeypatch):
    def copy(pools, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for p in pools:
            p[dst] = p[src]

    monkeypatch.setattr(paged, "copy_pages", copy)


def _append(cache, rows, T, counter, lengths=None):
    """A pass of T tokens: writes a running number into the rows that each sequence gains, in the pools and in the
    plain lists ``rows``."""
    step = cache.begin(len(cache._batch), T)
    k, v = cache.pools(0, 1, 1)
    for i, s in enumerate(cache._batch):
        if s is None:
            assert int(step.lens[i]) == -1
            continue
        n = int(step.lens[i])
        assert n == len(rows[s]) and step.positions[i].tolist() == list(range(n, n + T))
        for t in range(T if lengths is None else lengths[i]):
            counter[0] += 1
            page = int(step.table[i, (n + t) // cache.page_size])
            assert cache._refs[page] == 1, "rows go to a page of the sequence's own"
            k[page, 0, (n + t) % cache.page_size, 0] = counter[0] % 250  # (whole numbers that bf16 holds)
            v[page, 0, (n + t) % cache.page_size, 0] = -(counter[0] % 250)
            rows[s].append(counter[0] % 250)
    cache.commit()


def _check(cache, rows):
    used = [0] * cache.num_pages
    for s, want in rows.items():
        assert cache.length(s) == len(want)
        assert len(cache.pages(s)) >= -(-len(want) // cache.page_size)
        for p in cache.pages(s):
            used[p] += 1
        if want and cache._pools:
            k, v = cache.gather(s, 0)
            assert k[0, :, 0].tolist() == want and v[0, :, 0].tolist() == [-x for x in want]
    assert used == cache._refs
    assert sorted(cache._free) == [p for p in range(cache.num_pages) if not used[p]]


@pytest.mark.parametrize("seed", range(6))
def test_random_histories(cpu_copies, seed):
    """Random passes, forks, frees and compactions: every sequence keeps its rows, pages are counted right, and a
    refused call changes nothing."""
    rng = random.Random(seed)
    cache = LucidPagedCache(rng.choice([6, 20, 40]), rng.choice([1, 3, 4]), device="cpu")
    rows, counter = {}, [0]
    for _ in range(150):
        act = rng.choice(["new", "pass", "pass", "pass", "fork", "fork", "free", "compact"])
        try:
            if act == "new" and len(rows) < 8:
                rows.update({s: [] for s in cache.new(rng.choice([1, 2]))})
            elif act == "pass" and rows:
                some = rng.sample(sorted(rows), rng.randint(1, len(rows)))
                some.insert(rng.randint(0, len(some)), None)
                empty = not any(rows[s] for s in some if s is not None)
                T = rng.randint(1, 5)
                lengths = [rng.randint(0, T) for _ in some] if empty and rng.random() < 0.5 else None
                cache.select(some, lengths)
                _append(cache, rows, T, counter, lengths)
                if lengths is None and rng.random() < 0.5:  # the next pass goes on from the device's lengths
                    _append(cache, rows, 1, counter)
            elif act == "fork" and rows:
                s = rng.choice(sorted(rows))
                child = cache.fork(s)
                rows[child] = list(rows[s])
            elif act == "free" and rows:
                s = rng.choice(sorted(rows))
                cache.free(s)
                del rows[s]
            elif act == "compact":
                cache.compact()
                assert sorted(cache._free) == list(range(cache.num_pages - cache.free_pages, cache.num_pages))
        except OutOfPages:
            if rows and rng.random() < 0.5:
                s = rng.choice(sorted(rows))
                cache.free(s)
                del rows[s]
        _check(cache, rows)


def test_forks_share_full_pages_and_copy_the_partial_one(cpu_copies):
    cache = LucidPagedCache(10, 4, device="cpu")
    rows = {s: [] for s in cache.new(2)}
    cache.select([0, 1], [9, 4])
    _append(cache, rows, 9, [0], [9, 4])
    assert cache.pages(0) == [0, 1, 2] and cache.pages(1) == [3]
    a, b = cache.fork(0), cache.fork(1)
    rows[a], rows[b] = list(rows[0]), list(rows[1])
    assert cache.pages(a) == [0, 1, 4] and cache.pages(b) == [3] and cache.free_pages == 5
    cache.select([a, b, 0, 1])
    _append(cache, rows, 1, [100])
    _check(cache, rows)
    assert cache.pages(b) == [3, 5] and cache.pages(1) == [3, 6]
    cache.free(0, 1)
    assert cache.pages(a) == [0, 1, 4] and sorted(cache._free) == [2, 6, 7, 8, 9]
    rows = {a: rows[a], b: rows[b]}
    assert cache.compact() == 1 and cache.pages(b) == [3, 2]
    _check(cache, rows)


def test_refusals(cpu_copies):
    with pytest.raises(ValueError, match="positive"):
        LucidPagedCache(0)
    cache = LucidPagedCache(4, 4, device="cpu")
    a, b = cache.new(2)
    with pytest.raises(ValueError, match="twice"):
        cache.select([a, a])
    with pytest.raises(ValueError, match="no sequence"):
        cache.select([7])
    with pytest.raises(ValueError, match="one length"):
        cache.select([a, b], [1])
    cache.select([a, b])
    with pytest.raises(ValueError, match="selected sequences"):
        cache.begin(3, 1)
    with pytest.raises(OutOfPages):
        cache.begin(2, 9)
    assert cache.free_pages == 4 and cache.pages(a) == []
    with pytest.raises(RuntimeError, match="no forward pass"):
        cache.step
    cache.select([a, b], [3, 5])
    with pytest.raises(ValueError, match="at most its tokens"):
        cache.begin(2, 4)
    rows = {a: [], b: []}
    cache.select([a, b])
    _append(cache, rows, 5, [0])
    cache.select([a, b], [1, 1])
    with pytest.raises(ValueError, match="prefill"):
        cache.begin(2, 1)
    with pytest.raises(OutOfPages):  # the partial page has nowhere to go
        cache.fork(a)
    with pytest.raises(KeyError):
        cache.free(b, 99)
    with pytest.raises(ValueError, match="freed twice"):
        cache.free(b, b)
    assert cache.length(b) == 5
    with pytest.raises(ValueError, match="holds pages"):
        cache.pools(0, 2, 64)
    cache.free(a)
    with pytest.raises(ValueError, match="selected sequences"):  # a freed sequence ends the selection
        cache.begin(2, 1)
