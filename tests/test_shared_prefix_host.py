"""Host bookkeeping of shared pages: holders, prefixes of requests, forks, and the grouping of rows that share."""
import itertools
import random

import pytest
import torch

from delta_amd.scheduler import BatchSlots, PagePool, ServingRequest, shared_prefixes


def test_pages_go_back_with_their_last_holder():
    pool = PagePool(10, seed=0)
    a = pool.take(4)
    assert pool.share(a[:2]) == a[:2]
    pool.give_back(a)
    assert pool.available == 8 and not set(a[:2]) & set(pool._free) and set(a[2:]) <= set(pool._free)
    pool.give_back(a[:2])
    assert pool.available == 10 and sorted(pool._free) == list(range(10))
    pool.give_back(a)  # nobody's: nothing happens
    assert pool.available == 10
    with pytest.raises(RuntimeError, match="not held"):
        pool.share([a[0]])


def _saved(row_prefix, prefixes):
    users = [list(row_prefix.values()).count(p) for p in range(len(prefixes))]
    return sum((n - 1) * len(p) for n, p in zip(users, prefixes))


def _best(rows):
    """Most pages that any choice of disjoint groups with a common prefix spares, by trying all partitions."""
    def partitions(xs):
        if not xs:
            yield []
            return
        for rest in partitions(xs[1:]):
            yield [[xs[0]]] + rest
            for i in range(len(rest)):
                yield rest[:i] + [[xs[0]] + rest[i]] + rest[i + 1:]
    top = 0
    for part in partitions(list(rows)):
        got = 0
        for g in part:
            n = len(list(itertools.takewhile(lambda c: len(set(c)) == 1, zip(*[rows[s] for s in g]))))
            got += (len(g) - 1) * n
        top = max(top, got)
    return top


def test_shared_prefixes_are_the_rows_first_pages_and_spare_the_most():
    rng = random.Random(3)
    for trial in range(60):
        ids = itertools.count()
        rows = {}
        for s in range(rng.randint(1, 6)):  # a random tree of forks
            base = list(rows[rng.choice(list(rows))]) if rows and rng.random() < 0.8 else []
            base = base[:rng.randint(0, len(base))]
            rows[s] = base + [next(ids) for _ in range(rng.randint(1, 5))]
        row_prefix, prefixes = shared_prefixes(rows)
        for s, p in row_prefix.items():
            assert prefixes[p] and rows[s][:len(prefixes[p])] == prefixes[p]
        assert all(list(row_prefix.values()).count(p) >= 2 for p in range(len(prefixes)))
        assert _saved(row_prefix, prefixes) == _best(rows)


def test_shared_prefixes_of_nothing():
    assert shared_prefixes({}) == ({}, [])
    assert shared_prefixes({3: [1, 2]}) == ({}, [])
    assert shared_prefixes({0: [1, 2], 1: [3]}) == ({}, [])
    assert shared_prefixes({0: [1, 2], 1: [1, 2], 4: [1]}) in [({0: 0, 1: 0}, [[1, 2]]), ({0: 0, 1: 0, 4: 0}, [[1]])]


@pytest.mark.parametrize("n_prefix,own,shared", [(40, [5, 9], 32), (32, [5, 1], 32), (32, [0, 7], 16), (15, [3, 3], 0),
                                                 (48, [0], 32), (1, [20], 0)])
def test_submit_with_a_prefix(n_prefix, own, shared):
    """Whole pages are shared, and every request keeps at least one token to feed."""
    pool = PagePool(50, seed=0)
    s = BatchSlots(4, pool, verbose=False)
    prefix = torch.arange(100, 100 + n_prefix)
    s.submit([torch.arange(n) for n in own], 200, [], prefix)
    for r, n in zip(s.requests, own):
        assert r.prompt.tolist() == prefix.tolist() + list(range(n))
        assert (0 if r.prefix is None else len(r.prefix.tokens)) == shared
    if not shared:
        return
    px = s.requests[0].prefix
    assert all(r.prefix is px for r in s.requests) and px.tokens.tolist() == prefix[:shared].tolist()
    px.reserve()
    for _, r in s.fill_free_slots():
        r.admit()
        assert r.pages[:-1] == px.pages and r.kv_len() == shared and r.next_input().tolist() == r.prompt[shared:].tolist()
        r.reserve(len(r.next_input()))
        assert r.kv_len() == len(r.prompt)
    for i, r in enumerate(s.requests):
        assert px.pages
        r.record(7)
        r.finish()
    assert pool.available == 50 and px.pages == [] and px.users == 0


def test_a_lone_request_with_a_prefix_fits_a_pool_of_its_own_size():
    """A slot's pages are enough for a request however its prompt is split: the prefix holds whole pages only."""
    for n in (33, 47, 48, 63):
        pool = PagePool(63 // 16 + 1, seed=0)
        s = BatchSlots(1, pool, verbose=False)
        s.submit([torch.arange(63 - n + 0)], 64, [], torch.arange(n))
        (_, r), = s.fill_free_slots()
        if r.prefix is not None:
            r.prefix.reserve()
        r.admit()
        r.reserve(len(r.next_input()))
        assert r.kv_len() == 63


def test_fork_shares_full_pages_and_keeps_the_rest():
    pool = PagePool(60, seed=2)
    r = ServingRequest(0, torch.arange(37), 100, [], pool)
    r.admit()
    r.reserve(37)
    r.record(70)
    r.reserve(1)  # 38 cached
    r.record(71)
    c = r.fork(1, torch.tensor([5, 6]), 90, [9])
    assert c.pages[:-1] == r.pages[:-1] and c.pages[-1] not in r.pages and c.fill == r.fill == 6
    assert c.prompt.tolist() == list(range(37)) + [70, 71, 5, 6]
    assert c.next_input().tolist() == [71, 5, 6] and c.kv_len() == 38
    c.reserve(3)
    assert c.kv_len() == 41 and r.kv_len() == 38
    g = c.fork  # a fork of a fork holds the first pages too
    c.record(80)
    d = g(2, torch.tensor([1]), 90, [])
    assert d.pages[:2] == r.pages[:2] and pool._held[r.pages[0]] == 3
    for x in (r, c, d):
        x.finish()
    assert pool.available == 60


def test_place_needs_a_free_slot():
    pool = PagePool(20, seed=0)
    s = BatchSlots(1, pool, verbose=False)
    s.submit([torch.arange(3)], 20, [])
    (_, r), = s.fill_free_slots()
    r.admit()
    assert s.free_slot() is None
    with pytest.raises(RuntimeError, match="no free slot"):
        s.place(r)
