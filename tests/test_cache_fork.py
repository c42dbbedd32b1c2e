"""Requests that share pages, in the cache manager's bookkeeping (no GPU): forks, pages of one's own before a write, tokens forgotten."""
import random

import pytest

from celeg_amd.cache import CacheManager, PageError, cache_layout


def manager(n_pages=12, window=None, max_requests=4):
    groups = [(2, 8, None, 2)] + ([(1, 8, window, 1)] if window else [])
    return CacheManager(cache_layout(kv_groups=groups, kv_of_step={0: (0, 0, True), 1: (0, 1, True)}), page_tokens=16,
                        n_pages=[n_pages] * len(groups), max_requests=max_requests, max_context=256)


def test_a_fork_shares_pages_until_one_of_the_two_writes():
    m = manager()
    a = m.open()
    assert m.prepare(a, 0, 40)
    before = m.pages_held(a)[0]
    m.drain_table_updates()
    b = m.fork(a, 40)
    assert m.pages_held(b) == m.pages_held(a) and m.free_pages() == [9]
    assert m.drain_table_updates() == [[(b, i, p) for i, p in enumerate(before)]]
    m.check()
    # the page that both go on writing is no longer good for a step; the first to prepare gets a copy
    assert not m.covers(a, 40, 1) and not m.covers(b, 40, 1) and m.pages_needed(a, 40, 1) == [1]
    assert m.prepare(b, 40, 1)
    mine = m.pages_held(b)[0]
    assert mine[:2] == before[:2] and mine[2] not in before and m.free_pages() == [8]
    assert m.covers(a, 40, 1) and m.covers(b, 40, 1) and m.pages_needed(a, 40, 1) == [0]
    assert m.drain_table_updates() == [[(b, 2, mine[2])]]
    # going back into a shared page: a page of its own for that one too
    assert not m.covers(a, 20, 3) and m.prepare(a, 20, 3) and m.pages_held(a)[0][1] not in before
    assert m.covers(b, 16, 25)
    m.check()
    m.close(a)
    m.check()
    assert m.free_pages() == [9] and m.pages_held(b)[0] == mine
    m.close(b)
    assert m.free_pages() == [12]


def test_a_fork_of_part_and_of_nothing():
    m = manager()
    a = m.open()
    assert m.prepare(a, 0, 100)
    b, c = m.fork(a, 17), m.fork(a, 0)
    assert m.pages_held(b)[0] == m.pages_held(a)[0][:2] and m.pages_held(c) == [[]]
    assert m.covers(a, 32, 68) and not m.covers(a, 31, 1)
    with pytest.raises(PageError):
        m.fork(a, 101)
    with pytest.raises(PageError):
        m.fork(a, -1)
    with pytest.raises(PageError):
        m.fork(3, 0)
    d = m.fork(b, 17)
    assert m.fork(a, 10) is None            # every slot is taken, and nothing is held for the fifth
    for s in (b, a, d, c):
        m.check()
        m.close(s)
    m.check()
    assert m.free_pages() == [12]


def test_too_few_pages_for_a_copy():
    m = manager(n_pages=3)
    a = m.open()
    assert m.prepare(a, 0, 40)
    b = m.fork(a, 40)
    assert not m.prepare(b, 40, 1) and m.pages_held(a) == m.pages_held(b)      # nothing was taken
    m.close(a)
    assert m.prepare(b, 40, 1) and m.covers(b, 40, 1)                          # nobody shares it any more
    m.check()


def test_forgetting_tokens_gives_pages_back():
    m = manager()
    a = m.open()
    assert m.prepare(a, 0, 100) and m.free_pages() == [5]
    m.truncate(a, 33)
    assert m.free_pages() == [9] and m.covers(a, 33, 15) and not m.covers(a, 33, 16) and m.table(0, a, 3) == -1
    m.check()
    for bad in (34, -1):
        with pytest.raises(PageError):
            m.truncate(a, bad)
    m.truncate(a, 0)
    assert m.free_pages() == [12] and m.holds(a, 0, 0) and not m.holds(a, 0, 1) and not m.holds(2, 0, 0)


def test_forks_in_a_window_group():
    m = manager(window=20)
    a = m.open()
    pos = 0
    for n in (30, 30, 30):
        assert m.prepare(a, pos, n)
        pos += n
    b = m.fork(a, 90)
    assert m.pages_held(b) == m.pages_held(a)
    assert not m.holds(b, 0, 1) and m.holds(b, 80, 10)
    for s in (a, b):
        assert m.prepare(s, 90, 30) and m.covers(s, 90, 30)
        m.check()
    m.close(a)
    m.check()
    m.truncate(b, 95)
    assert m.prepare(b, 95, 2) and m.covers(b, 95, 2)
    m.close(b)
    m.check()
    assert m.free_pages() == [12, 12]


@pytest.mark.parametrize("seed", range(4))
def test_random_calls_lose_no_page(seed):
    rng = random.Random(seed)
    m = manager(n_pages=20, window=24 if seed % 2 else None, max_requests=5)
    length = {}
    for _ in range(400):
        slots = sorted(length)
        what = rng.choice(["open", "close", "fork", "fork", "prepare", "prepare", "prepare", "truncate"])
        if what == "open":
            s = m.open()
            if s is not None:
                length[s] = 0
        elif slots:
            s = rng.choice(slots)
            if what == "close":
                m.close(s)
                del length[s]
            elif what == "fork":
                other = m.fork(s, length[s])
                if other is not None:
                    length[other] = length[s]
            elif what == "prepare":
                n = rng.randint(1, 40)
                if length[s] + n <= 256 and m.prepare(s, length[s], n):
                    assert m.covers(s, length[s], n)
                    length[s] += n
            elif not seed % 2:
                length[s] = rng.randint(0, length[s])
                m.truncate(s, length[s])
        m.check()
    for s in list(length):
        m.close(s)
    m.check()
    assert m.free_pages()[0] == 20
