"""Shared pages and positions of which there are none (the cache manager's bookkeeping, no GPU)."""
from test_cache_fork import manager


def test_nothing_to_write_needs_no_page_of_ones_own():
    m = manager()
    a = m.open()
    assert m.prepare(a, 0, 40)
    b = m.fork(a, 40)
    for slot in (a, b):
        for start in (0, 5, 16, 21, 39, 40):
            assert m.pages_needed(slot, start, 0) == [0], start
            assert m.covers(slot, start, 0), start
    assert m.pages_needed(b, 21, 1) == [1] and not m.covers(b, 21, 1)
