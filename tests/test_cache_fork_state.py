"""Requests of models that keep state beside keys and values fork only where that state stands (the cache manager's bookkeeping, no GPU)."""
import pytest

from celeg_amd.cache import CacheManager, PageError, cache_layout


def manager(**more):
    layout = cache_layout(kv_groups=[(2, 8, None, 1)], kv_of_step={0: (0, 0, True)}, states=[(1, "saved", (3, 8), "float32")])
    return CacheManager(layout, page_tokens=16, n_pages=[12], max_requests=3, max_context=256, **more)


def test_a_request_with_state_forks_where_it_stands():
    m = manager()
    a = m.open()
    assert m.prepare(a, 0, 40)
    held, free = m.pages_held(a), m.free_pages()
    for length in (40, 1):                                # nothing has been stepped yet
        with pytest.raises(PageError, match="state"):
            m.fork(a, length)
    m.stepped(a, 37)
    for length in (0, 16, 36, 38, 40):
        with pytest.raises(PageError, match="behind 37 tokens"):
            m.fork(a, length)
    assert m.pages_held(a) == held and m.free_pages() == free and m.n_free_slots == 2
    m.check()
    b = m.fork(a, 37)
    c = m.fork(b, 37)                                     # (the fork stands where its origin stood)
    with pytest.raises(PageError, match="behind 37 tokens"):
        m.fork(b, 20)
    m.check()
    for s in (a, b, c):
        m.close(s)
    m.check()
    a = m.open()                                          # a slot used again starts anew
    assert m.prepare(a, 0, 40)
    with pytest.raises(PageError, match="behind 0 tokens"):
        m.fork(a, 37)
    assert m.fork(a, 0) is not None


def test_slots_that_do_not_exist():
    m = manager()
    for slot in (-1, 3):
        with pytest.raises(PageError):
            m.stepped(slot, 1)
