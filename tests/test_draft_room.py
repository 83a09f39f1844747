"""What steps leave of the cache's room where it runs out, and what steps of drafts leave behind the tokens that they keep
(bookkeeping on the host, without a device)."""
import numpy as np
import pytest

from lumenllm_b200 import DraftEntry, Engine, StepEntry, StepError
from lumenllm_b200.cache import CacheFull, CacheNeed, KVCache
from lumenllm_b200.engine.context import pack_step

PAGE = 64


def books(cache):
    """Everything that the groups say of their pages."""
    cache.check()
    return [(g.table.copy(), g.end_page.copy(), g.first_page.copy(), g.n_held.copy(), list(g.pool._free)) for g in cache.groups]


def same(a, b):
    return all(np.array_equal(x, y) for ga, gb in zip(a, b) for x, y in zip(ga, gb))


def filled(lengths, pages=10, needs=None, slots=5):
    """A cache with one live slot a length, as ordinary steps leave it."""
    c = KVCache(needs or {0: CacheNeed(1, 16)}, pages * PAGE, slots, max_positions=pages * PAGE)
    for n in lengths:
        s = c.alloc_slot()
        c.reserve(s, n)
        c.commit(s, n)
    return c


def drafting(cache):
    """An Engine's bookkeeping around a cache, without a device."""
    e = Engine.__new__(Engine)
    e.cache, e.model = cache, type("M", (), {"tree_safe": True})()
    e.runtime, e.steps_run = None, 0
    e.vocab_size, e.max_seq_len, e.max_step_tokens = 100, 640, 640
    return e


def star(slot, nodes):
    return DraftEntry(slot, [1] * nodes, [-1] + [0] * (nodes - 1))


@pytest.mark.parametrize("window", [0, 100])
def test_a_refused_step_of_drafts_leaves_the_pages_as_they_were(window):
    """Four of ten pages are free; the first tree takes three of them, the second is refused: plain steps of the others still fit."""
    c = filled([130, 60, 64, 64], needs={0: CacheNeed(1, 16, window), 1: CacheNeed(1, 16)})
    eng, before, free = drafting(c), books(c), c.free_tokens()
    with pytest.raises(StepError, match="slot 1.*full"):
        eng.verify([star(0, 200), star(1, 200)])
    assert same(before, books(c)) and c.free_tokens() == free == 4 * PAGE
    assert [c.reserve(s, 1) for s in (2, 3)] == [64, 64]


def test_a_refused_ordinary_step_leaves_the_pages_as_they_were():
    c = filled([100, 10, 5], pages=6)
    before = books(c)
    with pytest.raises(CacheFull, match="slot 2"):
        pack_step(c, [StepEntry(0, [1] * 60, []), StepEntry(1, [1] * 100, []), StepEntry(2, [1] * 150, [])])
    assert same(before, books(c))


def test_a_reservation_that_one_group_refuses_is_none():
    """The first group has room where the second has not: the slot keeps what it had in both."""
    c = filled([64, 64], pages=4, needs={0: CacheNeed(1, 16, 16), 1: CacheNeed(1, 16)})
    s = c.alloc_slot()
    c.groups[1].pool.take(1)                       # one page fewer than the other group
    before = [(g.table.copy(), g.pool.free_count) for g in c.groups]
    for ask in (lambda: c.reserve(s, 128), lambda: c.reserve_all([(0, 1), (s, 128)]), lambda: c.reserve_all([(0, 1), (1, 1)])):
        with pytest.raises(CacheFull):
            ask()
        assert all(np.array_equal(t, g.table) and n == g.pool.free_count for (t, n), g in zip(before, c.groups))
    assert c.groups[0].pool.free_count == 2 and c.groups[1].pool.free_count == 1
