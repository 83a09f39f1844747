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


class Stopped(RuntimeError):
    pass


def host_only(monkeypatch, eng, kept, fails=None):
    """The device's part of verify by stand-ins: every sequence keeps kept[slot] tokens of its tree, or `fails` raises Stopped."""
    import torch
    from lumenllm_b200.engine import engine as module

    def context(cache, runtime, drafts):
        cache.reserve_all([(d.slot, len(d.tokens)) for d in drafts])
        eng.slots_now = [d.slot for d in drafts]
        return type("C", (), dict(tokens=None, cu_q=None, seq_start=None, block_tables=[None] * len(cache.groups)))(), None

    def stage(name, result):
        def f(*a, **kw):
            if fails == name:
                raise Stopped(name)
            return result()
        return f

    accepted = lambda: tuple(torch.tensor(x) for x in
                             ([kept[s] for s in eng.slots_now], [[0] * 9] * len(eng.slots_now), [[7] * 9] * len(eng.slots_now)))
    monkeypatch.setattr(module, "tree_context", context)
    monkeypatch.setattr(module.K, "argmax", lambda logits: None)
    monkeypatch.setattr(module.K, "tree_accept", stage("accept", accepted))
    monkeypatch.setattr(module.K, "cache_compact", stage("compact", lambda: None))
    monkeypatch.setattr(eng, "check_kernels", stage("check", lambda: None), raising=False)
    eng.model.forward = stage("forward", lambda: None)


@pytest.mark.parametrize("window", [0, 40, 100])
def test_pages_of_rejected_drafts_are_given_back(monkeypatch, window):
    """After a step of drafts the cache is as after ordinary steps of the kept tokens: a page less than a page's tokens of room."""
    needs = {0: CacheNeed(1, 16, window), 1: CacheNeed(1, 16)}
    c, alike = (filled([10, 60, 63], pages=24, needs=needs) for _ in range(2))
    eng = drafting(c)
    kept = {0: 1, 1: 5, 2: 1}
    host_only(monkeypatch, eng, kept)
    assert eng.verify([star(s, 200) for s in range(3)]) == [[7], [7] * 5, [7]]
    for s, n in kept.items():
        alike.reserve(s, n)
        alike.commit(s, n)
    assert c.lengths.tolist() == alike.lengths.tolist() == [11, 65, 64, 0, 0]
    books(c)
    for g, h in zip(c.groups, alike.groups):
        assert (g.n_held == h.n_held).all() and (g.end_page == h.end_page).all() and (g.first_page == h.first_page).all()
        assert ((g.table != 0) == (h.table != 0)).all() and g.pool.free_count == h.pool.free_count
        assert g._changed >= {0, 1, 2}                   # the rows on the device are out of date
    # a prompt that fits beside the tokens themselves fits
    s = c.alloc_slot()
    c.reserve(s, (24 - 4) * PAGE)


def test_room_that_a_slot_had_before_stays_its_own(monkeypatch):
    c = filled([10], pages=8)
    c.reserve(0, 3 * PAGE)
    eng = drafting(c)
    host_only(monkeypatch, eng, {0: 2})
    eng.verify([star(0, 250)])
    assert c.length(0) == 12 and c.groups[0].end_page[0] == 4
    books(c)


@pytest.mark.parametrize("stage", ["forward", "accept", "compact", "check"])
def test_a_step_of_drafts_that_fails_leaves_the_sequences_as_they_were(monkeypatch, stage):
    c = filled([10, 60, 64], pages=12, needs={0: CacheNeed(1, 16, 30), 1: CacheNeed(1, 16)})
    eng, before = drafting(c), books(c)
    host_only(monkeypatch, eng, {0: 1, 1: 1, 2: 1}, fails=stage)
    with pytest.raises(Stopped, match=stage):
        eng.verify([star(s, 150) for s in range(3)])
    assert same(before, books(c)) and c.lengths.tolist() == [10, 60, 64, 0, 0]
