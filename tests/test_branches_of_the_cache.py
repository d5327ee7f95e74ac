"""Forked sequences, moved pages, and streams that keep their first positions: the cache's books on the host, and no GPU."""
import random

import pytest
import torch

from palm_infra_amd.cache import CacheFull, CacheMisuse, KVNeed, ModelCache, PageTable, RowsNeed, StateNeed


def make(needs=None, max_tokens=64 * 12, max_seqs=8, **more):
    needs = needs or [[KVNeed(2, 8), StateNeed("s", (3,))], [KVNeed(2, 8)], [RowsNeed("r", (5,))]]
    return ModelCache(needs, [None] * len(needs), max_tokens, max_seqs, 4096, torch.float32, "cpu", **more)


def grow(c, slot, n):
    c.reserve([(slot, n)])
    c.commit([(slot, n)])


def fill(c):
    g = torch.Generator().manual_seed(1)
    for group in c.groups:
        for t in [group.k, group.v] if hasattr(group, "k") else [group.data]:
            t.copy_(torch.randn(t.shape, generator=g))


def rows_of(c, slot):
    """What the cache holds of a sequence, position by position, in every layer and storage."""
    n, out = c.lengths[slot], []
    for g in c.groups:
        if g.table is None:
            out.append(g.data[:, slot].clone())
            continue
        pages = [g.table.slot_pages[slot][p // 64] for p in range(n)]
        assert [int(x) for x in g.table_dev[slot, :(n + 63) // 64]] == g.table.slot_pages[slot][:(n + 63) // 64]
        if hasattr(g, "k"):
            out += [torch.stack([g.k[:, pages[p], :, p % 64] for p in range(n)]), torch.stack([g.v[:, pages[p], :, :, p % 64] for p in range(n)])]
        else:
            out.append(torch.stack([g.data[:, pages[p], p % 64] for p in range(n)]))
    return out


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("length", [1, 63, 64, 65, 130, 192])
def test_branches_share_full_pages_and_have_the_rest_for_themselves(length):
    c = make()
    a = c.open()
    grow(c, a, length)
    fill(c)
    before = rows_of(c, a)
    free = [g.table.pages.free_count for g in c.paged_groups]
    b, d = c.fork(a, 2)
    c.check()
    assert c.lengths[b] == c.lengths[d] == length and len({a, b, d}) == 3
    assert [f - g.table.pages.free_count for f, g in zip(free, c.paged_groups)] == [2 * (length % 64 != 0)] * len(free)
    assert same(rows_of(c, a), before) and same(rows_of(c, b), before) and same(rows_of(c, d), before)
    # each goes on by itself: what one writes behind the fork the others do not see
    for g in c.paged_groups:
        mine, its = g.table.slot_pages[a], g.table.slot_pages[b]
        assert mine[:length // 64] == its[:length // 64]
        assert length % 64 == 0 or mine[-1] != its[-1]
    for s in (a, b):
        grow(c, s, 1)
    c.check()
    for g in c.paged_groups:
        assert g.table.slot_pages[a][length // 64] != g.table.slot_pages[b][length // 64]
    c.close(a)
    c.check()
    for g in c.paged_groups:                             # the branches' pages are still theirs
        assert all(g.table.pages.is_held(p) for s in (b, d) for p in g.table.slot_pages[s])
    c.close(b)
    c.close(d)
    c.check()
    assert all(g.table.pages.free_count == g.n_pages for g in c.paged_groups)


def test_a_fork_that_does_not_fit_takes_nothing():
    c = make(max_tokens=64 * 4, max_seqs=6)
    a = c.open()
    grow(c, a, 64 * 2 + 1)
    with pytest.raises(CacheFull, match="2 more pages"):
        c.fork(a, 2)
    c.check()
    assert c.slots.held_count == 1 and c.paged_groups[0].table.pages.free_count == 1
    with pytest.raises(CacheFull, match="6 branches"):
        c.fork(a, 6)
    with pytest.raises(CacheMisuse, match="not open"):
        c.fork(5)
    with pytest.raises(CacheMisuse, match="0 branches"):
        c.fork(a, 0)
    b, = c.fork(a)
    c.check()
    with pytest.raises(CacheFull):
        c.fork(b)
    c.close(b)
    c.check()


def test_a_branch_of_an_empty_sequence_and_of_a_branch():
    c = make()
    a = c.open()
    b, = c.fork(a)
    grow(c, b, 70)
    fill(c)
    d, = c.fork(b)
    e, = c.fork(d)
    c.check()
    assert c.lengths[a] == 0 and same(rows_of(c, d), rows_of(c, b)) and same(rows_of(c, e), rows_of(c, b))
    for s in (b, d, a, e):
        c.close(s)
        c.check()


def test_a_page_listed_more_often_than_counted_is_found():
    c = make()
    a = c.open()
    grow(c, a, 64)
    b, = c.fork(a)
    t = c.paged_groups[0].table
    t.users[t.slot_pages[a][0]] = 1
    with pytest.raises(CacheMisuse, match="in 2 slots and counted for 1"):
        c.check()
    t.users[t.slot_pages[a][0]] = 2
    t.slot_pages[b] = t.slot_pages[b] * 2
    with pytest.raises(CacheMisuse, match="twice"):
        c.check()


def test_moved_pages_are_the_lowest_and_hold_what_they_held():
    c = make(max_tokens=64 * 20, max_seqs=10)
    slots = [c.open() for _ in range(6)]
    for i, s in enumerate(slots):
        grow(c, s, 40 + 50 * i)
    fill(c)
    branch, = c.fork(slots[5])
    for s in (slots[0], slots[2], slots[4]):
        c.close(s)
    left = [slots[1], slots[3], slots[5], branch]
    before = {s: rows_of(c, s) for s in left}
    held = [g.table.pages.held_count for g in c.paged_groups]
    moved = c.compact()
    c.check()
    assert moved > 0
    for g, n in zip(c.paged_groups, held):
        assert [g.table.pages.is_held(p) for p in range(g.n_pages)] == [p < n for p in range(g.n_pages)]
    assert all(same(rows_of(c, s), before[s]) for s in left)
    assert c.compact() == 0
    for s in left:
        grow(c, s, 30)
    c.check()


def test_random_traffic_of_branches_keeps_the_books():
    rng = random.Random(4)
    needs = [[KVNeed(1, 4)], [KVNeed(1, 4, 100)], [KVNeed(1, 4, 90, kept=70)], [RowsNeed("r", (2,), None, 64)], [StateNeed("s", (2,))]]
    c = ModelCache(needs, [None] * 5, 64 * 40, 12, 2000, torch.float32, "cpu")
    live, seen = [], 0
    for turn in range(600):
        what = rng.random()
        try:
            if what < 0.2 and c.slots.free_count:
                live.append(c.open())
            elif what < 0.35 and live:
                live += c.fork(rng.choice(live), rng.randint(1, 3))
                seen += 1
            elif what < 0.5 and live:
                c.close(live.pop(rng.randrange(len(live))))
            elif what < 0.55:
                c.compact()
            elif live:
                grow(c, rng.choice(live), rng.choice([1, 1, 5, 64, 130]))
        except CacheFull:
            pass
        c.check()
    assert seen > 20
    for s in live:
        c.close(s)
    c.check()
    assert all(g.table.pages.free_count == g.n_pages for g in c.paged_groups)


def test_first_positions_stay_while_the_window_moves_on():
    c = make([[KVNeed(1, 4, 100, kept=70)]], max_tokens=64 * 12, stream_tokens=64 * 60)
    assert c.max_seq_tokens == 64 * 60 and c.max_tokens == 64 * 12
    s = c.open()
    t = c.paged_groups[0].table
    for n in range(1, 64 * 30):
        grow(c, s, 1)
        first = max(0, n - 99) // 64                     # the page of the oldest position that the next query sees
        assert [p >= 0 for p in t.slot_pages[s]] == [j < 2 or j >= first for j in range((n + 63) // 64)]
        assert t.pages.held_count <= 5
    c.check()
    b, = c.fork(s)
    grow(c, b, 200)
    c.check()
    c.close(s)
    c.close(b)
    c.check()
    assert t.pages.free_count == t.pages.n
    d = c.open()                                         # the slot's next sequence starts over
    grow(c, d, 300)
    assert [p >= 0 for p in t.slot_pages[d]] == [True, True, False, True, True]


def test_refusals():
    with pytest.raises(ValueError, match="stay behind a sliding window"):
        PageTable(4, 2, 4, None, False, 3)
    with pytest.raises(ValueError, match="stay behind a sliding window"):
        PageTable(4, 2, 4, 64, True, 3)
    with pytest.raises(ValueError, match="stay behind a sliding window"):
        PageTable(4, 2, 4, 64, False, -1)
    with pytest.raises(ValueError, match="needs a window"):
        make(stream_tokens=10000)
    with pytest.raises(ValueError, match="needs a window"):
        make([[KVNeed(1, 4, 100, kept=4)], [RowsNeed("r", (2,))]], stream_tokens=10000)
    assert make([[KVNeed(1, 4, 100, kept=4)], [StateNeed("s", (2,))]], stream_tokens=10000).max_seq_tokens == 4096      # (the model's own limit)

    class Odd:
        def make_group(self, *a):
            return type("G", (), {"need": self, "table": None, "sync": lambda s: None, "on_open": lambda s, slot: None, "attach": lambda s, lc, e: None,
                                  "nbytes": lambda s: 0})()
    c = ModelCache([[Odd()]], [None], 128, 4, 128, torch.float32, "cpu")
    a = c.open()
    with pytest.raises(CacheMisuse, match="cannot be forked"):
        c.fork(a)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("length", [64, 70])
def test_a_fork_whose_copy_fails_keeps_nothing(which, length):
    """Whichever storage it is that fails: pages in order, states, rows or a windowed group's pages."""
    c = make([[KVNeed(2, 8), StateNeed("s", (3,))], [RowsNeed("r", (5,))], [KVNeed(2, 8, 60, kept=3)]])
    a = c.open()
    grow(c, a, length)
    fill(c)
    before = rows_of_held(c, a)
    free, group = [g.table.pages.free_count for g in c.paged_groups], c.groups[which]

    def fails(src, dst, tokens=None):
        raise RuntimeError("no copy")
    group.copy = fails
    if group.table is None or length % 64:
        with pytest.raises(RuntimeError, match="no copy"):
            c.fork(a, 2)
        c.check()
        assert c.slots.held_count == 1 and [g.table.pages.free_count for g in c.paged_groups] == free
    del group.copy
    b, d = c.fork(a, 2)
    c.check()
    assert all(same(rows_of_held(c, s), before) for s in (a, b, d)) and c.lengths[b] == c.lengths[d] == length
    for s in (a, b, d):
        c.close(s)
    c.check()
    assert all(g.table.pages.free_count == g.n_pages for g in c.paged_groups)


def rows_of_held(c, slot):
    """``rows_of`` of the groups that keep every position; of the windowed one the positions that it still has."""
    n, out = c.lengths[slot], []
    for g in c.groups:
        if g.table is None:
            out.append(g.data[:, slot].clone())
            continue
        for p in range(n):
            page = g.table.slot_pages[slot][p // 64]
            if page >= 0:
                out += [g.k[:, page, :, p % 64].clone(), g.v[:, page, :, :, p % 64].clone()] if hasattr(g, "k") else [g.data[:, page, p % 64].clone()]
    return out


@pytest.mark.parametrize("which", range(2))
def test_pages_whose_copy_fails_stay_where_they_are(which):
    c = make([[KVNeed(2, 8)], [RowsNeed("r", (5,))]], max_tokens=64 * 20, max_seqs=10)
    slots = [c.open() for _ in range(4)]
    for i, s in enumerate(slots):
        grow(c, s, 60 + 50 * i)
    fill(c)
    left = [slots[1], slots[3]] + c.fork(slots[3])
    for s in (slots[0], slots[2]):
        c.close(s)
    before = {s: rows_of(c, s) for s in left}
    group = c.paged_groups[which]

    def fails(src, dst, tokens=None):
        raise RuntimeError("no copy")
    group.copy = fails
    with pytest.raises(RuntimeError, match="no copy"):
        c.compact()
    c.check()
    assert all(same(rows_of(c, s), before[s]) for s in left)
    del group.copy
    assert c.compact() > 0
    c.check()
    assert all(same(rows_of(c, s), before[s]) for s in left) and c.compact() == 0
