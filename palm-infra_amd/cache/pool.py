"""Bookkeeping of the cache, on the host: which pages are free, which slot holds which pages.

Keys and values are kept in pages of ``PAGE_TOKENS`` positions.  A sequence has a slot; the slot has a
list of pages, as many as its length needs.  When a sequence ends its pages and its slot go back and
are handed out again without being cleared: nothing reads a page beyond its slot's length.

A full page is never written again, so sequences that begin alike may share it (a sequence and its branches): a page
goes back when the last slot that lists it lets go of it.
"""
from __future__ import annotations

PAGE_TOKENS = 64


class CacheFull(RuntimeError):
    """No page (or no slot) is free for what a step needs."""


class CacheMisuse(RuntimeError):
    """A slot or page was freed twice, or used without being held."""


def pages_for(tokens: int) -> int:
    return (tokens + PAGE_TOKENS - 1) // PAGE_TOKENS


class FreeList:
    """Integers 0..n-1, each either free or held.  Lowest free number first, so that what was given
    back is used again soon (and tests can say which one)."""

    def __init__(self, n: int, what: str):
        self.n, self.what = int(n), what
        self._free = list(range(self.n - 1, -1, -1))  # pop() gives the lowest
        self._held = [False] * self.n

    @property
    def free_count(self) -> int:
        return len(self._free)

    @property
    def held_count(self) -> int:
        return self.n - len(self._free)

    def is_held(self, i: int) -> bool:
        return 0 <= i < self.n and self._held[i]

    def take(self) -> int:
        if not self._free:
            raise CacheFull(f"no free {self.what}: all {self.n} are held")
        i = self._free.pop()
        self._held[i] = True
        return i

    def take_many(self, k: int) -> list[int]:
        if k > len(self._free):
            raise CacheFull(f"{k} {self.what}s needed, {len(self._free)} of {self.n} free")
        return [self.take() for _ in range(k)]

    def give_back(self, i: int) -> None:
        if not 0 <= i < self.n:
            raise CacheMisuse(f"{self.what} {i} does not exist (there are {self.n})")
        if not self._held[i]:
            raise CacheMisuse(f"{self.what} {i} is given back but not held")
        self._held[i] = False
        self._free.append(i)
        # keep "lowest first": the list is small next to the work of a step
        self._free.sort(reverse=True)

    def exchange(self, moves) -> None:
        """For each (held, free): the one is given back and the other taken in its place."""
        for held, free in moves:
            if not self.is_held(held) or not 0 <= free < self.n or self._held[free]:
                raise CacheMisuse(f"{self.what} {held} cannot be exchanged for {free}")
            self._held[held], self._held[free] = False, True
        self._free = [i for i in range(self.n - 1, -1, -1) if not self._held[i]]

    def check(self) -> None:
        """Every number is either free once or held; none lost, none twice."""
        free = sorted(self._free)
        if len(set(free)) != len(free):
            raise CacheMisuse(f"a {self.what} is free twice")
        for i in range(self.n):
            if self._held[i] == (i in set(free)):
                raise CacheMisuse(f"{self.what} {i} is {'both held and free' if self._held[i] else 'lost'}")


class PageTable:
    """The pages of every slot for one group of layers.

    ``window``: if set, only the last ``window`` positions before a query are ever read, so pages
    that lie wholly below ``length - window`` are given back as the sequence grows (their entries in
    the slot's list become -1).  ``chunked``: a query only ever reads positions of its own chunk of ``window``
    positions, so what lies wholly below the next query's chunk is given back.  ``kept``: the sequence's first so many
    positions are read by every query beside its window, and their pages stay."""

    def __init__(self, n_pages: int, n_slots: int, max_pages_per_slot: int, window: int | None = None, chunked: bool = False, kept: int = 0):
        self.pages = FreeList(n_pages, "page")
        self.n_slots, self.max_pages_per_slot, self.window = n_slots, max_pages_per_slot, window
        if chunked and not window:
            raise ValueError("storage by chunks needs their size")
        if kept < 0 or (kept and (chunked or not window)):
            raise ValueError(f"first positions that stay ({kept}) stay behind a sliding window")
        self.chunked, self.kept = bool(chunked), int(kept)
        self.users = [0] * n_pages                              # slots that list the page
        self._trimmed = [pages_for(self.kept)] * n_slots        # pages of a slot below this one were looked at already
        self.slot_pages: list[list[int]] = [[] for _ in range(n_slots)]
        self.dirty: dict[int, tuple[int, int]] = {}   # slots whose device copy of the list is stale, and the places [from, to) of it that are

    def pages_needed(self, slot: int, new_length: int) -> int:
        return max(0, pages_for(new_length) - len(self.slot_pages[slot]))

    def grow(self, slot: int, new_length: int) -> None:
        """Make room for positions [0, new_length)."""
        need = pages_for(new_length)
        if need > self.max_pages_per_slot:
            raise CacheFull(f"a sequence of {new_length} tokens needs {need} pages; a slot holds at most "
                            f"{self.max_pages_per_slot}")
        have = self.slot_pages[slot]
        if need > len(have):
            new = self.pages.take_many(need - len(have))
            for p in new:
                self.users[p] = 1
            have.extend(new)
            self._changed(slot, need - len(new), need)

    def _changed(self, slot: int, begin: int, end: int) -> None:
        if begin < end:
            was = self.dirty.get(slot, (begin, end))
            self.dirty[slot] = min(was[0], begin), max(was[1], end)

    def _let_go(self, page: int) -> None:
        self.users[page] -= 1
        if self.users[page] == 0:
            self.pages.give_back(page)

    def trim(self, slot: int, length: int) -> None:
        """After a step: give back pages no later query can read (windowed groups only)."""
        if self.window is None:
            return
        # the next query sits at position `length`
        first_needed = length - length % self.window if self.chunked else max(0, length - self.window + 1)
        have = self.slot_pages[slot]
        end = min(first_needed // PAGE_TOKENS, len(have))
        for j in range(self._trimmed[slot], end):
            if have[j] >= 0:
                self._let_go(have[j])
                have[j] = -1
                self._changed(slot, j, j + 1)
        self._trimmed[slot] = max(self._trimmed[slot], end)

    def release(self, slot: int) -> None:
        for p in self.slot_pages[slot]:
            if p >= 0:
                self._let_go(p)
        self._changed(slot, 0, len(self.slot_pages[slot]))
        self.slot_pages[slot] = []
        self._trimmed[slot] = pages_for(self.kept)

    def fork_needs(self, slot: int, length: int) -> int:
        """Pages that a branch of the slot takes of its own: one, if its last page is not full."""
        last = length // PAGE_TOKENS
        return int(length % PAGE_TOKENS != 0 and last < len(self.slot_pages[slot]) and self.slot_pages[slot][last] >= 0)

    def fork(self, slot: int, new: int, length: int):
        """The empty slot ``new`` lists the pages of ``slot`` up to ``length``; the last one, if it is not full, a page of its own.
        Returns (page, its copy) then, which is to be made, else None."""
        pages, copy = self.slot_pages[slot][:pages_for(length)], None
        if self.fork_needs(slot, length):
            own = self.pages.take()
            copy, pages[-1] = (pages[-1], own), own
            self.users[own] = 0                                 # (counted below like the others)
        for p in pages:
            if p >= 0:
                self.users[p] += 1
        self.slot_pages[new] = pages
        self._trimmed[new] = self._trimmed[slot]
        self._changed(new, 0, len(pages))
        return copy

    def moves_to_compact(self) -> list[tuple[int, int]]:
        """By which the held pages become the pages numbered lowest, as few as it takes: (page, its new number) each.  The contents are to be
        moved before the books (``move``): no page is both read and written, and what is written nobody holds yet."""
        n = self.pages.held_count
        return list(zip([p for p in range(n, self.pages.n) if self.pages.is_held(p)], [p for p in range(n) if not self.pages.is_held(p)]))

    def move(self, moves) -> None:
        """For each (page, its new number): whoever lists the page lists the other one, which holds the same by now."""
        self.pages.exchange(moves)
        for old, new in moves:
            self.users[new], self.users[old] = self.users[old], 0
        where = dict(moves)
        for slot, pages in enumerate(self.slot_pages):
            for j, p in enumerate(pages):
                if p in where:
                    pages[j] = where[p]
                    self._changed(slot, j, j + 1)

    def check(self) -> None:
        self.pages.check()
        listed: dict[int, int] = {}
        for pages in self.slot_pages:
            own = [p for p in pages if p >= 0]
            if len(set(own)) != len(own):
                raise CacheMisuse("a slot lists a page twice")
            for p in own:
                listed[p] = listed.get(p, 0) + 1
        for p, n in listed.items():
            if self.users[p] != n:
                raise CacheMisuse(f"page {p} is in {n} slots and counted for {self.users[p]}")
        if len(listed) != self.pages.held_count or sum(self.users) != sum(listed.values()):
            raise CacheMisuse(f"{self.pages.held_count} pages are held but slots list {len(listed)}")
