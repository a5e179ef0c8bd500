"""Host-side accounting of cache pages and of fixed-size state slots.

A :class:`PagePool` owns the page ids of one cache group.  Pages are handed out LIFO, so
a page given back is the next one used again (no zeroing: lengths guard stale data).
Requests may *reserve* a number of pages at admission; a reserved page is not handed to
anyone else, so a request that was admitted with a full reservation can never run out
in the middle, which is the reference's no-deadlock rule in page units
(src/engine/kv.rs:36-67: ``reserve`` against ``free - sum(reserved)``, ``allocate`` from
the tail of the free list, ``release`` of everything at the end, src/engine/kv.rs:69-74).

A page may have several holders (continuations of one prompt hold its pages together): one owner has *drawn* it from the free
pages, others *share* it.  It goes back to the free pages when its last holder lets go, whoever drew it; a reservation counts
what its owner draws.

:class:`StateSlots` gives each live request one exclusive slot index, reusable after
release (src/engine/recurrent.rs:6-38).
"""

from __future__ import annotations

from typing import Dict, Hashable, List, Optional, Sequence, Set

import numpy as np


class OutOfPages(RuntimeError):
    """No page can be handed out without breaking another request's reservation."""


class PagePool:
    def __init__(self, num_pages: int, first_page: int = 0):
        if num_pages <= 0:
            raise ValueError("a page pool needs at least one page")
        self.num_pages = num_pages
        self.first_page = first_page
        # LIFO: the last element is handed out first; start so that low ids go first.
        self._free: List[int] = list(range(first_page + num_pages - 1, first_page - 1, -1))
        self._refs = np.zeros(num_pages, dtype=np.int32)    # holders of each page (from first_page on)
        self._ref = memoryview(self._refs)                  # the same a page at a time (a tenth of an array operation's time)
        self._quota: Dict[Hashable, int] = {}
        self._drawn: Dict[Hashable, Set[int]] = {}          # pages drawn by the owner (and not given back)
        self._borrowed: Dict[Hashable, Set[int]] = {}       # pages that it shares and others drew
        self._reserved_unallocated = 0

    # ---------------------------------------------------------------- queries
    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def used_pages(self) -> int:
        return self.num_pages - len(self._free)

    @property
    def available_to_reserve(self) -> int:
        return len(self._free) - self._reserved_unallocated

    def held_by(self, owner: Hashable) -> int:
        return len(self._drawn.get(owner, ())) + len(self._borrowed.get(owner, ()))

    def owner_of(self, page: int) -> Optional[Hashable]:
        holders = self.holders_of(page)
        return holders[0] if holders else None

    def holders_of(self, page: int) -> List[Hashable]:
        """Who holds the page: the one who drew it, if it has not ended, then those who share it."""
        return ([owner for owner, pages in self._drawn.items() if page in pages]
                + [owner for owner, pages in self._borrowed.items() if page in pages])

    # ---------------------------------------------------------------- reservations
    def reserve(self, owner: Hashable, pages: int) -> bool:
        """Set aside ``pages`` pages for ``owner`` (its peak simultaneous need)."""
        if owner in self._quota:
            return False
        if pages > self.available_to_reserve:
            return False
        self._enter(owner, pages)
        self._reserved_unallocated += pages
        return True

    def register(self, owner: Hashable) -> None:
        """Admit ``owner`` without a reservation: its pages come on demand."""
        if owner in self._quota:
            raise ValueError(f"{owner!r} is already registered in this pool")
        self._enter(owner, 0)

    def _enter(self, owner: Hashable, quota: int) -> None:
        self._quota[owner] = quota
        self._drawn[owner] = set()
        self._borrowed[owner] = set()

    # ---------------------------------------------------------------- pages
    def allocate(self, owner: Hashable) -> int:
        if owner not in self._quota:
            raise KeyError(f"{owner!r} is not registered in this pool")
        drawn = self._drawn[owner]
        if len(drawn) < self._quota[owner]:
            self._reserved_unallocated -= 1   # drawing on the owner's own reservation
        elif self.available_to_reserve <= 0:
            raise OutOfPages(f"cache pool exhausted: {self.num_pages} pages, {len(self._free)} free, "
                             f"{self._reserved_unallocated} reserved for other requests")
        page = self._free.pop()
        self._ref[page - self.first_page] = 1
        drawn.add(page)
        return page

    def share(self, owner: Hashable, pages: Sequence[int]) -> None:
        """``owner`` holds ``pages`` too, beside whoever holds them now."""
        if owner not in self._quota:
            raise KeyError(f"{owner!r} is not registered in this pool")
        new = set(pages)
        if len(new) != len(pages) or not new.isdisjoint(self._drawn[owner]) or not new.isdisjoint(self._borrowed[owner]):
            raise ValueError(f"a page is already held by {owner!r}, or named twice")
        places = np.asarray(pages, dtype=np.int64) - self.first_page
        if places.size and (places.min() < 0 or places.max() >= self.num_pages or not self._refs[places].all()):
            raise ValueError("a page to be shared is free")
        self._refs[places] += 1
        self._borrowed[owner] |= new

    def give_back(self, owner: Hashable, page: int) -> None:
        """Return one page while the owner lives on (a window has passed it)."""
        drawn, place = self._drawn.get(owner, ()), page - self.first_page
        if page in drawn:
            if self._ref[place] > 1:
                # (the reservation would be owed a page that is not free)
                raise ValueError(f"page {page} is shared and cannot be given back by the one who drew it before it ends")
            if len(drawn) <= self._quota[owner]:
                self._reserved_unallocated += 1   # the reservation covers the peak, so it is owed again
            drawn.remove(page)
        elif page in self._borrowed.get(owner, ()):
            self._borrowed[owner].remove(page)    # (another's draw: no reservation of the owner covers it)
        else:
            raise ValueError(f"page {page} is not held by {owner!r}")
        self._ref[place] -= 1
        if self._ref[place] == 0:
            self._free.append(page)

    def _let_go(self, pages: Sequence[int]) -> None:
        """One holder less for each page; those without one are free, in the order given."""
        places = np.asarray(pages, dtype=np.int64) - self.first_page
        self._refs[places] -= 1
        self._free.extend((places[self._refs[places] == 0] + self.first_page).tolist())

    def release(self, owner: Hashable, pages: List[int]) -> None:
        """The owner ends: it lets go of its remaining pages and its reservation is dropped."""
        if owner not in self._quota:
            return
        drawn, borrowed = self._drawn[owner], self._borrowed[owner]
        named = set(pages)
        if len(named) != len(pages) or not named <= drawn | borrowed:
            raise ValueError(f"a page named in the release is not held by {owner!r}, or named twice")
        if len(named) != len(drawn) + len(borrowed):
            raise ValueError(f"{owner!r} ended while still holding {len(drawn) + len(borrowed) - len(named)} pages not named in "
                             f"the release")
        self._reserved_unallocated -= max(0, self._quota.pop(owner) - len(drawn))
        del self._drawn[owner], self._borrowed[owner]
        if pages:
            self._let_go(pages)

    def compact(self) -> Dict[int, int]:
        """Rename the held pages so that they have the lowest ids, and hand out free ones from the lowest on again.  Returns where
        the pages that move go (free ids all: no page moves to where another one was)."""
        end = self.first_page + self.used_pages
        held = self._refs > 0
        targets = (np.flatnonzero(~held[:self.used_pages]) + self.first_page).tolist()
        sources = (np.flatnonzero(held[self.used_pages:]) + end).tolist()
        moves = dict(zip(sources, targets))
        if moves:
            at, to = np.asarray(sources) - self.first_page, np.asarray(targets) - self.first_page
            self._refs[to] = self._refs[at]
            self._refs[at] = 0
            for holdings in (self._drawn, self._borrowed):
                for owner, pages in holdings.items():
                    holdings[owner] = {moves.get(page, page) for page in pages}
        self._free = list(range(self.first_page + self.num_pages - 1, end - 1, -1))
        return moves

    def check(self) -> None:
        """Invariants: every page is free or held, its holders counted right; reservations are honoured."""
        refs = np.zeros(self.num_pages, dtype=np.int32)
        for owner in self._quota:
            drawn, borrowed = self._drawn[owner], self._borrowed[owner]
            if not drawn.isdisjoint(borrowed):
                raise AssertionError(f"{owner!r} holds a page twice")
            refs[np.asarray(sorted(drawn | borrowed), dtype=np.int64) - self.first_page] += 1
        if sum(len(d) for d in self._drawn.values()) != len(set().union(*self._drawn.values())):
            raise AssertionError("a page was drawn twice")
        if not (refs == self._refs).all():
            raise AssertionError("held counts disagree with ownership")
        if sorted(self._free) != (np.flatnonzero(refs == 0) + self.first_page).tolist():
            raise AssertionError("a page was lost, duplicated, or freed twice")
        expected = sum(max(0, self._quota[o] - len(self._drawn[o])) for o in self._quota)
        if expected != self._reserved_unallocated or self._reserved_unallocated > len(self._free):
            raise AssertionError("reservation accounting is inconsistent")


class StateSlots:
    def __init__(self, capacity: int):
        if capacity <= 0:
            raise ValueError("state slots need a positive capacity")
        self.capacity = capacity
        self._free: List[int] = list(range(capacity - 1, -1, -1))
        self._slot: Dict[Hashable, int] = {}

    @property
    def free_slots(self) -> int:
        return len(self._free)

    def allocate(self, owner: Hashable) -> Optional[int]:
        if owner in self._slot or not self._free:
            return None
        slot = self._free.pop()
        self._slot[owner] = slot
        return slot

    def get(self, owner: Hashable) -> Optional[int]:
        return self._slot.get(owner)

    def release(self, owner: Hashable) -> None:
        slot = self._slot.pop(owner, None)
        if slot is not None:
            self._free.append(slot)

    def check(self) -> None:
        ids = list(self._free) + list(self._slot.values())
        if sorted(ids) != list(range(self.capacity)):
            raise AssertionError("a state slot was lost, duplicated, or freed twice")
