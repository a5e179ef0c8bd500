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

from typing import Dict, Hashable, List, Optional


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
        self._holders: Dict[int, List[Hashable]] = {}      # page -> who holds it, the longest-standing holder first
        self._quota: Dict[Hashable, int] = {}
        self._held: Dict[Hashable, int] = {}                # pages drawn by the owner (and not given back)
        self._borrowed: Dict[Hashable, set] = {}            # pages that it shares and others drew
        self._reserved_unallocated = 0

    # ---------------------------------------------------------------- queries
    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def used_pages(self) -> int:
        return len(self._holders)

    @property
    def available_to_reserve(self) -> int:
        return len(self._free) - self._reserved_unallocated

    def held_by(self, owner: Hashable) -> int:
        return self._held.get(owner, 0) + len(self._borrowed.get(owner, ()))

    def owner_of(self, page: int) -> Optional[Hashable]:
        holders = self._holders.get(page)
        return holders[0] if holders else None

    def holders_of(self, page: int) -> List[Hashable]:
        return list(self._holders.get(page, ()))

    # ---------------------------------------------------------------- reservations
    def reserve(self, owner: Hashable, pages: int) -> bool:
        """Set aside ``pages`` pages for ``owner`` (its peak simultaneous need)."""
        if owner in self._quota or owner in self._held:
            return False
        if pages > self.available_to_reserve:
            return False
        self._quota[owner] = pages
        self._held[owner] = 0
        self._reserved_unallocated += pages
        return True

    def register(self, owner: Hashable) -> None:
        """Admit ``owner`` without a reservation: its pages come on demand."""
        if owner in self._held:
            raise ValueError(f"{owner!r} is already registered in this pool")
        self._quota[owner] = 0
        self._held[owner] = 0

    # ---------------------------------------------------------------- pages
    def allocate(self, owner: Hashable) -> int:
        if owner not in self._held:
            raise KeyError(f"{owner!r} is not registered in this pool")
        held, quota = self._held[owner], self._quota[owner]
        if held < quota:
            self._reserved_unallocated -= 1   # drawing on the owner's own reservation
        elif self.available_to_reserve <= 0:
            raise OutOfPages(f"cache pool exhausted: {self.num_pages} pages, {len(self._free)} free, "
                             f"{self._reserved_unallocated} reserved for other requests")
        page = self._free.pop()
        self._holders[page] = [owner]
        self._held[owner] = held + 1
        return page

    def share(self, owner: Hashable, page: int) -> None:
        """``owner`` holds ``page`` too, beside whoever holds it now."""
        if owner not in self._held:
            raise KeyError(f"{owner!r} is not registered in this pool")
        holders = self._holders.get(page)
        if holders is None:
            raise ValueError(f"page {page} is free")
        if owner in holders:
            raise ValueError(f"page {page} is already held by {owner!r}")
        holders.append(owner)
        self._borrowed.setdefault(owner, set()).add(page)

    def give_back(self, owner: Hashable, page: int) -> None:
        """Return one page while the owner lives on (a window has passed it)."""
        holders = self._holders.get(page, ())
        if owner not in holders:
            raise ValueError(f"page {page} is not held by {owner!r}")
        if page in self._borrowed.get(owner, ()):
            self._borrowed[owner].remove(page)              # (another's draw: no reservation of the owner covers it)
            self._let_go(owner, page)
            return
        if len(holders) > 1:
            # (the reservation would be owed a page that is not free)
            raise ValueError(f"page {page} is shared and cannot be given back by the one who drew it before it ends")
        self._let_go(owner, page)
        held = self._held[owner]
        self._held[owner] = held - 1
        if held <= self._quota[owner]:
            self._reserved_unallocated += 1   # the reservation covers the peak, so it is owed again

    def _let_go(self, owner: Hashable, page: int) -> None:
        holders = self._holders[page]
        holders.remove(owner)
        if not holders:
            del self._holders[page]
            self._free.append(page)

    def release(self, owner: Hashable, pages: List[int]) -> None:
        """The owner ends: it lets go of its remaining pages and its reservation is dropped."""
        if owner not in self._held:
            return
        borrowed = self._borrowed.pop(owner, set())
        drawn = 0
        for page in pages:
            if owner not in self._holders.get(page, ()):
                raise ValueError(f"page {page} is not held by {owner!r}")
            drawn += page not in borrowed
            self._let_go(owner, page)
        held = self._held.pop(owner) - drawn + len(borrowed) - (len(pages) - drawn)
        quota = self._quota.pop(owner)
        if held != 0:
            raise ValueError(f"{owner!r} ended while still holding {held} pages not named in the release")
        self._reserved_unallocated -= max(0, quota - drawn)

    def compact(self) -> Dict[int, int]:
        """Rename the held pages so that they have the lowest ids, and hand out free ones from the lowest on again.  Returns where
        the pages that move go (free ids all: no page moves to where another one was)."""
        end = self.first_page + len(self._holders)
        targets = [page for page in range(self.first_page, end) if page not in self._holders]
        sources = sorted(page for page in self._holders if page >= end)
        moves = dict(zip(sources, targets))
        for source, target in moves.items():
            self._holders[target] = self._holders.pop(source)
        for owner, pages in self._borrowed.items():
            self._borrowed[owner] = {moves.get(page, page) for page in pages}
        self._free = list(range(self.first_page + self.num_pages - 1, end - 1, -1))
        return moves

    def check(self) -> None:
        """Invariants: every page is free or owned, exactly once; reservations are honoured."""
        ids = list(self._free) + list(self._holders)
        if sorted(ids) != list(range(self.first_page, self.first_page + self.num_pages)):
            raise AssertionError("a page was lost, duplicated, or freed twice")
        counts: Dict[Hashable, int] = {}
        for page, holders in self._holders.items():
            if not holders or len(set(holders)) != len(holders):
                raise AssertionError(f"page {page} has no holder, or one twice")
            for owner in holders:
                counts[owner] = counts.get(owner, 0) + 1
        if any(counts.get(o, 0) != self.held_by(o) for o in self._held) or any(o not in self._held for o in counts):
            raise AssertionError("held counts disagree with ownership")
        expected = sum(max(0, self._quota[o] - self._held[o]) for o in self._held)
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
