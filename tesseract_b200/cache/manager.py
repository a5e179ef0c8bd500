"""The cache manager: pages with a block table per request, in groups, plus state slots.

Run entries with the same cache need (same kv heads, head size and window; or the same
fixed-size state) form a *group*.  A paged group has its own page pool and one block
table per live request, shared by the group's entries (each entry has its own storage
``[pages + 1, *need.page_shape(page_size)]`` addressed by the same page ids, for keys and
values ``[pages + 1, 2, kv_heads, page_size, head_dim]``; page 0 is a scratch page that no
request owns, for padded rows).  A state group has storage
``[entries, slots + 1, *shape]`` addressed by the request's state slot (the last slot is scratch).  Every live request
holds one state slot whether or not the model has state groups
(src/engine/recurrent.rs:6-38; groups after src/engine/state.rs:31-132).

Pages are allocated when a request's positions first reach them, returned one by one
once a sliding window has passed them (pages of first positions that a need keeps stay), and all returned when the request ends; returned
pages are handed out again first.  ``admit`` with ``reserve_tokens`` sets aside the
request's peak need in every group (src/engine/kv.rs:36-51), so an admitted request
cannot run out; without a reservation pages come on demand and ``extend`` raises
:class:`OutOfPages` when none is left.

``fork`` gives a request continuations that go on from where it is: pages that are full are held by all of them together, the
page that is still being filled and the fixed-size state are copied (as are the pages of groups that give pages back while a
request lives, whose window moves on for each by itself), all copies of a call in one launch.  ``compact`` moves pages to the
lowest ids.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from .. import kernels
from ..parts.base import CacheBinding, PagedKVNeed, PagedNeed, StateNeed
from .pages import OutOfPages, PagePool, StateSlots


@dataclass
class _Group:
    need: object
    entries: List[int]
    pool: Optional[PagePool] = None
    storage: Optional[torch.Tensor] = None
    tables: Optional[np.ndarray] = None       # int32 [slots, columns]; 0 where no page is held


@dataclass
class _Request:
    slot: int
    length: int = 0                            # tokens whose keys/values are stored
    pages: List[Dict[int, int]] = field(default_factory=list)   # per paged group: logical index -> page id
    first_live: List[int] = field(default_factory=list)         # per group: lowest logical page still held
    family: object = field(default_factory=object)              # the same for a request and its continuations


class CacheManager:
    def __init__(self, needs: Sequence[Optional[object]], cache_of: Sequence[Optional[int]], *, num_pages: int,
                 page_size: int, max_requests: int, dtype: torch.dtype, device, max_step_tokens: int = 1,
                 allocate_storage: bool = True):
        if len(needs) != len(cache_of):
            raise ValueError("needs and cache_of must describe the same run entries")
        self.page_size = page_size
        self.num_pages = num_pages
        self.max_requests = max_requests
        self.max_step_tokens = max(1, max_step_tokens)
        self.dtype = dtype
        self.device = device
        self.slots = StateSlots(max_requests)
        self.scratch_slot = max_requests       # one state slot more than requests: padded rows point here
        self.groups: List[_Group] = []
        # per run entry: (group, index in the group's storage) of each of its needs (one, or several for a tuple)
        self._places: List[List[Tuple[int, int]]] = [[] for _ in needs]
        by_need: Dict[object, int] = {}
        for entry, entry_need in enumerate(needs):
            if entry_need is None:
                continue
            for need in (entry_need if isinstance(entry_need, tuple) else (entry_need,)):
                if need not in by_need:
                    by_need[need] = len(self.groups)
                    self.groups.append(_Group(need=need, entries=[]))
                group = by_need[need]
                self._places[entry].append((group, len(self.groups[group].entries)))
                self.groups[group].entries.append(entry)
        for group in self.groups:
            need = group.need
            if isinstance(need, PagedNeed):
                pages = need.pool_pages(num_pages, max_requests)     # (fewer where an entry serves several positions)
                group.pool = PagePool(pages, first_page=1)
                group.tables = np.zeros((max_requests, 8), dtype=np.int32)
                if allocate_storage:      # the need says what a page looks like; page 0 is the scratch page
                    group.storage = torch.zeros(
                        (len(group.entries), pages + 1, *need.page_shape(page_size)),
                        dtype=need.dtype or dtype, device=device)
            elif isinstance(need, StateNeed):
                if allocate_storage:
                    group.storage = torch.zeros((len(group.entries), max_requests + 1, *need.shape),
                                                dtype=need.dtype, device=device)
            else:
                raise TypeError(f"a cache need is a PagedNeed or a StateNeed, got {need!r}")
        self.bindings: List[Optional[CacheBinding]] = []
        for entry, need in enumerate(needs):
            source = entry if cache_of[entry] is None else cache_of[entry]
            made = []
            for group, index in self._places[source]:
                g = self.groups[group]
                storage = g.storage[index] if g.storage is not None else None
                made.append(CacheBinding(group=group, storage=storage, writes=cache_of[entry] is None,
                                         page_size=page_size if g.pool is not None else 0))
            if not made:
                self.bindings.append(None)
            elif isinstance(needs[source], tuple):
                self.bindings.append(tuple(made))
            else:
                self.bindings.append(made[0])
        # bytes that a block of 64 tokens takes in an entry of the groups that continuations hold together (the largest)
        self.shared_block_bytes = max((64 * 2 * g.need.num_kv_heads * g.need.head_dim
                                       * torch.empty((), dtype=g.need.dtype or dtype).element_size()
                                       for i, g in enumerate(self.groups) if self.shares_keys(i)), default=0)
        self._requests: Dict[Hashable, _Request] = {}
        self.pages_reused = 0          # pages handed out that an earlier owner had given back
        self._ever_used: List[set] = [set() for _ in self.groups]

    # ------------------------------------------------------------------ sizes
    def pages_for(self, group: _Group, tokens: int) -> int:
        """Peak pages a request of ``tokens`` tokens holds in ``group`` at any one time."""
        total = -(-group.need.entries_for(tokens) // self.page_size)
        span = group.need.live_span()
        if span is not None:
            live = -(-(span + self.max_step_tokens) // self.page_size) + 1
            return min(total, live + self._pinned_pages(group))
        return total

    def bytes_per_token(self) -> int:
        total = 0
        for g in self.groups:
            if g.pool is not None:
                elem = torch.empty((), dtype=g.need.dtype or self.dtype).element_size()
                page = 1
                for extent in g.need.page_shape(self.page_size):
                    page *= extent
                total += len(g.entries) * (page // self.page_size) * elem
        return total

    # ------------------------------------------------------------------ lifecycle
    def can_admit(self, reserve_tokens: Optional[int]) -> bool:
        if self.slots.free_slots == 0:
            return False
        if reserve_tokens is None:
            return True
        return all(g.pool is None or self.pages_for(g, reserve_tokens) <= g.pool.available_to_reserve
                   for g in self.groups)

    def admit(self, request: Hashable, reserve_tokens: Optional[int] = None) -> bool:
        """Give ``request`` a state slot and (optionally) reserve its pages; False if it does not fit now."""
        if request in self._requests:
            raise ValueError(f"request {request!r} is already live")
        if not self.can_admit(reserve_tokens):
            return False
        slot = self.slots.allocate(request)
        assert slot is not None
        self._clear_state(slot)                      # a new request starts from empty state
        for g in self.groups:
            if g.pool is None:
                continue
            if reserve_tokens is None:
                g.pool.register(request)
            else:
                ok = g.pool.reserve(request, self.pages_for(g, reserve_tokens))
                assert ok
            g.tables[slot, :] = 0
        self._requests[request] = _Request(slot=slot, pages=[{} for _ in self.groups],
                                           first_live=[0 for _ in self.groups])
        return True

    def _clear_state(self, slot: int) -> None:
        stores = [g.storage for g in self.groups if g.pool is None and g.storage is not None and g.storage.numel()]
        if stores and all(s.is_cuda and s.device.index == torch.cuda.current_device() for s in stores):
            kernels.clear_slot(stores, slot)
        else:
            for store in stores:
                store[:, slot].zero_()

    def is_live(self, request: Hashable) -> bool:
        return request in self._requests

    def length(self, request: Hashable) -> int:
        return self._requests[request].length

    def slot(self, request: Hashable) -> int:
        return self._requests[request].slot

    def extend(self, request: Hashable, new_tokens: int) -> None:
        """Make sure pages exist for positions ``[length, length + new_tokens)`` in every paged group."""
        state = self._requests[request]
        for index, g in enumerate(self.groups):
            if g.pool is None:
                continue
            last = (g.need.entries_for(state.length + new_tokens) - 1) // self.page_size
            held = state.pages[index]
            if g.tables.shape[1] <= last:
                columns = max(last + 1, 2 * g.tables.shape[1])
                grown = np.zeros((self.max_requests, columns), dtype=np.int32)
                grown[:, :g.tables.shape[1]] = g.tables
                g.tables = grown
            first_needed = self._first_needed_page(g, state.length)
            begin = max(first_needed, state.first_live[index])
            if g.need.live_span() is None:
                begin = max(begin, len(held))         # (nothing has been given back: the pages up to there are held)
            for logical in range(begin, last + 1):
                if logical in held:
                    continue
                page = g.pool.allocate(request)       # may raise OutOfPages
                if page in self._ever_used[index]:
                    self.pages_reused += 1
                self._ever_used[index].add(page)
                held[logical] = page
                g.tables[state.slot, logical] = page

    def commit(self, request: Hashable, new_tokens: int) -> None:
        """The step stored ``new_tokens`` more tokens; give back pages a window has passed."""
        state = self._requests[request]
        state.length += new_tokens
        for index, g in enumerate(self.groups):
            if g.pool is None or g.need.live_span() is None:
                continue
            first_needed = self._first_needed_page(g, state.length)
            held = state.pages[index]
            for logical in range(max(state.first_live[index], self._pinned_pages(g)), first_needed):
                page = held.pop(logical, None)
                if page is not None:
                    g.pool.give_back(request, page)
                    g.tables[state.slot, logical] = 0
            state.first_live[index] = max(state.first_live[index], first_needed)

    def release(self, request: Hashable) -> None:
        """The request ends: all its pages and its state slot go back."""
        state = self._requests.pop(request, None)
        if state is None:
            return
        for index, g in enumerate(self.groups):
            if g.pool is None:
                continue
            g.pool.release(request, list(state.pages[index].values()))
            g.tables[state.slot, :] = 0
        self.slots.release(request)

    # ------------------------------------------------------------------ continuations
    def _shareable_pages(self, group: _Group, length: int) -> int:
        """Leading pages of a request of ``length`` tokens that nothing writes to any more and that stay while it lives."""
        if group.need.live_span() is not None:
            return 0
        return length // group.need.positions_per_entry // self.page_size

    def fork_pages(self, length: int, reserve_tokens: int) -> List[Tuple[int, int]]:
        """Per paged group: the pages that a continuation of a request of ``length`` tokens shares, and those it draws of its own
        until it has ``reserve_tokens``."""
        out = []
        for g in self.groups:
            if g.pool is not None:
                shared = self._shareable_pages(g, length)
                out.append((shared, self.pages_for(g, reserve_tokens) - shared))
        return out

    def fork(self, pairs: Sequence[Tuple[Hashable, Hashable]], reserve_tokens: Union[int, Sequence[int], None] = None) -> bool:
        """For every ``(parent, child)``: the new request ``child`` goes on from where ``parent`` is.  With ``reserve_tokens`` (a
        number, or one a pair) the pages that each child may need up to that many tokens are set aside.  All of them, or none and
        False if they do not fit now.  The copies are enqueued on the current stream, behind the step that filled the parents' last pages."""
        pairs = list(pairs)
        if reserve_tokens is None or isinstance(reserve_tokens, int):
            reserve_tokens = [reserve_tokens] * len(pairs)
        if len(reserve_tokens) != len(pairs):
            raise ValueError("one number of tokens for all continuations, or one each")
        children = [child for _, child in pairs]
        if len(set(children)) != len(children):
            raise ValueError("a continuation is named twice")
        for (parent, child), reserve in zip(pairs, reserve_tokens):
            if parent not in self._requests:
                raise ValueError(f"request {parent!r} is not live")
            if child in self._requests:
                raise ValueError(f"request {child!r} is already live")
            if reserve is not None and reserve < self._requests[parent].length:
                raise ValueError(f"request {parent!r} has more than {reserve} tokens already")
        if len(pairs) > self.slots.free_slots:
            return False
        draws = [0] * len(self.groups)
        for (parent, _), reserve in zip(pairs, reserve_tokens):
            state = self._requests[parent]
            for index, g in enumerate(self.groups):
                if g.pool is None:
                    continue
                shared = self._shareable_pages(g, state.length)
                if reserve is not None:
                    draws[index] += self.pages_for(g, reserve) - shared
                else:
                    draws[index] += len(state.pages[index]) - shared
        if any(g.pool is not None and draws[i] > g.pool.available_to_reserve for i, g in enumerate(self.groups)):
            return False
        moves: List[Tuple[List[int], List[int]]] = [([], []) for _ in self.groups]
        for (parent, child), reserve in zip(pairs, reserve_tokens):
            state = self._requests[parent]
            slot = self.slots.allocate(child)
            new = _Request(slot=slot, length=state.length, pages=[{} for _ in self.groups],
                           first_live=list(state.first_live), family=state.family)
            for index, g in enumerate(self.groups):
                sources, targets = moves[index]
                if g.pool is None:
                    sources.append(state.slot)
                    targets.append(slot)
                    continue
                shared = self._shareable_pages(g, state.length)
                if reserve is None:
                    g.pool.register(child)
                else:
                    g.pool.reserve(child, self.pages_for(g, reserve) - shared)
                held = dict(state.pages[index])
                own = [logical for logical in held if logical >= shared] if shared == 0 else list(range(shared, len(held)))
                if shared:                       # (of such a group every page from the first on is held)
                    g.pool.share(child, [held[logical] for logical in range(shared)])
                g.tables[slot, :] = g.tables[state.slot, :]
                for logical in own:
                    sources.append(held[logical])
                    page = g.pool.allocate(child)
                    targets.append(page)
                    self._ever_used[index].add(page)
                    held[logical] = page
                    g.tables[slot, logical] = page
                new.pages[index] = held
            self._requests[child] = new
        self._copy(moves)
        return True

    def compact(self) -> int:
        """Move the pages in use to the lowest ids of every group (one launch); returns how many moved.  The block tables of
        steps that are built from now on name the new places.

        No step needs it (any free page serves any request): it is for a caller of the cache that wants the pages in use together,
        to save them or to see how small the pool could be.  Steps that were launched on the current stream before finish on the old
        places, as the copies are behind them; a step that was built but not launched yet names places that are no longer its
        requests', so there must be none."""
        moves: List[Tuple[List[int], List[int]]] = []
        for index, g in enumerate(self.groups):
            renamed = g.pool.compact() if g.pool is not None else {}
            moves.append((list(renamed), list(renamed.values())))
            if not renamed:
                continue
            for state in self._requests.values():
                held = state.pages[index]
                for logical, page in held.items():
                    if page in renamed:
                        held[logical] = renamed[page]
                        g.tables[state.slot, logical] = renamed[page]
            self._ever_used[index].update(renamed.values())
        self._copy(moves)
        return sum(len(sources) for sources, _ in moves)

    def _copy(self, moves: Sequence[Tuple[List[int], List[int]]]) -> None:
        """Pages (or state slots) of every group from the first list's places to the second's, in all entries."""
        todo = [(g.storage, sources, targets) for g, (sources, targets) in zip(self.groups, moves)
                if g.storage is not None and g.storage.numel() and sources]
        if todo and all(s.is_cuda and s.device.index == torch.cuda.current_device() for s, _, _ in todo):
            kernels.copy_pages(todo)
        else:
            for storage, sources, targets in todo:
                storage[:, targets] = storage[:, sources]

    def shares_keys(self, group_index: int) -> bool:
        """Whether continuations hold full pages of this group together: keys and values of every token, an entry each."""
        need = self.groups[group_index].need
        return isinstance(need, PagedKVNeed) and need.live_span() is None

    def rows_in_common(self, requests: Sequence[Hashable]) -> Tuple[List[List[int]], List[int]]:
        """The rows of a step of ``requests`` (one a request) in groups whose first tokens lie in the same pages wherever full pages
        are held together, and how many tokens that is; a request without such company is a group of its own."""
        states = [self._requests[r] for r in requests]
        families: Dict[int, List[int]] = {}
        for row, state in enumerate(states):
            families.setdefault(id(state.family), []).append(row)
        groups, common = list(families.values()), []
        tables = [g.tables for i, g in enumerate(self.groups) if self.shares_keys(i)]
        for rows in groups:
            pages = min(states[row].length for row in rows) // self.page_size if len(rows) > 1 and tables else 0
            for table in tables if pages else ():
                mine = table[[states[row].slot for row in rows], :pages]
                same = (mine == mine[0]).all(axis=0)
                if not same.all():
                    pages = int(same.argmin())
            common.append(pages * self.page_size)
        return groups, common

    def has_company(self, requests: Sequence[Hashable]) -> bool:
        """Whether two of ``requests`` are continuations of one prompt."""
        return len({id(self._requests[r].family) for r in requests}) < len(requests)

    def _pinned_pages(self, group: _Group) -> int:
        """Leading pages that stay as long as the request lives (they hold positions that every later query reads)."""
        return -(-group.need.keep_first // self.page_size)

    def _first_needed_page(self, group: _Group, next_position: int) -> int:
        """Lowest logical page that a query at ``next_position`` or later can still read."""
        return group.need.first_needed_position(next_position) // self.page_size

    # ------------------------------------------------------------------ views
    def block_table_rows(self, group_index: int, slots: Sequence[int], columns: int) -> np.ndarray:
        """int32 ``[len(slots), columns]`` copy of the block tables of the given state slots."""
        tables = self.groups[group_index].tables
        have = min(columns, tables.shape[1])
        out = np.zeros((len(slots), columns), dtype=np.int32)
        out[:, :have] = tables[np.asarray(slots, dtype=np.int64), :have]
        return out

    def pages_of(self, request: Hashable, group_index: int = 0) -> Dict[int, int]:
        return dict(self._requests[request].pages[group_index])

    def used_pages(self) -> int:
        return sum(g.pool.used_pages for g in self.groups if g.pool is not None)

    def check(self) -> None:
        self.slots.check()
        for index, g in enumerate(self.groups):
            if g.pool is None:
                continue
            g.pool.check()
            seen: Dict[int, int] = {}
            for request, state in self._requests.items():
                for logical, page in state.pages[index].items():
                    seen[page] = seen.get(page, 0) + 1
                    if request not in g.pool.holders_of(page):
                        raise AssertionError(f"page {page} ownership disagrees")
                    if g.tables[state.slot, logical] != page:
                        raise AssertionError(f"the block table of {request!r} disagrees at page {logical}")
            if any(count != len(g.pool.holders_of(page)) for page, count in seen.items()):
                raise AssertionError("a page has holders that no request's table names")
            if len(seen) != g.pool.used_pages:
                raise AssertionError("pool holds pages that no request's table names")
