"""Pages with several holders, continuations and compaction: nothing lost, freed early or written twice (no GPU needed)."""

import random
import time

import numpy as np
import pytest
import torch
from hypothesis import given, settings, strategies as st

import tesseract_b200.parts  # noqa: F401
from tesseract_b200.cache import CacheManager, OutOfPages, PagePool
from tesseract_b200.parts import PagedKVNeed, StateNeed
from tesseract_b200.parts.base import PooledBlocksNeed


def test_a_shared_page_is_free_when_its_last_holder_lets_go():
    pool = PagePool(4)
    pool.register("a")
    pool.register("b")
    page = pool.allocate("a")
    pool.share("b", [page])
    assert pool.holders_of(page) == ["a", "b"] and pool.used_pages == 1 and pool.held_by("b") == 1
    pool.check()
    pool.release("a", [page])
    assert pool.free_pages == 3 and pool.owner_of(page) == "b"
    pool.check()
    pool.release("b", [page])
    assert pool.free_pages == 4
    pool.check()


def test_sharing_refuses_free_pages_strangers_and_a_second_time():
    pool = PagePool(4)
    pool.register("a")
    page = pool.allocate("a")
    with pytest.raises(KeyError):
        pool.share("b", [page])
    with pytest.raises(ValueError):
        pool.share("a", [page])
    pool.register("b")
    with pytest.raises(ValueError):
        pool.share("b", [page + 1])
    with pytest.raises(ValueError):
        pool.share("b", [page, page])
    for outside in (-1, 4):
        with pytest.raises(ValueError):
            pool.share("b", [outside])
    pool.share("b", [page])
    with pytest.raises(ValueError):
        pool.share("b", [page])
    with pytest.raises(ValueError):
        pool.give_back("a", page)          # shared: its reservation would be owed a page that is not free
    pool.give_back("b", page)              # a borrowed page may be let go of
    pool.give_back("a", page)
    pool.check()


def test_reservations_count_what_an_owner_draws():
    pool = PagePool(10)
    assert pool.reserve("a", 6)
    pages = [pool.allocate("a") for _ in range(3)]
    assert pool.reserve("b", 4)
    for page in pages[:2]:
        pool.share("b", [page])
    assert pool.available_to_reserve == 0
    own = [pool.allocate("b") for _ in range(4)]
    pool.check()
    pool.release("a", pages)
    assert pool.available_to_reserve == 4           # one page of a's is free again, and its remaining reservation of three
    pool.release("b", pages[:2] + own)
    assert pool.available_to_reserve == 10
    pool.check()


def test_compaction_takes_the_lowest_ids_and_moves_to_free_places_alone():
    pool = PagePool(8, first_page=1)
    for owner in "abc":
        pool.register(owner)
    pages = {o: [pool.allocate(o) for _ in range(2)] for o in "abc"}
    pool.share("c", [pages["b"][0]])
    pool.release("a", pages["a"])
    moves = pool.compact()
    assert moves == {5: 1, 6: 2}
    assert pool.holders_of(1) == ["c"] and pool.holders_of(3) == ["b", "c"]
    pool.check()
    assert pool.compact() == {}
    pool.register("d")
    assert [pool.allocate("d") for _ in range(2)] == [5, 6]


def manager(needs, num_pages=40, page_size=4, max_requests=6, storage=True):
    return CacheManager(needs, [None] * len(needs), num_pages=num_pages, page_size=page_size, max_requests=max_requests,
                        dtype=torch.float32, device="cpu", max_step_tokens=8, allocate_storage=storage)


class Shadow:
    """Writes a distinct number per (request lineage, position) into the cache's pages and states as steps would, and knows what
    each request must find there."""

    def __init__(self, cache):
        self.cache, self.tokens, self.state, self.next = cache, {}, {}, 1.0

    def step(self, request, count):
        cache = self.cache
        cache.extend(request, count)
        begin = cache.length(request)
        for position in range(begin, begin + count):
            self.tokens[request].append(self.next)
            for index, g in enumerate(cache.groups):
                if g.pool is None:
                    g.storage[:, cache.slot(request)] = self.next
                    continue
                entry = position // g.need.positions_per_entry
                page = int(cache.block_table_rows(index, [cache.slot(request)], entry // cache.page_size + 1)[0, -1])
                assert page > 0
                g.storage.view(g.storage.shape[0], g.storage.shape[1], -1)[:, page, entry % cache.page_size] = self.next
            self.state[request] = self.next
            self.next += 1.0
        cache.commit(request, count)

    def check(self):
        cache = self.cache
        cache.check()
        for request, tokens in self.tokens.items():
            assert cache.length(request) == len(tokens)
            for index, g in enumerate(cache.groups):
                if g.pool is None:
                    assert bool((g.storage[:, cache.slot(request)] == self.state[request]).all())
                    continue
                first = g.need.first_needed_position(len(tokens))
                table = cache.block_table_rows(index, [cache.slot(request)], 64)[0]
                flat = g.storage.view(g.storage.shape[0], g.storage.shape[1], -1)
                pool = g.need.positions_per_entry
                for entry in range(first // pool, g.need.entries_for(len(tokens))):
                    written = tokens[min(len(tokens), (entry + 1) * pool) - 1]
                    got = flat[:, int(table[entry // cache.page_size]), entry % cache.page_size]
                    assert bool((got == written).all()), (request, entry)


NEEDS = {
    "all keys": [PagedKVNeed(1, 1)],
    "a window": [PagedKVNeed(1, 1), PagedKVNeed(1, 1, 6)],
    "states": [PagedKVNeed(1, 1), StateNeed((3,))],
    "blocks": [PooledBlocksNeed(num_kv_heads=1, key_dim=1, value_dim=1, pool=3), PagedKVNeed(1, 1)],
    "states alone": [StateNeed((2, 2))],
}


@pytest.mark.parametrize("name", NEEDS)
@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8, 11, 12, 13])
def test_continuations_see_what_their_parent_wrote_and_not_each_other(name, length):
    cache = manager(NEEDS[name])
    shadow = Shadow(cache)
    assert cache.admit("p", reserve_tokens=30)
    shadow.tokens["p"], shadow.state["p"] = [], 0.0
    if length:
        shadow.step("p", length)
    assert cache.fork([("p", "x"), ("p", "y")], reserve_tokens=30)
    for child in "xy":
        shadow.tokens[child], shadow.state[child] = list(shadow.tokens["p"]), shadow.state["p"]
    shadow.check()
    for request, count in [("x", 1), ("p", 3), ("y", 2), ("x", 5)]:
        shadow.step(request, count)
        shadow.check()
    cache.release("p")
    del shadow.tokens["p"]
    shadow.step("y", 4)
    shadow.check()
    cache.compact()
    shadow.check()
    shadow.step("x", 2)
    shadow.check()
    for child in "xy":
        cache.release(child)
    assert cache.used_pages() == 0
    cache.check()
    for g in cache.groups:
        if g.pool is not None:
            assert g.pool.available_to_reserve == g.pool.num_pages


def test_full_pages_are_held_together_and_the_page_being_filled_is_copied():
    cache = manager([PagedKVNeed(1, 1)], storage=False)
    cache.admit("p")
    cache.extend("p", 10)
    cache.commit("p", 10)
    assert cache.fork([("p", "x")])
    a, b = cache.pages_of("p"), cache.pages_of("x")
    assert a[0] == b[0] and a[1] == b[1] and a[2] != b[2] and cache.used_pages() == 4
    assert cache.rows_in_common(["p", "x"]) == ([[0, 1]], [8])
    assert cache.has_company(["p", "x"]) and not cache.has_company(["x"])


def test_rows_in_common_over_forks_of_forks_and_strangers():
    cache = manager([PagedKVNeed(1, 1), PagedKVNeed(1, 1, 8)], num_pages=60, storage=False)
    for name, tokens in (("p", 9), ("s", 30)):
        cache.admit(name)
        for _ in range(tokens):
            cache.extend(name, 1)
            cache.commit(name, 1)
    cache.fork([("p", "x")])
    cache.extend("x", 8)
    cache.commit("x", 8)                                    # x: 17 tokens, p: 9
    cache.fork([("x", "y")])
    assert cache.rows_in_common(["x", "s", "y"]) == ([[0, 2], [1]], [16, 0])
    assert cache.rows_in_common(["y", "x", "p", "s"]) == ([[0, 1, 2], [3]], [8, 0])
    assert cache.shares_keys(0) and not cache.shares_keys(1)                # a window moves on for each by itself
    cache.check()


def test_forks_fit_all_or_not_at_all():
    cache = manager([PagedKVNeed(1, 1)], num_pages=10, max_requests=4, storage=False)
    assert cache.admit("p", reserve_tokens=16)              # four pages, of ten
    cache.extend("p", 9)
    cache.commit("p", 9)
    assert not cache.fork([("p", "a"), ("p", "b"), ("p", "c"), ("p", "d")], reserve_tokens=16)     # a slot short
    assert cache.fork([("p", "a"), ("p", "b"), ("p", "c")], reserve_tokens=16)                     # two of their own each: all of it
    assert cache.groups[0].pool.available_to_reserve == 0
    assert cache.fork_pages(9, 16) == [(2, 2)]
    for request in ("p", "a", "b", "c"):
        cache.extend(request, 7)                            # what was set aside is there
        cache.commit(request, 7)
    cache.check()
    cache.release("c")
    assert not cache.fork([("p", "e")], reserve_tokens=40)
    assert not cache.is_live("e")
    cache.check()


def test_forks_refuse_what_makes_no_sense():
    cache = manager([PagedKVNeed(1, 1)], storage=False)
    cache.admit("p")
    cache.extend("p", 6)
    cache.commit("p", 6)
    for pairs, reserve in [([("q", "x")], None), ([("p", "p")], None), ([("p", "x"), ("p", "x")], None), ([("p", "x")], 5),
                           ([("p", "x"), ("p", "y")], [9])]:
        with pytest.raises(ValueError):
            cache.fork(pairs, reserve)
    assert cache.fork([]) and cache.compact() == 0
    cache.check()


def test_without_a_reservation_pages_come_on_demand():
    cache = manager([PagedKVNeed(1, 1)], num_pages=3, storage=False)
    cache.admit("p")
    cache.extend("p", 6)
    cache.commit("p", 6)
    assert cache.fork([("p", "x")])
    assert not cache.fork([("p", "y")])                     # no page left for the copy
    cache.extend("x", 2)
    cache.commit("x", 2)
    with pytest.raises(OutOfPages):
        cache.extend("x", 1)
    cache.release("p")
    cache.extend("x", 1)
    cache.check()


@settings(max_examples=60, deadline=None)
@given(st.integers(0, 10 ** 6), st.sampled_from(sorted(NEEDS)))
def test_random_lives(seed, name):
    rng = random.Random(seed)
    cache = manager(NEEDS[name], num_pages=rng.randint(20, 60), page_size=rng.choice([1, 3, 4]))
    shadow, names = Shadow(cache), iter(range(10 ** 6))
    limit = 16
    for _ in range(40):
        live = list(shadow.tokens)
        act = rng.random()
        if act < 0.2 or not live:
            new = next(names)
            if cache.admit(new, reserve_tokens=limit):
                shadow.tokens[new], shadow.state[new] = [], 0.0
        elif act < 0.6:
            request = rng.choice(live)
            room = limit - cache.length(request)
            if room:
                shadow.step(request, rng.randint(1, min(room, 8)))
        elif act < 0.8:
            pairs = [(rng.choice(live), next(names)) for _ in range(rng.randint(1, 3))]
            if cache.fork(pairs, reserve_tokens=limit):
                for parent, child in pairs:
                    shadow.tokens[child], shadow.state[child] = list(shadow.tokens[parent]), shadow.state[parent]
        elif act < 0.95:
            request = rng.choice(live)
            cache.release(request)
            del shadow.tokens[request], shadow.state[request]
        else:
            cache.compact()
        shadow.check()
    for request in list(shadow.tokens):
        cache.release(request)
    assert cache.used_pages() == 0
    cache.check()


def test_a_page_given_back_costs_the_host_about_what_drawing_it_did():
    """A window that moves on gives pages back one at a time: no array operations for each (they took fifteen times a draw)."""
    pool = PagePool(2000, 1)
    pool.register("a")
    ratios = []
    for _ in range(7):
        begin = time.perf_counter()
        pages = [pool.allocate("a") for _ in range(2000)]
        between = time.perf_counter()
        for page in pages:
            pool.give_back("a", page)
        ratios.append((time.perf_counter() - between) / (between - begin))
    pool.check()
    assert pool.used_pages == 0 and min(ratios) < 5
