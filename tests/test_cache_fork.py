"""Pages held by several requests: forks, releases in any order, compaction (host bookkeeping, no GPU)."""

from __future__ import annotations

import random

import numpy as np
import pytest

from rapid_llm_b200.cache import CacheManager, plan_groups
from rapid_llm_b200.cache.manager import CacheError, PagePool
from rapid_llm_b200.parts.base import CacheNeed


def manager(pages=40, slots=6, needs=None, page_size=4, max_seq_len=64):
    groups, _ = plan_groups(needs or [CacheNeed("full", 1, 16)])
    return CacheManager(groups, page_size=page_size, num_pages=pages, max_num_seqs=slots, max_seq_len=max_seq_len)


def test_a_page_is_free_when_its_last_holder_gives_it_back():
    pool = PagePool(4)
    pages = pool.allocate(3)
    pool.share(pages[:2])
    pool.free(pages)
    assert pool.num_free == 2 and pool.holders(pages[0]) == 1
    pool.check()
    with pytest.raises(CacheError):
        pool.free([pages[2]])
    with pytest.raises(CacheError):
        pool.share([pages[2]])
    pool.free(pages[:2])
    assert pool.num_free == 4
    pool.check()


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 8, 11])
def test_a_fork_shares_whole_pages_and_copies_the_ragged_one(tokens):
    cache = manager()
    cache.admit("p")
    assert cache.reserve("p", tokens)
    before = cache.num_free_pages()
    copies = cache.fork("p", ["a", "b"])
    whole, ragged = divmod(tokens, 4)
    parent = cache.pages_of("p")[0]
    assert [len(c) for c in copies] == [2 if ragged else 0] and before - cache.num_free_pages() == (2 if ragged else 0)
    for child in ("a", "b"):
        mine = cache.pages_of(child)[0]
        assert mine[:whole] == parent[:whole] and cache.num_tokens(child) == tokens
        assert list(cache.block_tables[0][cache.slot_of(child), : len(mine)]) == mine
        if ragged:
            assert (parent[whole], mine[whole]) in copies[0] and mine[whole] not in parent
        assert cache.shared_prefix(child) == cache.shared_prefix("p")
        assert cache.shared_prefix(child) is None if whole == 0 else cache.shared_prefix(child)[1] == whole * 4
    cache.check()
    # everyone grows on pages of its own
    for name in ("p", "a", "b"):
        assert cache.reserve(name, tokens + 6)
    grown = [set(cache.pages_of(name)[0][whole:]) for name in ("p", "a", "b")]
    assert not (grown[0] & grown[1] or grown[0] & grown[2] or grown[1] & grown[2])
    cache.check()
    for name in ("p", "b", "a"):
        cache.release(name)
        cache.check()
    assert cache.num_free_pages() == 40


def test_nothing_is_taken_when_slots_or_pages_are_short():
    cache = manager(pages=4, slots=3)
    cache.admit("p")
    assert cache.reserve("p", 10)
    assert cache.fork("p", ["a", "b", "c"]) is None            # slots
    assert cache.fork("p", ["a", "b"]) is None                 # a page each, one is left
    assert cache.num_free_pages() == 1 and cache.num_free_slots == 2 and not cache.has("a")
    assert cache.fork("p", ["a"]) is not None
    for wrong in (["a"], ["x", "x"], ["p"]):
        with pytest.raises(CacheError):
            cache.fork("p", wrong)
    with pytest.raises(CacheError):
        cache.fork("nobody", ["x"])
    assert cache.fork("p", []) == [[]]
    cache.check()


def test_windows_keep_what_they_still_need():
    cache = manager(needs=[CacheNeed("full", 1, 16), CacheNeed("window", 1, 16, 6), CacheNeed("chunk", 1, 16, chunk=8)])
    cache.admit("p")
    assert cache.reserve("p", 18)
    cache.release_passed("p")
    assert cache.fork("p", ["a"]) is not None
    cache.check()
    for _ in range(6):
        for name in ("p", "a"):
            assert cache.reserve(name, cache.num_tokens(name) + 3)
            cache.release_passed(name)
            cache.check()
    cache.release("p")
    cache.release("a")
    cache.check()
    assert all(pool.num_free == 40 for pool in cache.pools)


def test_compaction_moves_held_pages_to_the_lowest_ids():
    cache = manager(pages=30, slots=4)
    for name, tokens in (("a", 20), ("b", 13), ("c", 9)):
        cache.admit(name)
        assert cache.reserve(name, tokens)
    cache.fork("b", ["d"])
    cache.release("a")
    content = {page: f"content {page}" for page in range(31)}
    before = {name: [content[page] for page in cache.pages_of(name)[0]] for name in "bcd"}
    moves = cache.compact(0)
    assert moves and len({t for _, t in moves}) == len(moves) and not {t for _, t in moves} & {s for s, _ in moves}
    for source, target in moves:
        content[target] = content[source]
    after = {name: [content[page] for page in cache.pages_of(name)[0]] for name in "bcd"}
    assert after == before
    held = cache.pools[0].num_held
    assert {page for name in "bcd" for page in cache.pages_of(name)[0]} == set(range(1, held + 1))
    assert cache.take_dirty(0) and all((cache.block_tables[0][cache.slot_of(n), : len(cache.pages_of(n)[0])] == cache.pages_of(n)[0]).all() for n in "bcd")
    assert cache.compact(0) == []
    cache.check()


@pytest.mark.parametrize("seed", range(8))
def test_random_lives(seed):
    """Admissions, growth, forks of forks, compaction and releases in any order: the tables always name each request's own history."""
    rng = random.Random(seed)
    cache = manager(pages=rng.choice((12, 25, 60)), slots=7, needs=[CacheNeed("full", 1, 16), CacheNeed("window", 1, 16, 9)])
    memory = [dict(), dict()]                    # group -> (page, offset) -> token
    history: dict[int, list[int]] = {}
    names = iter(range(10_000))
    for step in range(300):
        kind = rng.choice(("admit", "grow", "grow", "grow", "fork", "release", "compact"))
        if kind == "admit" and cache.num_free_slots:
            name = next(names)
            cache.admit(name)
            history[name] = []
        elif kind == "grow" and history:
            name = rng.choice(list(history))
            count = rng.randint(1, 7)
            if len(history[name]) + count <= 64 and cache.reserve(name, len(history[name]) + count):
                for group in range(2):
                    dest = cache.kv_destinations(group, cache.slot_of(name), len(history[name]), count)
                    for i, place in enumerate(dest):
                        memory[group][int(place)] = (name, step, i)
                history[name] += [(name, step, i) for i in range(count)]
                cache.release_passed(name)
        elif kind == "fork" and history:
            name = rng.choice(list(history))
            children = [next(names) for _ in range(rng.randint(1, 3))]
            copies = cache.fork(name, children)
            if copies is not None:
                for group in range(2):
                    for source, target in copies[group]:
                        for offset in range(4):
                            memory[group][target * 4 + offset] = memory[group].get(source * 4 + offset)
                for child in children:
                    history[child] = list(history[name])
        elif kind == "release" and history:
            name = rng.choice(list(history))
            cache.release(name)
            del history[name]
        elif kind == "compact":
            for group in range(2):
                for source, target in cache.compact(group):
                    for offset in range(4):
                        memory[group][target * 4 + offset] = memory[group].get(source * 4 + offset)
        cache.check()
        for name, tokens in history.items():
            family = cache.shared_prefix(name)
            for group in range(2):
                table = cache.block_tables[group][cache.slot_of(name)]
                first = 0 if group == 0 else max(len(tokens) - 9 + 1, 0)
                for position in range(first, len(tokens)):
                    assert memory[group][int(table[position // 4]) * 4 + position % 4] == tokens[position]
            if family is not None:
                for other in history:
                    if cache.shared_prefix(other) is not None and cache.shared_prefix(other)[0] == family[0]:
                        count = family[1] // 4
                        assert (cache.block_tables[0][cache.slot_of(other), :count] == cache.block_tables[0][cache.slot_of(name), :count]).all()
                        assert cache.shared_prefix(other) == family and len(history[other]) >= family[1]
    assert isinstance(cache.block_tables[0], np.ndarray)


def test_who_is_left_of_a_family_forks_anew():
    cache = manager()
    cache.admit("p")
    assert cache.reserve("p", 9)
    cache.fork("p", ["a", "b"])
    assert cache.reserve("p", 21)
    cache.release("a")
    assert cache.fork("p", ["c"]) == [[(cache.pages_of("p")[0][5], cache.pages_of("c")[0][5])]]
    assert cache.shared_prefix("c") == cache.shared_prefix("b") == cache.shared_prefix("p") and cache.shared_prefix("p")[1] == 8
    cache.release("b"), cache.release("c")
    cache.fork("p", ["d"])
    assert cache.shared_prefix("d") == cache.shared_prefix("p") and cache.shared_prefix("d")[1] == 20
    cache.check()
