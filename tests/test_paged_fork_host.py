"""Forks, compaction, pools of another size and bounds of a PagedKVCache on the host, with the stand-ins of
tests/test_paged_cache_host.py; copies of pages are carried out on a table of what each page holds."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from cortex.cache import PagedKVCache, paged
from test_paged_cache_host import Host, rows, state


class ForkHost(Host):
    def __init__(self, patch):
        super().__init__(patch)
        allocate = paged.KVPages.allocate

        def bounded_allocate(*args, tracked=False, bounded=False):
            pages = allocate(*args, tracked=tracked)
            pages.bounds = torch.zeros(1) if bounded else None
            self.log.append(("allocate", args[0]))
            return pages

        patch.setattr(paged.KVPages, "allocate", bounded_allocate)
        patch.setattr(paged, "kv_copy_pages",
                      lambda pages, src, dst, into=None: self.log.append(("copy", pages, src.tolist(), dst.tolist(), into)))
        patch.setattr(paged, "kv_block_bounds", lambda pages, table, lengths, **kw: self.log.append(("bounds", pages, lengths, kw)))
        patch.setattr(paged, "paged_block_select",
                      lambda q, pages, table, lengths, count, **kw: self.log.append(("select", count, kw)) or ("table", "lengths"))


@pytest.fixture
def host(monkeypatch):
    return ForkHost(monkeypatch)


def grow(cache, name, n):
    batch = cache.extend([name], [n])
    for layer in range(len(cache.layers)):
        cache.append(batch, rows(n), rows(n), layer)
    return batch


def consistent(cache):
    users = np.zeros(cache.num_pages, dtype=int)
    for s in cache._sessions.values():
        pages = s.pages[:s.used].tolist()
        assert len(set(pages)) == len(pages) and s.used == -(-s.length // cache.page_size)
        users[pages] += 1
    assert (users == cache._users).all()
    assert sorted(cache._free) == np.flatnonzero(users == 0).tolist()
    assert cache.pages_used == int((users > 0).sum())


def test_a_fork_shares_full_pages_and_copies_the_last(host):
    cache = PagedKVCache(20, 1, 16, page_size=8, layers=2)
    grow(cache, "a", 20)
    a = cache._sessions["a"].pages[:3].tolist()
    cache.fork("a", ["b", "c"])
    b, c = (cache._sessions[n].pages[:3].tolist() for n in "bc")
    assert b[:2] == c[:2] == a[:2] and len({a[2], b[2], c[2]}) == 3
    copies = host.of("copy")
    assert [e[0] for e in copies] == cache.layers and all(e[1:] == ([a[2], a[2]], [b[2], c[2]], None) for e in copies)
    assert cache.pages_used == 5 and [cache.length(n) for n in "abc"] == [20] * 3 and cache.sessions == ["a", "b", "c"]
    assert cache.extend(["b"]).positions.tolist() == [20]
    consistent(cache)
    # shared pages go back when their last user does
    assert cache.evict_session("a") == 1 and cache.evict_session("b") == 1 and cache.evict_session("c") == 3
    assert cache.pages_used == 0
    consistent(cache)


def test_a_fork_at_the_end_of_a_page_copies_nothing(host):
    cache = PagedKVCache(4, 1, 16, page_size=8)
    grow(cache, "a", 16)
    cache.fork("a", ["b"])
    cache.extend(["e"], [0])
    cache.fork("e", ["f"])
    cache.fork("a", [])
    assert not host.of("copy") and cache.pages_used == 2
    one, two = cache.extend(["a"]).block_table[0].tolist(), cache.extend(["b"]).block_table[0].tolist()
    assert one[:2] == two[:2] and one[2] != two[2]
    consistent(cache)


def test_a_tracked_cache_shares_nothing(host):
    cache = PagedKVCache(9, 1, 16, page_size=8, tracked=True)
    grow(cache, "a", 20)
    cache.fork("a", ["b", "c"])
    assert cache.pages_used == 9 and (cache._users == 1).all()
    a = cache._sessions["a"].pages[:3].tolist()
    assert host.of("copy")[0][1] == a + a
    cache.evict(["b"], 8, 2)
    assert cache.pages_used == 7
    consistent(cache)


def test_refused_forks(host):
    cache = PagedKVCache(4, 1, 16, page_size=8, layers=2)
    batch = cache.extend(["a"], [20])
    cache.append(batch, rows(20), rows(20), 0)
    before = state(cache)
    for args, error in [(("x", ["b"]), KeyError), (("a", ["a"]), ValueError), (("a", "b"), ValueError),
                        (("a", ["b", "b"]), ValueError), (("a", ["b"]), RuntimeError)]:
        with pytest.raises(error):
            cache.fork(*args)
    cache.append(batch, rows(20), rows(20), 1)
    with pytest.raises(MemoryError):
        cache.fork("a", ["b", "c"])
    assert {**state(cache), "sessions": None} == {**before, "sessions": None} and not host.of("copy")
    cache.attend(batch, rows(1), 0)  # it still holds
    cache.fork("a", ["b"])
    for call in (lambda: cache.attend(batch, rows(1), 0), lambda: cache.append(batch, rows(20), rows(20), 0)):
        with pytest.raises(RuntimeError, match="out of date"):
            call()
    consistent(cache)


def test_who_gives_way_for_a_fork(host):
    cache = PagedKVCache(6, 1, 16, page_size=8)
    grow(cache, "old", 9)
    grow(cache, "new", 8)
    grow(cache, "a", 20)
    cache.fork("a", ["b"])
    assert cache.sessions == ["new", "a", "b"]
    consistent(cache)
    # a session whose pages others keep stays: it would free none
    cache = PagedKVCache(6, 1, 16, page_size=8)
    grow(cache, "a", 16)
    cache.fork("a", ["twin"])
    grow(cache, "last", 25)
    cache.extend(["twin"], [0])
    assert cache.sessions == ["a", "last", "twin"]
    cache.extend(["twin"], [1])
    assert cache.sessions == ["a", "twin"]
    consistent(cache)
    # two that share go together
    cache = PagedKVCache(4, 1, 16, page_size=8)
    grow(cache, "a", 24)
    cache.fork("a", ["b"])
    cache.extend(["c"], [8])
    assert cache.sessions == ["a", "b", "c"]
    cache.extend(["c"], [8])
    assert cache.sessions == ["c"] and cache.pages_used == 2
    consistent(cache)


def test_who_gives_way_is_found_without_a_look_at_every_page(host):
    """A cache that is full lets sessions go at every step: that goes by their pages, however large the pools are."""

    class Users(np.ndarray):
        def copy(self, *args, **kw):
            raise AssertionError("the counts of all pages were copied")

    cache = PagedKVCache(6, 1, 16, page_size=8)
    cache._users = cache._users.view(Users)
    grow(cache, "old", 9)
    grow(cache, "twin", 16)
    cache.fork("twin", ["other"])
    cache.extend(["old"], [0])
    users = np.array(cache._users)
    with pytest.raises(MemoryError):
        cache.extend(["new"], [8 * 7])
    assert (cache._users == users).all() and cache.sessions == ["twin", "other", "old"]
    cache.extend(["new"], [8 * 3])
    assert cache.sessions == ["old", "new"]
    consistent(cache)


def test_compaction(host):
    cache = PagedKVCache(12, 1, 16, page_size=8, layers=2)
    for name in "abcd":
        grow(cache, name, 17)
    held = cache.batch(["a"])
    moving = cache.batch(["d"])
    cache.evict_session("b")
    cache.evict_session("c")
    cache.fork("d", ["e"])
    assert cache.pages_used == 7
    shared = cache._sessions["d"].pages[:2].tolist()
    tables = {n: cache._sessions[n].pages[:3].tolist() for n in "ade"}
    high = [p for p in range(7, 12) if cache._users[p]]
    assert cache.compact() == len(high) and high
    (_, src, dst, into), (_, src2, dst2, _) = host.of("copy")[-2:]
    assert src == src2 == high and dst == dst2 and into is None and all(p < 7 for p in dst)
    place = dict(zip(src, dst))
    for n, before in tables.items():
        assert cache._sessions[n].pages[:3].tolist() == [place.get(p, p) for p in before]
    assert cache._sessions["e"].pages[:2].tolist() == [place.get(p, p) for p in shared]
    consistent(cache)
    cache.attend(held, rows(1))
    with pytest.raises(RuntimeError, match="out of date"):
        cache.attend(moving, rows(1))
    count = len(host.of("copy"))
    assert cache.compact() == 0 and len(host.of("copy")) == count
    assert cache.extend(["f"], [1]).block_table.tolist() == [[7]]


def test_compaction_waits_for_rows(host):
    cache = PagedKVCache(6, 1, 16, page_size=8, layers=2)
    grow(cache, "a", 17)
    batch = cache.extend(["b"], [9])
    cache.append(batch, rows(9), rows(9), 0)
    cache.evict_session("a")
    before = state(cache)
    with pytest.raises(RuntimeError, match="append them first"):
        cache.compact()
    with pytest.raises(RuntimeError, match="append them first"):
        cache.resize(3)
    assert state(cache) == before and not host.of("copy")
    assert cache.resize(8) == 0  # nothing of it moves
    cache.append(batch, rows(9), rows(9), 1)
    assert cache.compact() == 2
    consistent(cache)


def test_pools_of_another_size(host):
    cache = PagedKVCache(10, 1, 16, page_size=8, layers=2)
    assert cache.resize(9) == 0 and not host.of("copy")
    for name in "abc":
        grow(cache, name, 20)
    cache.evict_session("a")
    old = list(cache.layers)
    with pytest.raises(MemoryError):
        cache.resize(5)
    with pytest.raises(ValueError):
        cache.resize(0)
    assert cache.layers == old
    held = cache.batch(["b"])
    tables = {n: cache._sessions[n].pages[:3].tolist() for n in "bc"}
    moved = cache.resize(6)
    assert moved == sum(p >= 6 for t in tables.values() for p in t) > 0
    assert cache.num_pages == 6 and not {id(p) for p in old} & {id(p) for p in cache.layers}
    copies = host.of("copy")[-2:]
    assert [e[0] for e in copies] == old and [e[3] for e in copies] == cache.layers
    place = dict(zip(*copies[0][1:3]))
    for n, before in tables.items():
        assert cache._sessions[n].pages[:3].tolist() == [place[p] for p in before]
    consistent(cache)
    if [place[p] for p in tables["b"]] == tables["b"]:
        cache.attend(held, rows(1))
    with pytest.raises(MemoryError):
        cache.extend(["b", "c"], [8, 8])
    assert cache.resize(30) == 0
    cache.extend(["b", "c"], [8, 8])
    consistent(cache)


@pytest.mark.parametrize("what", ["fork", "compact", "resize"])
def test_more_pages_than_one_launch_takes(host, monkeypatch, what):
    """The copies come after the tables were rewritten: pages that are too many for a launch go in several."""
    monkeypatch.setattr(paged, "_COPY_ROWS", 5 * 8)
    cache = PagedKVCache(40, 1, 16, page_size=8, layers=2, tracked=True)
    grow(cache, "a", 8 * 13)
    grow(cache, "b", 8 * 13)
    a, b = (cache._sessions[n].pages[:13].tolist() for n in "ab")
    if what == "fork":
        cache.fork("b", ["c"])
        want = list(zip(b, cache._sessions["c"].pages[:13].tolist()))
    elif what == "compact":
        cache.evict_session("a")
        cache.compact()
        want = list(zip(b, cache._sessions["b"].pages[:13].tolist()))
    else:
        cache.resize(80)
        want = list(zip(a + b, a + b))
    copies = host.of("copy")
    assert all(len(src) == len(dst) <= 5 for _, src, dst, _ in copies)
    for layer in (0, 1):
        half = copies[len(copies) // 2 * layer:len(copies) // 2 * (layer + 1)]
        assert len({id(pages) for pages, *_ in half}) == 1
        assert sorted(p for _, src, dst, _ in half for p in zip(src, dst)) == sorted(want)
    consistent(cache)


def test_pools_of_another_size_stay_on_their_device(host, monkeypatch):
    """The device that the cache was made on, whatever device is current by then."""
    allocate, where = paged.KVPages.allocate, []

    def follow(num_pages, kv_heads, page_size, head_dim, dtype, device, **kw):
        where.append(device)
        return allocate(num_pages, kv_heads, page_size, head_dim, dtype, device, **kw)

    monkeypatch.setattr(paged.KVPages, "allocate", follow)
    cache = PagedKVCache(10, 1, 16, page_size=8, layers=2, device="cuda")
    grow(cache, "a", 20)
    assert where == ["cuda"] * 2
    cache.resize(12)
    assert where[2:] == [cache.device] * 2 and cache.device.type == "cpu"  # (where the stand-ins' pools are)


@pytest.mark.parametrize("what", ["fork", "compact", "resize"])
def test_what_fails_changes_nothing(host, monkeypatch, what):
    cache = PagedKVCache(12, 1, 16, page_size=8)
    for name in "abc":
        grow(cache, name, 20)
    cache.evict_session("a")
    batch = cache.batch(["c"])
    before, users, layers = state(cache), cache._users.copy(), list(cache.layers)
    call = {"fork": lambda: cache.fork("c", ["x", "y"]), "compact": cache.compact, "resize": lambda: cache.resize(7)}[what]
    copies = len(host.of("copy"))
    with monkeypatch.context() as m:
        empty = torch.empty

        def no_device(*args, **kw):
            if "device" in kw:
                raise torch.OutOfMemoryError("out of memory")
            return empty(*args, **kw)

        m.setattr(torch, "empty", no_device)
        with pytest.raises(torch.OutOfMemoryError):
            call()
    with monkeypatch.context() as m, host.on("captured"):
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            call()
    assert state(cache) == before and (cache._users == users).all() and cache.layers == layers and cache.num_pages == 12
    assert len(host.of("copy")) == copies
    cache.attend(batch, rows(1))
    call()
    consistent(cache)


@pytest.mark.parametrize("where", ["pools", "ids"])
def test_no_room_for_other_pools_is_a_memory_error(host, monkeypatch, where):
    """As for pages in use that are too many; torch's own error, which callers of other operators expect, too."""
    cache = PagedKVCache(10, 1, 16, page_size=8, layers=2)
    batch = grow(cache, "a", 20)
    before, layers, users = state(cache), list(cache.layers), cache._users.copy()

    def none_left(*args, **kw):
        raise torch.OutOfMemoryError("out of memory")

    for error in (MemoryError, torch.OutOfMemoryError):
        with monkeypatch.context() as m, pytest.raises(error, match="no room"):
            m.setattr(*((paged.KVPages, "allocate") if where == "pools" else (PagedKVCache, "_upload")), none_left)
            cache.resize(1 << 20)
    assert state(cache) == before and cache.layers == layers and (cache._users == users).all() and cache.num_pages == 10
    cache.attend(batch, rows(1))
    assert cache.resize(20) == 0
    consistent(cache)


def test_bounds_follow_appends_and_evictions(host):
    cache = PagedKVCache(20, 1, 16, page_size=8, layers=2, tracked=True, bounded=True)
    first = cache.extend(["a"], [20])
    second = cache.extend(["a"])
    with pytest.raises(RuntimeError, match="earlier batch"):
        cache.append(second, rows(1), rows(1), 0)
    cache.append(first, rows(20), rows(20), 0)
    pages, lengths, kw = host.of("bounds")[-1]
    assert pages is cache.layers[0] and lengths is first.lengths and kw["since"] is first.before and kw["max_new"] == 20
    cache.append(second, rows(1), rows(1), 0)
    assert host.of("bounds")[-1][2]["max_new"] == 1
    with pytest.raises(RuntimeError, match="already"):
        cache.append(first, rows(20), rows(20), 0)
    cache.append(first, rows(20), rows(20), -1)
    cache.append(second, rows(1), rows(1), 1)
    cache.attend(second, rows(1), 1, blocks=2)
    assert host.of("select") == [(2, {"first": 1, "recent": 1, "max_length": 21})]
    monkey = paged.kv_evict_plan

    def plan(*args, **kw):
        made = monkey(*args, **kw)
        made.lengths = "after"
        return made

    paged.kv_evict_plan = plan
    try:
        cache.evict(["a"], 8, 2)
    finally:
        paged.kv_evict_plan = monkey
    assert [e[:2] for e in host.of("bounds")[-2:]] == [(p, "after") for p in cache.layers]
    plain = PagedKVCache(20, 1, 16, page_size=8)
    batch = grow(plain, "a", 9)
    plain.append(batch, rows(9), rows(9))  # (the same rows again)
    with pytest.raises(ValueError, match="bounded"):
        plain.attend(batch, rows(1), blocks=2)


def test_bounds_of_ragged_steps_are_sized_by_the_longest(host):
    """What one session got at most, not all of them together: the launch has that many workgroups for each."""
    cache = PagedKVCache(60, 1, 16, page_size=8, bounded=True)
    for counts, most in (([20, 1, 7], 20), ([0, 3, 30], 30), ([1, 1, 1], 1), (None, 1), ([0, 0, 0], 0)):
        batch = cache.extend(["a", "b", "c"], counts)
        cache.append(batch, rows(batch.tokens), rows(batch.tokens))
        assert host.of("bounds")[-1][2]["max_new"] == most
    cache.append(cache.extend([]), rows(0), rows(0))
    assert host.of("bounds")[-1][2]["max_new"] == 0


def test_a_selection_needs_a_scale_above_zero(host):
    """Pages are ranked by bounds of q . k: with a scale that turns or levels the scores they say nothing."""
    cache = PagedKVCache(20, 1, 16, page_size=8, bounded=True)
    batch = grow(cache, "a", 20)
    for scale in (-0.125, 0.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            cache.attend(batch, rows(1), scale=scale, blocks=2)
        cache.attend(batch, rows(1), scale=scale)
    assert not host.of("select")
    cache.attend(batch, rows(1), scale=0.125, blocks=2)
    cache.attend(batch, rows(1), blocks=2)
    assert len(host.of("select")) == 2


@pytest.mark.parametrize("seed", range(6))
def test_random_steps_keep_pages_apart(host, seed):
    """What each session's slots hold, carried through every copy: no step of one session changes another's."""
    rng = random.Random(seed)
    tracked = seed % 2 == 1
    cache = PagedKVCache(24, 1, 16, page_size=8, tracked=tracked)
    pool = {}  # (page, row) -> what was written there
    want: dict[str, list] = {}
    seen = 0

    def follow():
        nonlocal seen, pool
        copies = host.of("copy")
        for _, src, dst, into in copies[seen:]:
            before, pool = pool, ({} if into is not None else dict(pool))
            for a, b in zip(src, dst):
                for r in range(8):
                    pool[b, r] = before.get((a, r))
        seen = len(copies)

    for n in range(150):
        names = cache.sessions
        what = rng.choice(["extend"] * 4 + ["fork", "fork", "drop", "compact", "resize"])
        try:
            if what == "extend" or not names:
                name = rng.choice(names + [f"s{n}"])
                count = rng.randint(0, 20)
                batch = cache.extend([name], [count])
                cache.append(batch, rows(count), rows(count))
                at = batch.before[0].item()
                for i in range(count):
                    pool[batch.block_table[0, (at + i) // 8].item(), (at + i) % 8] = (name, n, i)
                want[name] = want.get(name, []) if at else []
                want[name] = want[name] + [(name, n, i) for i in range(count)]
            elif what == "fork":
                name = rng.choice(names)
                new = [f"f{n}-{i}" for i in range(rng.randint(1, 3))]
                cache.fork(name, new)
                for x in new:
                    want[x] = list(want[name])
            elif what == "drop":
                name = rng.choice(names)
                cache.evict_session(name)
            elif what == "compact":
                cache.compact()
                assert cache._free == list(range(cache.num_pages - 1, cache.pages_used - 1, -1))
            else:
                cache.resize(rng.randint(16, 30))
        except MemoryError:
            pass
        follow()
        consistent(cache)
        for name in cache.sessions:
            s = cache._sessions[name]
            held = [pool.get((int(s.pages[j // 8]), j % 8)) for j in range(s.length)]
            assert held == want[name], (n, what, name)
        want = {k: v for k, v in want.items() if k in cache._sessions}
