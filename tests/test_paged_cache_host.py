"""What PagedKVCache does on the host, on the CPU: streams, events and operators are stand-ins that write down what they
were asked for."""

from __future__ import annotations

import contextlib
from types import SimpleNamespace

import pytest
import torch

from cortex.cache import PagedKVCache, paged


class Stream:
    def __init__(self, log, name):
        self.log, self.name = log, name

    def wait_event(self, event):
        self.log.append(("wait", self.name, event.on))

    def __repr__(self):
        return self.name


class Host:
    """The stand-ins: ``log`` has what was asked, in order; ``on(name)`` makes a stream the current one."""

    def __init__(self, patch):
        self.log = log = []
        self.streams: dict[str, Stream] = {}
        self.current = self.stream("first")
        host = self

        class Event:
            on = None

            def record(self, stream):
                self.on = stream.name

            def synchronize(self):
                pass

        def allocate(num_pages, kv_heads, page_size, head_dim, dtype, device, *, tracked=False):
            shape = (num_pages, kv_heads, page_size)
            made = {n: torch.zeros(*shape, head_dim) for n in ("k", "v")}
            for n, there in [("k_scale", False), ("v_scale", False), ("weight", tracked), ("position", tracked)]:
                made[n] = torch.zeros(shape) if there else None
            return SimpleNamespace(**made, device=torch.device("cpu"), page_size=page_size, kv_heads=kv_heads)

        def plan(pages, table, lengths, budget, recent, **kw):
            log.append(("plan", pages))
            return SimpleNamespace(of=pages)

        patch.setattr(torch.cuda, "Event", Event)
        patch.setattr(torch.cuda, "current_stream", lambda device=None: host.current)
        patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        patch.setattr(torch.Tensor, "pin_memory", lambda t: t, raising=False)
        patch.setattr(torch.Tensor, "record_stream", lambda t, s: log.append(("record", s.name, t)), raising=False)
        patch.setattr(paged.KVPages, "allocate", allocate)
        patch.setattr(paged, "paged_kv_append", lambda pages, *a, **kw: log.append(("append", pages)))
        patch.setattr(paged, "paged_attention", lambda q, pages, table, lengths, **kw: log.append(("attend", pages)))
        patch.setattr(paged, "kv_evict_plan", plan)
        patch.setattr(paged, "kv_evict_apply", lambda pages, table, plan: log.append(("apply", pages)))

    def stream(self, name):
        return self.streams.setdefault(name, Stream(self.log, name))

    @contextlib.contextmanager
    def on(self, name):
        before, self.current = self.current, self.stream(name)
        yield
        self.current = before

    def of(self, what):
        return [e[1:] for e in self.log if e[0] == what]


@pytest.fixture
def host(monkeypatch):
    return Host(monkeypatch)


def rows(n):
    return torch.zeros(n, 1, 16)


def test_the_first_call_on_another_stream_waits_for_the_fill(host):
    """The pools are zeroed on the stream that is current where the cache is made: a first call on another one waits for
    that, and the pools are recorded for it."""
    with host.on("made"):
        cache = PagedKVCache(8, 1, 16, page_size=8, layers=2, tracked=True)
    with host.on("side"):
        batch = cache.extend(["a"], [3])
        assert host.of("wait") == [("side", "made")]
        cache.append(batch, rows(3), rows(3), 1)
    assert host.of("wait") == [("side", "made")]
    held = [t for name, t in host.of("record") if name == "side"]
    for p in cache.layers:
        assert all(any(t is x for x in held) for t in (p.k, p.v, p.weight, p.position))
    with host.on("made"):
        cache.attend(cache.extend(["b"], [0]), rows(1))
    assert host.of("wait") == [("side", "made"), ("made", "side")]


def test_calls_on_the_stream_of_the_fill_wait_for_nothing(host):
    cache = PagedKVCache(8, 1, 16, page_size=8)
    batch = cache.extend(["a"], [3])
    cache.append(batch, rows(3), rows(3))
    cache.attend(batch, rows(1))
    assert not host.of("wait") and not host.of("record")


def test_attend_refuses_slots_of_earlier_batches_without_rows(host):
    """Every slot that a call reads must have its row in that layer, not only those of the batch's own tokens."""
    cache = PagedKVCache(8, 1, 16, page_size=8, layers=2, tracked=True)
    first = cache.extend(["a"], [20])
    cache.append(first, rows(20), rows(20), 0)
    second = cache.extend(["a"])
    for layer in (0, 1):
        cache.append(second, rows(1), rows(1), layer)
    cache.attend(second, rows(1), 0)
    for layer in (1, -1):  # what the pages' last owner left there is in the first 20
        with pytest.raises(RuntimeError, match="no rows in layer"):
            cache.attend(second, rows(1), layer)
        with pytest.raises(RuntimeError, match="no rows in layer"):
            cache.attend(cache.batch(["a"]), rows(1), layer)
    assert len(host.of("attend")) == 1
    cache.append(first, rows(20), rows(20), -1)
    for batch in (first, second, cache.batch(["a"])):
        for layer in (0, 1, -1, -2):
            cache.attend(batch, rows(1), layer)


def test_attend_refuses_sessions_that_were_only_extended(host):
    cache = PagedKVCache(8, 1, 16, page_size=8, tracked=True)
    given = cache.extend(["a"], [5])
    cache.append(given, rows(5), rows(5))
    missing = cache.extend(["b"], [5])
    for batch in (missing, cache.batch(["b"]), cache.batch(["a", "b"]), cache.extend(["b", "c"], [0, 0])):
        with pytest.raises(RuntimeError, match="no rows in layer"):
            cache.attend(batch, rows(len(batch.sessions)))
    both = cache.batch(["a", "b"])
    cache.attend(cache.batch(["a"]), rows(1))  # the others are not in the call
    cache.append(missing, rows(5), rows(5))
    cache.attend(both, rows(2))
    # one call for several sessions is one batch: its rows come together
    joint = cache.extend(["a", "b"], [1, 2])
    with pytest.raises(RuntimeError, match="no rows in layer"):
        cache.attend(cache.batch(["a"]), rows(1))
    cache.attend(both, rows(2))  # made before: it reads none of the new slots
    cache.append(joint, rows(3), rows(3))
    cache.attend(cache.batch(["a"]), rows(1))


def test_a_dropped_session_starts_anew(host):
    """A batch that is given up leaves slots without rows: dropping its session frees them."""
    cache = PagedKVCache(8, 1, 16, page_size=8)
    given_up = cache.extend(["a"], [5])
    assert cache.evict_session("a") == 1
    batch = cache.extend(["a"], [2])
    cache.append(batch, rows(2), rows(2))
    cache.attend(batch, rows(1))
    cache.attend(cache.batch(["a"]), rows(1))
    with pytest.raises(RuntimeError, match="out of date"):
        cache.append(given_up, rows(5), rows(5))


def test_steps_keep_no_record_of_what_is_complete(host):
    """What a batch and a session hold about missing rows does not grow with the steps taken."""
    cache = PagedKVCache(64, 1, 16, page_size=8, layers=2)
    for _ in range(100):
        batch = cache.extend(["a", "b"])
        for layer in (0, 1):
            cache.append(batch, rows(2), rows(2), layer)
            cache.attend(batch, rows(2), layer)
    assert len(batch.needs) == 1 and all(len(s.pending) <= 2 for s in cache._sessions.values())
    assert not cache.batch(["a", "b"]).needs


def state(cache):  # (of the records of missing rows those that miss some)
    return {"free": list(cache._free), "order": cache.sessions, "epoch": cache._epoch,
            "sessions": {n: (s.pages[:s.used].tolist(), s.length, s.seen, s.version, [set(f) for f in s.pending if len(f) < len(cache.layers)])
                         for n, s in cache._sessions.items()}}


@pytest.mark.parametrize("fails", ["memory of the device", "pinned memory", "copy"])
def test_an_extend_that_fails_changes_nothing(host, monkeypatch, fails):
    """Neither the sessions of the call nor those that would have given way."""
    cache = PagedKVCache(700, 1, 16, page_size=8)
    for name, count in [("a", 8 * 600), ("b", 8 * 90), ("c", 9)]:
        batch = cache.extend([name], [count])
        cache.append(batch, rows(count), rows(count))
    pending = cache.extend(["c"])
    before = state(cache)

    def out_of_memory(*args, **kw):
        raise torch.OutOfMemoryError("out of memory")

    with monkeypatch.context() as m:
        if fails == "pinned memory":
            m.setattr(torch.Tensor, "pin_memory", out_of_memory, raising=False)
            cache._stage = cache._stage[:1]
        elif fails == "copy":
            m.setattr(torch.Tensor, "copy_", out_of_memory)
        else:
            empty = torch.empty

            def no_device(*args, **kw):
                return out_of_memory() if "device" in kw else empty(*args, **kw)

            m.setattr(torch, "empty", no_device)
        for names, counts in [(["c"], [4000]), (["d", "b"], [4095, 1]), (["d"], [0]), (["c", "d"], [1, 8 * 650])]:
            with pytest.raises(torch.OutOfMemoryError):
                cache.extend(names, counts)
            assert state(cache) == before
    cache.append(pending, rows(1), rows(1))
    batch = cache.extend(["d", "c"], [4000, 1])
    assert cache.sessions == ["b", "d", "c"] and cache.length("c") == 11 and batch.positions[-1] == 10
    assert sorted(cache._free + [p for s in cache._sessions.values() for p in s.pages[:s.used].tolist()]) == list(range(700))


def test_an_eviction_that_fails_moves_nothing(host, monkeypatch):
    """The plans of all layers are made before the first row of any layer moves."""
    cache = PagedKVCache(8, 1, 16, page_size=8, layers=3, tracked=True)
    batch = cache.extend(["a"], [20])
    for layer in range(3):
        cache.append(batch, rows(20), rows(20), layer)
    before = state(cache)
    plan = paged.kv_evict_plan
    with monkeypatch.context() as m:
        def out_of_memory(pages, *args, **kw):
            if pages is cache.layers[2]:
                raise torch.OutOfMemoryError("out of memory")
            return plan(pages, *args, **kw)

        m.setattr(paged, "kv_evict_plan", out_of_memory)
        with pytest.raises(torch.OutOfMemoryError):
            cache.evict(["a"], 8, 2)
    assert not host.of("apply") and state(cache) == before
    cache.attend(batch, rows(1))  # still holds
    assert cache.evict(["a"], 8, 2) == 2
    assert host.of("apply") == [(p,) for p in cache.layers]


def test_steps_are_not_captured(host, monkeypatch):
    """A graph would replay the copy of a buffer that has moved on, or wait for work outside of it."""
    cache = PagedKVCache(8, 1, 16, page_size=8)
    batch = cache.extend(["a"], [5])
    cache.append(batch, rows(5), rows(5))
    before = state(cache)
    with monkeypatch.context() as m, host.on("captured"):
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: host.current.name == "captured")
        for call in (lambda: cache.extend(["a"]), lambda: cache.batch(["a"]), lambda: cache.attend(batch, rows(1)),
                     lambda: cache.append(batch, rows(5), rows(5))):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert state(cache) == before and not host.of("wait") and not host.of("record")
    cache.attend(batch, rows(1))
