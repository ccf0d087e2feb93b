"""PagedKVCache: sessions over the paged K/V cache operators, against plain lists of rows in 64 bits."""

from __future__ import annotations

import pytest
import torch

from _paged import DEV, codes, evict64

pytestmark = pytest.mark.gpu


class Plain:
    """The rows of every session, layer and key head, in slot order: (k, v, weight, position)."""

    def __init__(self, layers, kv):
        self.layers, self.kv, self.rows, self.seen = layers, kv, {}, {}

    def append(self, name, layer, k, v, int8):
        rows = self.rows.setdefault(name, [[[] for _ in range(self.kv)] for _ in range(self.layers)])[layer]
        for i in range(k.shape[0]):
            for h in range(self.kv):
                pair = []
                for t in (k, v):
                    x = t[i, h]
                    if int8:
                        c, s = codes(x.float())
                        x = c.double() * s.double()
                    pair.append(x.double())
                rows[h].append([*pair, 0.0, self.seen.get(name, 0) + i])

    def attend(self, name, layer, q):
        """``(out, sum p |v|)`` and the weights added."""
        group = q.shape[0] // self.kv
        out, mass = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        for i in range(q.shape[0]):
            rows = self.rows[name][layer][i // group]
            k, v = (torch.stack([r[x] for r in rows]) for x in (0, 1))
            p = torch.softmax(k @ q[i].double() * q.shape[1] ** -0.5, 0)
            out[i], mass[i] = p @ v, p @ v.abs()
            for r, w in zip(rows, p.tolist()):
                r[2] += w
        return out, mass


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8])
def test_sessions_against_plain_rows(dtype):
    """Prompts of several lengths, then tokens, sessions that come and go, cuts to a budget, two layers."""
    from cortex.cache import PagedKVCache

    layers, kv, heads, dim = 2, 2, 6, 32
    g = torch.Generator().manual_seed(5)
    cache = PagedKVCache(64, kv, dim, page_size=8, dtype=dtype, layers=layers, tracked=True)
    x = torch.float32 if dtype == torch.float32 else torch.bfloat16
    plain = Plain(layers, kv)
    names = ["a", "b", "c"]
    half = 0.0 if dtype == torch.float32 else 2.0 ** -8
    for step in range(24):
        active = names if step % 5 else names[:2]
        counts = [17, 0, 33] if step == 0 else [1] * len(active) if step % 3 else [2, 0, 1][:len(active)]
        if step == 0:
            active = names
        batch = cache.extend(active, counts)
        assert batch.lengths.tolist() == [cache.length(n) for n in active]
        for layer in range(layers):
            k, v = (torch.randn(sum(counts), kv, dim, generator=g).to(x) for _ in range(2))
            cache.append(batch, k.to(DEV), v.to(DEV), layer)
            at = 0
            for n, c in zip(active, counts):
                plain.append(n, layer, k[at:at + c], v[at:at + c], dtype == torch.int8)
                at += c
            q = torch.randn(len(active), heads, dim, generator=g).to(x)
            got = cache.attend(batch, q.to(DEV), layer).double().cpu()
            for i, n in enumerate(active):
                if not cache.length(n):
                    assert (got[i] == 0).all()
                    continue
                want, mass = plain.attend(n, layer, q[i])
                # 2^-15 for the probabilities, 2^-8 for the result (bf16, int8), fp32 sums below 1e-4
                assert ((got[i] - want).abs() <= (2.0 ** -15 + 1e-4) * mass + half * want.abs()).all(), (step, n)
        for n, c in zip(active, counts):
            plain.seen[n] = plain.seen.get(n, 0) + c
        if step % 6 == 5:  # (the plain side follows the kernel's weights, which differ from its own by rounding)
            over = [n for n in names if cache.length(n) > 20]
            table = cache.batch(names).block_table.cpu()
            kept = {}
            for layer in range(layers):
                w, pos = cache.layers[layer].weight.cpu(), cache.layers[layer].position.cpu()
                for n in over:
                    slots = torch.arange(cache.length(n))
                    at = table[names.index(n)][slots // 8].long(), slice(None), slots % 8
                    for h in range(kv):
                        rows = plain.rows[n][layer][h]
                        torch.testing.assert_close(w[at][:, h].double(), torch.tensor([r[2] for r in rows], dtype=torch.float64),
                                                   rtol=1e-4, atol=1e-6)
                        assert pos[at][:, h].tolist() == [r[3] for r in rows]
                        kept[n, layer, h] = evict64(w[at][:, h], pos[at][:, h], len(slots), 20, 5)
            free = cache.num_pages - cache.pages_used
            freed = cache.evict(names, 20, 5)
            assert cache.num_pages - cache.pages_used == free + freed
            for (n, layer, h), (dst, src) in kept.items():
                rows = plain.rows[n][layer][h]
                for d, s in zip(dst, src):
                    rows[d] = rows[s]
                del rows[20:]
                assert cache.length(n) == 20
    assert cache.evict_session("a") > 0 and cache.length("a") == 0 and cache.evict_session("a") == 0


def test_pages_come_from_the_least_recently_used_session():
    from cortex.cache import PagedKVCache

    cache = PagedKVCache(6, 1, 16, page_size=8)
    cache.extend(["a", "b"], [16, 8])
    cache.extend(["c"], [16])
    assert cache.pages_used == 5 and cache.sessions == ["a", "b", "c"]
    old = cache.batch(["a", "b"])  # now c is the oldest
    assert cache.sessions == ["c", "a", "b"]
    rows = torch.ones(24, 1, 16, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(MemoryError):
        cache.extend(["b", "d"], [0, 41])  # a and c and what is free hold five pages
    assert cache.sessions == ["c", "a", "b"] and cache.pages_used == 5
    new = cache.extend(["b", "d"], [0, 24])
    assert cache.sessions == ["a", "b", "d"] and cache.pages_used == 6 and cache.length("c") == 0
    cache.append(new, rows, rows)
    cache.attend(old, torch.ones(2, 1, 16, dtype=torch.bfloat16, device=DEV))  # neither a nor b was touched
    newer = cache.extend(["d"], [8])
    assert cache.sessions == ["b", "d"]
    q = torch.ones(2, 1, 16, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="out of date"):
        cache.attend(old, q)  # a is gone
    cache.attend(new, q)
    cache.append(newer, rows[:8], rows[:8])
    assert (cache.attend(cache.batch(["d"]), q[:1]) == 1).all()


def test_pages_come_from_the_oldest_session():
    from cortex.cache import PagedKVCache

    cache = PagedKVCache(6, 1, 16, page_size=8)
    rows = torch.ones(24, 1, 16, dtype=torch.bfloat16, device=DEV)
    for names, counts in [(["a", "b"], [16, 8]), (["c"], [16])]:
        cache.append(cache.extend(names, counts), rows[:sum(counts)], rows[:sum(counts)])
    assert cache.pages_used == 5 and cache.sessions == ["a", "b", "c"]
    old = cache.batch(["a", "b"])  # now c is the oldest
    assert cache.sessions == ["c", "a", "b"]
    with pytest.raises(MemoryError):
        cache.extend(["b", "d"], [0, 41])  # a and c and what is free hold five pages
    assert cache.sessions == ["c", "a", "b"] and cache.pages_used == 5
    new = cache.extend(["b", "d"], [0, 24])
    assert cache.sessions == ["a", "b", "d"] and cache.pages_used == 6 and cache.length("c") == 0
    cache.append(new, rows * 2, rows * 2)
    q = torch.ones(2, 1, 16, dtype=torch.bfloat16, device=DEV)
    assert (cache.attend(old, q) == 1).all()  # neither a nor b was touched
    newer = cache.extend(["d"], [8])
    assert cache.sessions == ["b", "d"]
    with pytest.raises(RuntimeError, match="out of date"):
        cache.attend(old, q)  # a is gone
    assert cache.attend(new, q).tolist() == [[[1.0] * 16], [[2.0] * 16]]
    with pytest.raises(RuntimeError, match="no rows in layer"):
        cache.attend(cache.batch(["d"]), q[:1])  # its last page is a's
    cache.append(newer, rows[:8] * 2, rows[:8] * 2)
    assert (cache.attend(cache.batch(["d"]), q[:1]) == 2).all()


def test_slots_of_earlier_batches_are_not_read_without_rows():
    from cortex.cache import PagedKVCache

    cache = PagedKVCache(8, 1, 16, page_size=8, layers=2, tracked=True)
    rows = torch.randn(20, 1, 16, device=DEV).bfloat16()
    q = torch.randn(1, 2, 16, device=DEV).bfloat16()
    first = cache.extend(["a"], [20])
    cache.append(first, rows, rows, 0)
    second = cache.extend(["a"])
    for layer in range(2):
        cache.append(second, rows[:1], rows[:1], layer)
    cache.attend(second, q, 0)
    before = cache.layers[1].weight.clone()
    for batch in (second, cache.batch(["a"])):
        with pytest.raises(RuntimeError, match="no rows in layer 1"):
            cache.attend(batch, q, 1)
    assert torch.equal(cache.layers[1].weight, before)
    cache.append(first, rows, rows, 1)
    # (the weights of layer 0 are of two calls, those of layer 1 of one: the results do not depend on them)
    assert torch.equal(cache.attend(second, q, 0), cache.attend(second, q, 1))


def test_cut_sessions_refuse_older_batches():
    from cortex.cache import PagedKVCache

    cache = PagedKVCache(32, 2, 16, page_size=8, tracked=True)
    rows = torch.randn(60, 2, 16, device=DEV).bfloat16()
    batch = cache.extend(["a", "b"], [40, 20])
    cache.append(batch, rows, rows)
    q = torch.randn(2, 2, 16, device=DEV).bfloat16()
    cache.attend(batch, q)
    assert cache.evict(["a", "b"], 24, 4) == 2 and cache.length("a") == 24 and cache.length("b") == 20
    with pytest.raises(RuntimeError, match="out of date"):
        cache.attend(batch, q)
    cache.attend(cache.batch(["a", "b"]), q)
    assert cache.evict(["a", "b"], 24, 4) == 0


def test_slots_without_rows_are_not_read():
    """Slots of new tokens hold what the pages' last owner left there until the rows are appended."""
    from cortex.cache import PagedKVCache

    cache = PagedKVCache(8, 1, 16, page_size=8, layers=2, tracked=True)
    rows = torch.randn(20, 1, 16, device=DEV).bfloat16()
    q = torch.randn(1, 2, 16, device=DEV).bfloat16()
    first = cache.extend(["a"], [20])
    cache.append(first, rows, rows, 0)
    cache.attend(first, q, 0)
    for layer in (1, -1):
        with pytest.raises(RuntimeError, match="layer"):
            cache.attend(first, q, layer)
    second = cache.extend(["a"])
    for layer in (0, -1):
        cache.append(second, rows[:1], rows[:1], layer)
    with pytest.raises(RuntimeError, match="without rows"):
        cache.evict(["a"], 8, 2)  # layer 1 lacks the rows of the first batch
    assert cache.length("a") == 21 and cache.pages_used == 3
    assert cache.evict(["a"], 21, 2) == 0  # nothing to cut
    cache.append(first, rows, rows, 1)
    cache.attend(second, q, 1)
    assert cache.evict(["a"], 8, 2) == 2
    cache.attend(cache.batch(["a"]), q, 1)
    third = cache.extend(["a"])
    for layer in (0, 1):
        cache.append(third, rows[:1], rows[:1], layer)
    assert cache.evict(["a"], 8, 2) == 1


def test_streams_follow_each_other():
    """Appends on one stream and attention on another, without a synchronisation by the caller."""
    from cortex.cache import PagedKVCache

    g = torch.Generator(DEV).manual_seed(3)
    rows = [torch.randn(2, 4, 64, generator=g, device=DEV).bfloat16() for _ in range(200)]
    q = torch.randn(2, 8, 64, generator=g, device=DEV).bfloat16()

    def play(streams):
        cache = PagedKVCache(64, 4, 64)
        out = []
        for i, r in enumerate(rows):
            with torch.cuda.stream(streams[0]):
                batch = cache.extend(["x", "y"])
                cache.append(batch, r, r)
            if i % 9 == 0:
                with torch.cuda.stream(streams[1]):
                    out.append(cache.attend(batch, q))
            del batch
        torch.cuda.synchronize()
        return torch.stack(out)

    one = torch.cuda.current_stream()
    torch.cuda.synchronize()
    assert torch.equal(play([one, one]), play([torch.cuda.Stream(), torch.cuda.Stream()]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_first_rows_on_another_stream_outlast_the_fill(dtype):
    """The pools' zero fills wait behind other work of their stream while the first rows come on another one."""
    from cortex.cache import PagedKVCache

    rows = torch.randn(40, 2, 64, device=DEV).bfloat16()
    busy = torch.empty(1 << 30, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(40):  # 4 GiB each
        busy.fill_(i)
    cache = PagedKVCache(64, 2, 64, page_size=8, dtype=dtype, layers=2, tracked=True)
    with torch.cuda.stream(side):
        batch = cache.extend(["a"], [40])
        for layer in range(2):
            cache.append(batch, rows, rows, layer)
    torch.cuda.synchronize()
    slots = torch.arange(40)
    at = batch.block_table[0].cpu()[slots // 8].long(), slice(None), slots % 8
    for p in cache.layers:
        want = rows.cpu().double()
        for pool, scale in ((p.k, p.k_scale), (p.v, p.v_scale)):
            got = pool.cpu()[at].double()
            if dtype == torch.int8:
                c, s = codes(want.float())
                assert torch.equal(got, c.double()) and torch.equal(scale.cpu()[at], s)
            else:
                assert torch.equal(got, want)
        assert p.position.cpu()[at].tolist() == [[i, i] for i in range(40)]


def test_refusals():
    from cortex.cache import PagedKVCache

    for kw in [{"num_pages": 0}, {"layers": 0}, {"page_size": 12}, {"head_dim": 20}, {"dtype": torch.float16}]:
        with pytest.raises(ValueError):
            PagedKVCache(**{"num_pages": 4, "kv_heads": 1, "head_dim": 16, **kw})
    cache = PagedKVCache(4, 1, 16, page_size=8)
    for names, counts in [(["a", "a"], None), ("ab", None), (["a"], [1, 2]), (["a"], [-1])]:
        with pytest.raises(ValueError):
            cache.extend(names, counts)
    with pytest.raises(KeyError):
        cache.batch(["a"])
    with pytest.raises(ValueError):
        cache.evict([], 4, 1)  # not tracked
    batch = cache.extend(["a"])
    with pytest.raises(ValueError):
        cache.append(batch, *[torch.zeros(2, 1, 16, dtype=torch.bfloat16, device=DEV)] * 2)
    tracked = PagedKVCache(4, 1, 16, page_size=8, tracked=True)
    for budget, recent in [(0, 0), (4, 5), (4, -1)]:
        with pytest.raises(ValueError):
            tracked.evict([], budget, recent)
    with pytest.raises(KeyError):
        tracked.evict(["a"], 4, 1)
    assert tracked.evict([], 4, 1) == 0
    empty = cache.extend([])
    assert cache.attend(empty, torch.zeros(0, 2, 16, dtype=torch.bfloat16, device=DEV)).shape == (0, 2, 16)
