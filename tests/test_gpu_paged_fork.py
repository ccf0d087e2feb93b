"""PagedKVCache on the GPU: forks, compaction, pools of another size and selected pages, against the rows that each session
was given."""

from __future__ import annotations

import random

import pytest
import torch

from _blocks import select64
from _paged import DEV, attention64, codes

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8}
KV, HEADS, DIM, PAGE = 2, 6, 32, 8


class Mirror:
    """A cache, and beside it the rows of every session by layer."""

    def __init__(self, dtype, seed, *, layers=2, num_pages=60, **kw):
        from cortex.cache import PagedKVCache

        self.dtype, self.g = DTYPES[dtype], torch.Generator().manual_seed(seed)
        self.cache = PagedKVCache(num_pages, KV, DIM, page_size=PAGE, dtype=self.dtype, layers=layers, **kw)
        self.rows = {}

    def values(self, x):
        """Rows as the pages hold them."""
        if self.dtype == torch.int8:
            c, s = codes(x.float())
            return c.float() * s[..., None]
        return x.to(self.dtype)

    def extend(self, names, counts=None):
        batch = self.cache.extend(names, counts)
        counts = [1] * len(names) if counts is None else counts
        x = torch.float32 if self.dtype == torch.float32 else torch.bfloat16
        known = set(self.cache.sessions)
        self.rows = {n: r for n, r in self.rows.items() if n in known}
        for layer in range(len(self.cache.layers)):
            k, v = (torch.randn(sum(counts), KV, DIM, generator=self.g).to(x) for _ in range(2))
            self.cache.append(batch, k.to(DEV), v.to(DEV), layer)
            at = 0
            for n, c in zip(names, counts):
                held = self.rows.setdefault(n, [[[], []] for _ in self.cache.layers])[layer]
                held[0].append(self.values(k[at:at + c])), held[1].append(self.values(v[at:at + c]))
                at += c
        return batch

    def fork(self, name, names):
        self.cache.fork(name, names)
        for n in names:
            self.rows[n] = [[list(k), list(v)] for k, v in self.rows[name]]
        known = set(self.cache.sessions)
        self.rows = {n: r for n, r in self.rows.items() if n in known}

    def check(self, names, layer, *, blocks=None):
        """Attention of the sessions as they stand."""
        batch = self.cache.batch(names)
        q = torch.randn(len(names), HEADS, DIM, generator=self.g).to(self.cache.layers[layer].query_dtype)
        got = self.cache.attend(batch, q.to(DEV), layer, accumulate=False, blocks=blocks).double().cpu()
        for i, n in enumerate(names):
            k, v = (torch.cat(x) for x in self.rows[n][layer])
            length = self.cache.length(n)
            assert k.shape[0] == length
            for h in range(KV):
                group = HEADS // KV
                keep = torch.arange(length)
                if blocks is not None and length:
                    count = -(-length // PAGE)
                    parts = [k[j * PAGE:(j + 1) * PAGE, h].double() for j in range(count)]
                    bounds = torch.stack([torch.stack([p.amax(0), p.amin(0)]) for p in parts])
                    chosen = select64(list(range(count)), bounds.numpy(), q[i, h * group:(h + 1) * group].double().numpy(),
                                      length, PAGE, blocks, 1, 1, count)
                    keep = torch.cat([torch.arange(j * PAGE, min(length, (j + 1) * PAGE)) for j in chosen])
                one = type("", (), {})()
                one.kv_heads, one.lens = 1, [keep.shape[0]]
                one.k, one.v = k[keep, h:h + 1][None].transpose(1, 2), v[keep, h:h + 1][None].transpose(1, 2)
                one.at = lambda b, slots: (torch.zeros_like(slots), slice(None), slots)
                want, _, tol, _ = attention64(one, q[i:i + 1, h * group:(h + 1) * group])
                off = (got[i:i + 1, h * group:(h + 1) * group] - want).abs()
                assert (off <= tol).all(), (n, layer, h, float((off / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tracked", [False, True], ids=["shared", "tracked"])
def test_forks_go_on_by_themselves(dtype, tracked):
    m = Mirror(dtype, 1, tracked=tracked, bounded=True)
    m.extend(["a", "z"], [29, 3])
    m.fork("a", ["b", "c"])
    m.check(["a", "b", "c", "z"], 0)
    for _ in range(6):
        m.extend(["a", "b", "c"])
        m.check(["b", "a", "z", "c"], 1)
    m.extend(["c"], [17])
    m.fork("c", ["d"])
    m.extend(["d", "a"], [2, 9])
    for layer in (0, 1):
        m.check(["a", "b", "c", "d", "z"], layer)
        m.check(["a", "b", "c", "d", "z"], layer, blocks=3)
    m.cache.evict_session("a")
    m.cache.compact()
    m.cache.resize(45)
    m.extend(["b", "e"], [1, 20])
    for layer in (0, 1):
        m.check(["b", "c", "d", "e", "z"], layer)
        m.check(["b", "c", "d", "e", "z"], layer, blocks=2)


@pytest.mark.parametrize("seed", range(4))
def test_random_sessions(seed):
    rng = random.Random(seed)
    m = Mirror(["bf16", "fp32", "int8", "bf16"][seed], seed, num_pages=40, bounded=True, tracked=seed == 3)
    for n in range(60):
        names = m.cache.sessions
        what = rng.choice(["extend"] * 4 + ["fork", "drop", "compact", "resize"])
        try:
            if what == "extend" or not names:
                some = sorted({rng.choice(names + [f"s{n}"]) for _ in range(3)})
                m.extend(some, [rng.randint(0, 24) for _ in some])
            elif what == "fork":
                m.fork(rng.choice(names), [f"f{n}"])
            elif what == "drop":
                m.cache.evict_session(rng.choice(names))
            elif what == "compact":
                m.cache.compact()
            else:
                m.cache.resize(rng.randint(30, 50))
        except MemoryError:
            pass
        names = m.cache.sessions
        if names:
            m.check(names, n % 2, blocks=None if n % 3 else rng.randint(2, 5))


def test_the_bounds_of_an_evicted_session():
    """After an eviction every page's bounds are those of the keys that are left."""
    from cortex.kernels.paged_kv import kv_block_bounds

    m = Mirror("bf16", 5, tracked=True, bounded=True)
    batch = m.extend(["a", "b"], [90, 30])
    q = torch.randn(2, HEADS, DIM, generator=m.g).bfloat16().to(DEV)
    for layer in (0, 1):
        m.cache.attend(batch, q, layer)
    assert m.cache.evict(["a", "b"], 44, 4) == 6
    batch = m.cache.batch(["a", "b"])
    for pages in m.cache.layers:
        for s, n in (("a", 44), ("b", 30)):
            ids = m.cache._sessions[s].pages[:-(-n // PAGE)].tolist()
            for j, p in enumerate(ids):
                k = pages.k[p, :, :min(PAGE, n - j * PAGE)].float()
                assert torch.equal(pages.bounds[p, :, 0].float(), k.amax(1)) and torch.equal(pages.bounds[p, :, 1].float(), k.amin(1))
    out = m.cache.attend(batch, q, 0, blocks=3)
    assert out.isfinite().all()


def test_forks_on_another_stream():
    m = Mirror("bf16", 6, bounded=True)
    m.extend(["a"], [30])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        m.fork("a", ["b"])
        m.extend(["b"], [4])
    m.check(["a", "b"], 0)
    with torch.cuda.stream(side):
        m.cache.evict_session("a")
        m.cache.resize(20)
        m.check(["b"], 1, blocks=2)
    m.check(["b"], 1)
    m.cache.compact()
    m.check(["b"], 0)
