"""Copies of pages, bounds and selections of pages bit for bit, and attention over selected pages within the bounds of
tests/_paged.py, against plain computations in 64 bits."""

from __future__ import annotations

import pytest
import torch

from _blocks import BoundedCache, select64
from _paged import DEV, attention64

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8}


def check(got, want, tol, what):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max())} times allowed"


def same(a, b):
    """Equal, NaN where the other has one."""
    return torch.equal(torch.nan_to_num(a.double().cpu(), nan=12345.0), torch.nan_to_num(b.double().cpu(), nan=12345.0))


# ------------------------------------------------------------------------------- copies


ARRAYS = ("k", "v", "k_scale", "v_scale", "weight", "position", "bounds")


def filled(pages, seed):
    """Every array of the pages with numbers of its own."""
    g = torch.Generator().manual_seed(seed)
    for name in ARRAYS:
        t = getattr(pages, name)
        if t is not None:
            t.copy_(torch.randint(-100, 100, t.shape, generator=g).to(t.dtype))
    return {n: getattr(pages, n).clone() for n in ARRAYS if getattr(pages, n) is not None}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,page,dim", [(1, 8, 16), (3, 16, 48), (8, 16, 128), (2, 1024, 64), (12, 64, 112), (5, 32, 96)])
@pytest.mark.parametrize("extra", ["none", "all"])
def test_copies(dtype, kv_heads, page, dim, extra):
    from cortex.kernels.paged_kv import KVPages, kv_copy_pages

    pages = KVPages.allocate(23, kv_heads, page, dim, DTYPES[dtype], DEV, tracked=extra == "all", bounded=extra == "all")
    want = filled(pages, dim)
    order = torch.randperm(23, generator=torch.Generator().manual_seed(page)).int()
    for n in (0, 1, 2, 11):
        src, dst = order[:n].to(DEV), order[11:11 + n].to(DEV)
        kv_copy_pages(pages, src, dst)
        for name, t in want.items():
            t[dst.long()] = t[src.long()]
            assert torch.equal(getattr(pages, name), t), name
    # one page to several, and a page onto itself
    src, dst = torch.tensor([3, 3, 3, 5], dtype=torch.int32, device=DEV), torch.tensor([1, 2, 0, 5], dtype=torch.int32, device=DEV)
    kv_copy_pages(pages, src, dst)
    for name, t in want.items():
        t[dst.long()] = t[src.long()]
        assert torch.equal(getattr(pages, name), t), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pages", [1, 700, 4000])
def test_copies_of_few_and_many_pages(dtype, pages):
    from cortex.kernels.paged_kv import KVPages, kv_copy_pages

    pool = KVPages.allocate(2 * pages, 2, 32, 64, DTYPES[dtype], DEV, tracked=True)
    want = filled(pool, pages)
    order = torch.randperm(2 * pages, generator=torch.Generator().manual_seed(1)).int().to(DEV)
    kv_copy_pages(pool, order[:pages], order[pages:])
    for name, t in want.items():
        t[order[pages:].long()] = t[order[:pages].long()]
        assert torch.equal(getattr(pool, name), t), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["head", "row", "gap"])
def test_copies_between_pools_and_layouts(dtype, layout):
    from cortex.kernels.paged_kv import KVPages, kv_copy_pages

    c = BoundedCache([100, 31], 3, 64, 16, DTYPES[dtype], layout=layout, tracked=True)
    before = {n: getattr(c.pages, n).clone() for n in ARRAYS if getattr(c.pages, n) is not None}
    other = KVPages.allocate(40, 3, 16, 64, DTYPES[dtype], DEV, tracked=True, bounded=True)
    want = filled(other, 1)
    src = torch.arange(c.num, dtype=torch.int32, device=DEV)
    dst = torch.randperm(40, generator=c.g)[:c.num].int().to(DEV)
    kv_copy_pages(c.pages, src, dst, into=other)
    for name, t in want.items():
        t[dst.long()] = before[name]
        assert same(getattr(other, name), t), name
        assert same(getattr(c.pages, name), before[name]), name
    back = torch.roll(src, 1)
    kv_copy_pages(other, dst, back, into=c.pages)
    for name, t in before.items():
        t[back.long()] = want[name][dst.long()]
        assert same(getattr(c.pages, name), t), name
    if layout == "gap":  # what lies between the rows
        assert (c.gk._base[:, 0] == 77).all() and (c.gk._base[:, 1, :, :, :16] == 77).all()


def test_copies_of_pages_that_are_not_there():
    from cortex.kernels.paged_kv import KVPages, kv_copy_pages

    small = KVPages.allocate(4, 1, 8, 16, torch.float32, DEV)
    large = KVPages.allocate(9, 1, 8, 16, torch.float32, DEV)
    want, _ = filled(large, 0), filled(small, 1)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    src = torch.tensor([0, -1, 4, 3, 1, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    dst = torch.tensor([8, 1, 2, 3, 9, -2 ** 31], dtype=torch.int32, device=DEV)
    kv_copy_pages(small, src, dst, into=large, err_flag=flag)
    for name in ("k", "v"):
        want[name][8], want[name][3] = getattr(small, name)[0], getattr(small, name)[3]
        assert torch.equal(getattr(large, name), want[name])
    assert flag.item() == 4
    flag.zero_()
    kv_copy_pages(small, src[:1], dst[:1], into=large, err_flag=flag)
    assert flag.item() == 0


def test_pages_past_4_gib():
    from cortex.kernels.paged_kv import KVPages, kv_block_bounds, kv_copy_pages, paged_block_select

    pages = KVPages.allocate(300000, 1, 64, 128, torch.bfloat16, DEV, bounded=True)  # 4.9 GB of keys
    pages.k[7] = torch.randn(1, 64, 128, device=DEV).bfloat16()
    pages.v[7] = 3.0
    ids = torch.tensor([299999, 262144, 5], dtype=torch.int32, device=DEV)
    kv_copy_pages(pages, torch.full_like(ids, 7), ids)
    for i in ids.tolist():
        assert torch.equal(pages.k[i], pages.k[7]) and torch.equal(pages.v[i], pages.v[7])
    lengths = torch.tensor([3 * 64], device=DEV)
    kv_block_bounds(pages, ids[None], lengths)
    for i in ids.tolist():
        assert torch.equal(pages.bounds[i, 0, 0], pages.k[7, 0].amax(0)) and torch.equal(pages.bounds[i, 0, 1], pages.k[7, 0].amin(0))
    pages.bounds[262144] -= 9.0
    q = torch.ones(1, 1, 128, dtype=torch.bfloat16, device=DEV)
    got = paged_block_select(q, pages, ids[None], lengths, 2, first=0)
    assert got.table.tolist() == [[[299999, 5]]] and got.lengths.tolist() == [128]


# ------------------------------------------------------------------------------- bounds


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,dim,page,layout", [(1, 16, 8, "head"), (8, 128, 16, "head"), (3, 96, 32, "row"),
                                                      (2, 48, 128, "gap"), (1, 112, 1024, "head"), (12, 64, 64, "row")])
def test_bounds_of_all_pages(dtype, kv_heads, dim, page, layout):
    from cortex.kernels.paged_kv import kv_block_bounds

    lens = [0, 1, 7, 8, 9, page - 1, page, page + 1, 3 * page + 5, 200]
    c = BoundedCache(lens, kv_heads, dim, page, DTYPES[dtype], seed=dim, layout=layout)
    kv_block_bounds(c.pages, c.block_table, c.lengths)
    got = c.gb.clone()
    want = c.fill_bounds()
    if dtype == "int8":
        want = torch.where(want == 7, want, want.float().double())
    assert torch.equal(got.double().cpu(), want.to(got.dtype).double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_new", [None, 1, 100])
def test_bounds_since(dtype, max_new):
    """Only pages that got a slot are written; more new slots than max_new says are found all the same."""
    from cortex.kernels.paged_kv import kv_block_bounds

    lens = [0, 1, 16, 17, 32, 33, 100, 250, 250, 250, 40]
    since = [0, 0, 15, 16, 31, 33, 2, 249, 250, 300, -5]
    c = BoundedCache(lens, 2, 64, 16, DTYPES[dtype], seed=3)
    kv_block_bounds(c.pages, c.block_table, c.lengths, since=torch.tensor(since, device=DEV), max_new=max_new)
    want = torch.full(c.gb.shape, 7.0, dtype=torch.float64)
    for b, n in enumerate(lens):
        for i in range(max(0, since[b]) // 16, -(-n // 16) if since[b] < n else 0):
            want[int(c.table[b][i])] = c.bounds64(b, i)
    assert torch.equal(c.gb.cpu(), want.to(c.gb.dtype))


@pytest.mark.parametrize("batch,length", [(1, 20000), (300, 40), (64, 700)])
def test_bounds_of_many_pages(batch, length):
    from cortex.kernels.paged_kv import kv_block_bounds

    c = BoundedCache([length - b % 7 for b in range(batch)], 4, 64, 16, torch.bfloat16, seed=batch)
    kv_block_bounds(c.pages, c.block_table, c.lengths)
    got = c.gb.clone()
    c.fill_bounds()
    assert torch.equal(got, c.gb)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_of_keys_without_numbers(dtype):
    c = BoundedCache([40], 1, 32, 8, DTYPES[dtype], seed=1)
    page = [int(p) for p in c.table[0][:5]]
    if dtype == "int8":
        c.pages.k_scale[page[1], 0, 3] = float("nan")
        c.pages.k_scale[page[2], 0, 0] = float("inf")
    else:
        c.pages.k[page[1], 0, 3, 5] = float("nan")
        c.pages.k[page[2], 0, 0, 7] = float("inf")
        c.pages.k[page[2], 0, 7, 8] = float("-inf")
    from cortex.kernels.paged_kv import kv_block_bounds

    kv_block_bounds(c.pages, c.block_table, c.lengths)
    k = c.pages.k.float() if dtype != "int8" else c.pages.k.float() * c.pages.k_scale[..., None]
    for p in page:  # (torch's largest and smallest of rows with a NaN is NaN)
        assert same(c.gb[p, 0, 0], k[p, 0].amax(0)) and same(c.gb[p, 0, 1], k[p, 0].amin(0))


def test_bounds_with_malformed_pages_and_lengths():
    from cortex.kernels.paged_kv import kv_block_bounds

    c = BoundedCache([40, 40, 40, 40], 1, 32, 8, torch.bfloat16, seed=2)
    c.block_table[1, 2], c.block_table[2, 0] = -1, c.num
    c.lengths[3], c.lengths[0] = -3, 10 ** 12
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    kv_block_bounds(c.pages, c.block_table, c.lengths, err_flag=flag)
    want = torch.full(c.gb.shape, 7.0, dtype=torch.float64)
    for b in (0, 1, 2):
        for i in range(5):
            if (b, i) not in ((1, 2), (2, 0)):
                want[int(c.table[b][i])] = c.bounds64(b, i)
    assert flag.item() == 4 and torch.equal(c.gb.cpu(), want.to(c.gb.dtype))
    # cut to max_length
    c.gb.fill_(7.0)
    flag.zero_()
    c.lengths.fill_(40)
    kv_block_bounds(c.pages, c.block_table[:1], c.lengths[:1], max_length=12, err_flag=flag)
    want.fill_(7.0)
    for i in range(2):
        want[int(c.table[0][i])] = c.bounds64(0, i, 12)
    assert flag.item() == 4 and torch.equal(c.gb.cpu(), want.to(c.gb.dtype))
    for kw in ({"max_length": 0}, {"max_length": 0, "since": c.lengths[:1] * 0, "max_new": 0}):
        flag.zero_()
        kv_block_bounds(c.pages, c.block_table[:1], c.lengths[:1], err_flag=flag, **kw)
        assert flag.item() == 4
    flag.zero_()
    kv_block_bounds(c.pages, c.block_table[:1, :0], c.lengths[:1] * 0, err_flag=flag)
    assert flag.item() == 0 and torch.equal(c.gb.cpu(), want.to(c.gb.dtype))


# ------------------------------------------------------------------------------- selection


def expected(c, q, count, first, recent, lens=None, table=None):
    """The table and lengths of a selection, from the bounds as they are on the GPU."""
    lens = c.lens if lens is None else lens
    table = c.table if table is None else table
    bounds, q = c.gb.double().cpu().numpy(), q.double().cpu().numpy()
    keep = min(count, c.width)
    group = q.shape[1] // c.kv_heads
    out = torch.full((len(lens), c.kv_heads, keep), -1, dtype=torch.int32)
    left = []
    for b, n in enumerate(lens):
        blocks = -(-n // c.page)
        left.append(n - (blocks - min(blocks, count)) * c.page)
        for h in range(c.kv_heads):
            kept = select64(table[b], bounds[:, h], q[b, h * group:(h + 1) * group], n, c.page, count, first, recent, c.num)
            out[b, h, :len(kept)] = table[b][kept]
    return out, left


def check_selection(c, q, count, first=1, recent=1, **kw):
    from cortex.kernels.paged_kv import paged_block_select

    got = paged_block_select(q.to(DEV), c.pages, c.block_table, c.lengths, count, first=first, recent=recent, **kw)
    want, left = expected(c, q, count, first, recent)
    assert got.lengths.tolist() == left
    bad = (got.table.cpu() != want).nonzero()
    assert got.table.shape == want.shape and not len(bad), f"{len(bad)} entries differ, first at {bad[0].tolist()}"
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 16), (2, 2, 32), (3, 1, 48), (8, 2, 64), (5, 1, 80), (12, 2, 96),
                                                (8, 1, 112), (32, 2, 128), (17, 1, 64), (40, 1, 128)])
def test_selection_heads_and_dims(dtype, heads, kv_heads, dim):
    c = BoundedCache([0, 5, 300, 170, 129], kv_heads, dim, 16, DTYPES[dtype], seed=heads + dim)
    c.fill_bounds()
    for count in (2, 9, 12):
        check_selection(c, c.query(heads), count)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [8, 64, 512])
def test_selection_lengths_around_blocks(dtype, page):
    lens = [0, 1, page - 1, page, page + 1, 2 * page, 4 * page - 1, 4 * page, 4 * page + 1, 5 * page, 17 * page, 18 * page - 3]
    c = BoundedCache(lens, 2, 32, page, DTYPES[dtype], seed=page)
    c.fill_bounds()
    q = c.query(4)
    for count, first, recent in [(1, 0, 1), (2, 1, 1), (4, 1, 1), (4, 0, 4), (5, 3, 2), (17, 1, 1), (18, 9, 9), (1000, 1, 1)]:
        check_selection(c, q, count, first, recent)


@pytest.mark.parametrize("lens", [[8 * 255], [8 * 256], [8 * 257 - 1], [8 * 1025], [8 * 4096 + 3], [8 * 20011], [8 * 1500 - i * 77 for i in range(130)]],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_selection_of_many_blocks(lens):
    c = BoundedCache(lens, 1, 16, 8, torch.bfloat16, seed=lens[0])
    g = torch.Generator().manual_seed(1)
    edge = torch.randn(c.gb.shape, generator=g)
    c.gb.copy_(torch.stack([edge.amax(2), edge.amin(2)], 2).to(c.gb.dtype))
    q = c.query(2)
    for count in (2, 100, 700):
        check_selection(c, q, count)


@pytest.mark.parametrize("batch,kv_heads,dim,blocks", [(3, 1, 16, 100), (70, 4, 48, 60), (300, 1, 128, 130), (50, 4, 32, 1030),
                                                       (200, 1, 16, 1500), (110, 1, 16, 2500), (24, 2, 64, 300), (2, 2, 64, 2049)])
@pytest.mark.parametrize("dtype,heads", [("bf16", 1), ("fp32", 5), ("int8", 3), ("bf16", 18)])
def test_selection_of_few_and_many_sequences(dtype, heads, batch, kv_heads, dim, blocks):
    """The one launch of 256 and of 512 threads, the two, with one and with four tiles a wavefront: on either side of
    where one takes over from the other."""
    from types import SimpleNamespace

    from cortex.kernels.paged_kv import KVPages

    g = torch.Generator().manual_seed(batch + blocks)
    c = SimpleNamespace(kv_heads=kv_heads, page=8, width=blocks, num=blocks + 40)
    c.lens = [8 * blocks - 8 * (37 * b % blocks) - b % 8 for b in range(batch)]
    c.table = torch.stack([torch.randperm(c.num, generator=g)[:blocks] for _ in range(batch)]).int()
    c.pages = KVPages.allocate(c.num, kv_heads, 8, dim, DTYPES[dtype], DEV, bounded=True)
    edge = torch.randn(c.num, kv_heads, 2, dim, generator=g)
    c.gb = c.pages.bounds
    c.gb.copy_(torch.stack([edge.amax(2), edge.amin(2)], 2).to(c.gb.dtype))
    c.block_table, c.lengths = c.table.to(DEV), torch.tensor(c.lens, device=DEV)
    q = torch.randn(batch, heads * kv_heads, dim, generator=g).to(c.pages.query_dtype)
    for count in (3, blocks // 3):
        check_selection(c, q, count)


@pytest.mark.parametrize("dtype", DTYPES)
def test_selection_ties(dtype):
    """Scores of few different values, of one value, and of both zeros: equal ones by the lower block."""
    c = BoundedCache([8 * 900, 8 * 300 + 1, 8 * 40], 2, 32, 8, DTYPES[dtype], seed=1)
    g = torch.Generator().manual_seed(2)
    q = torch.zeros(3, 4, 32)
    q[:, :, 3] = 1.0
    q[:, :, 4] = -1.0
    q = q.to(c.pages.query_dtype)
    for values in (torch.randint(0, 3, (c.num, 2, 2, 32), generator=g).float(), torch.full((c.num, 2, 2, 32), 1.5),
                   torch.where(torch.rand(c.num, 2, 2, 32, generator=g) < 0.5, 0.0, -0.0)):
        c.gb.copy_(values.to(c.gb.dtype))
        for count in (2, 37, 200):
            check_selection(c, q, count)
            check_selection(c, q, count, first=0, recent=1)


def test_selection_does_not_depend_on_the_order_of_sums():
    """Large terms that cancel: the small ones between them decide, and sums in fewer than 64 bits would lose them."""
    c = BoundedCache([8 * 200], 1, 128, 8, torch.float32, seed=1)
    g = torch.Generator().manual_seed(7)
    small = torch.rand(c.num, generator=g)
    q = torch.ones(1, 1, 128)
    for place in range(0, 128, 9):
        bounds = torch.zeros(c.num, 1, 2, 128)
        bounds[:, :, :, place] = 2.0 ** 30
        bounds[:, :, :, (place + 64) % 128] = -2.0 ** 30
        bounds[:, 0, 0, (place + 5) % 128] = small
        bounds[:, 0, 1, (place + 5) % 128] = 0.0
        c.gb.copy_(bounds)
        got = check_selection(c, q, 20)
        kept = small[got.table[0, 0, 1:-1].cpu().long()]
        others = sorted(small[c.table[0][1:199].long()].tolist(), reverse=True)[:18]
        assert sorted(kept.tolist(), reverse=True) == others


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_selection_of_values_at_the_ends(dtype):
    """NaN before every number, infinities, scores past the range of fp32, pages that are not there last."""
    c = BoundedCache([16 * 40, 16 * 40], 1, 64, 16, DTYPES[dtype], seed=4)
    c.fill_bounds()
    q = c.query(3)
    rows = c.table[0]
    c.gb[int(rows[5]), 0, 0, 3] = float("nan")
    c.gb[int(rows[6]), 0, 1, 60] = float("nan")
    c.gb[int(rows[7]), 0, 0] = float("inf")
    c.gb[int(rows[8]), 0, 0], c.gb[int(rows[8]), 0, 1] = float("-inf"), float("-inf")
    c.gb[int(rows[9]), 0, 0] = 3e38
    c.gb[int(rows[10]), 0, 0] = 3.2e38
    for count in (2, 3, 4, 5, 6, 10, 38, 39):
        check_selection(c, q, count)
    q[1, 2, 7] = float("nan")  # all scores of that sequence are alike
    check_selection(c, q, 7)
    q[1, 2, 7] = float("inf")
    check_selection(c, q, 7)


def test_selection_with_malformed_pages_and_lengths():
    from cortex.kernels.paged_kv import paged_attention, paged_block_select

    c = BoundedCache([16 * 12, 16 * 12, 16 * 12, 16 * 3], 2, 32, 16, torch.bfloat16, seed=6)
    c.fill_bounds()
    q = c.query(4)
    table = c.table.clone()
    table[0, 4], table[0, 5], table[3, 1] = -1, c.num, c.num + 7
    c.block_table.copy_(table)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    for count in (2, 10, 11, 12):
        flag.zero_()
        got = paged_block_select(q.to(DEV), c.pages, c.block_table, c.lengths, count, err_flag=flag)
        want, left = expected(c, q, count, 1, 1, table=table)
        assert torch.equal(got.table.cpu(), want) and got.lengths.tolist() == left and flag.item() == 4
    out = paged_attention(q.to(DEV), c.pages, got.table, got.lengths)  # such pages hold no keys
    assert out.isfinite().all()
    flag.zero_()
    paged_block_select(q[1:2].to(DEV), c.pages, c.block_table[1:2], c.lengths[1:2], 4, err_flag=flag)
    assert flag.item() == 0
    lengths = torch.tensor([-1, 10 ** 15, 16 * 12, 0], device=DEV)
    got = paged_block_select(q.to(DEV), c.pages, c.block_table, lengths, 5, err_flag=flag)
    want, left = expected(c, q, 5, 1, 1, lens=[0, 16 * 12, 16 * 12, 0], table=table)
    assert torch.equal(got.table.cpu(), want) and got.lengths.tolist() == left and flag.item() == 4
    # cut to max_length
    got = paged_block_select(q[1:3].to(DEV), c.pages, c.block_table[1:3], c.lengths[1:3], 4, max_length=100)
    bounds = c.gb.double().cpu().numpy()
    assert got.lengths.tolist() == [100 - 3 * 16] * 2
    for b in (0, 1):
        for h in range(2):
            kept = select64(table[1 + b], bounds[:, h], q[1 + b, 2 * h:2 * h + 2].double().numpy(), 100, 16, 4, 1, 1, c.num)
            assert got.table[b, h].tolist() == table[1 + b][kept].tolist()


def test_selection_of_nothing():
    from cortex.kernels.paged_kv import paged_attention, paged_block_select

    c = BoundedCache([0, 0], 2, 32, 16, torch.bfloat16)
    got = check_selection(c, c.query(2), 4)
    assert (paged_attention(c.query(2).to(DEV), c.pages, got.table, got.lengths) == 0).all()
    got = paged_block_select(c.query(2).to(DEV), c.pages, c.block_table[:, :0], c.lengths, 4)
    assert got.table.shape == (2, 2, 0) and got.lengths.tolist() == [0, 0]
    assert (paged_attention(c.query(2).to(DEV), c.pages, got.table, got.lengths) == 0).all()
    got = paged_block_select(c.query(2)[:0].to(DEV), c.pages, c.block_table[:0], c.lengths[:0], 4)
    assert got.table.shape == (0, 2, 1) and got.lengths.shape == (0,)


# ------------------------------------------------------------------------------- attention by key heads


class ByHead:
    """Pages of a sequence chosen by hand for each key head, as a plain cache of each head."""

    def __init__(self, c, kept):
        # kept[b][h]: blocks of sequence b, the same number for every head
        most = max(1, max(len(k) for row in kept for k in row))
        self.table = torch.full((len(kept), c.kv_heads, most), -1, dtype=torch.int32)
        self.lens = []
        for b, row in enumerate(kept):
            blocks = -(-c.lens[b] // c.page)
            for h, ids in enumerate(row):
                self.table[b, h, :len(ids)] = c.table[b][ids]
            self.lens.append(len(row[0]) * c.page - (blocks * c.page - c.lens[b] if len(row[0]) else 0))
        self.c, self.kept = c, kept

    def attention64(self, q, **kw):
        c, group = self.c, q.shape[1] // self.c.kv_heads
        out, tol, added, added_tol = [], [], [], []
        for h in range(c.kv_heads):
            one = type("", (), {})()
            one.kv_heads, one.lens, one.k, one.v = 1, self.lens, c.k[:, h:h + 1], c.v[:, h:h + 1]
            one.at = lambda b, slots, h=h: (self.table[b, h][slots // c.page].long(), slice(None), slots % c.page)
            o, a, t, at = attention64(one, q[:, h * group:(h + 1) * group], **kw)
            out.append(o), tol.append(t), added.append(a), added_tol.append(at)
        return torch.cat(out, 1), torch.cat(tol, 1), added, added_tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,longest", [(4, 4, 64, 16, 40), (8, 2, 128, 16, 150), (34, 2, 96, 64, 60),
                                                            (6, 3, 32, 8, 300), (12, 12, 64, 32, 20)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_over_pages_by_key_head(dtype, heads, kv_heads, dim, page, longest, accumulate):
    from cortex.kernels.paged_kv import paged_attention

    lens = [longest * page - 3, 0, 1, page, 11 * page + 2]
    c = BoundedCache(lens, kv_heads, dim, page, DTYPES[dtype], seed=dim, tracked=True)
    g = torch.Generator().manual_seed(3)
    kept = []
    for n in lens:
        blocks = -(-n // page)
        few = max(0, min(blocks - 1, blocks * 2 // 3))
        kept.append([sorted(torch.randperm(max(blocks - 1, 0), generator=g)[:few].tolist()) + [blocks - 1] * (blocks > 0)
                     for _ in range(kv_heads)])
    by = ByHead(c, kept)
    q = c.query(heads)
    want, tol, added, wtol = by.attention64(q)
    before = c.pages.weight.cpu().clone()
    got = paged_attention(q.to(DEV), c.pages, by.table.to(DEV), torch.tensor(by.lens, device=DEV), accumulate=accumulate)
    check(got, want, tol, "out")
    after, total, allowed = c.pages.weight.cpu(), before.double(), torch.zeros(before.shape, dtype=torch.float64)
    if accumulate:
        for b, n in enumerate(by.lens):
            slots = torch.arange(n)
            for h in range(kv_heads):
                at = by.table[b, h][slots // page].long(), h, slots % page
                total[at] += added[h][b][:, 0]
                allowed[at] = wtol[h][b][:, 0] + 2.0 ** -24 * total[at]
    there = ~before.isnan()
    check(after[there], total[there], allowed[there], "weight")


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_a_cache_together(dtype):
    """Prompts and tokens: norm and rotation, append, bounds, selection, attention; a fork in the middle."""
    from cortex.kernels.paged_kv import (KVPages, kv_block_bounds, kv_copy_pages, paged_attention, paged_block_select,
                                         paged_kv_append)
    from cortex.kernels.rotary import qk_norm_rope, rotary_frequencies

    kv, heads, dim, page = 2, 8, 64, 16
    x = torch.float32 if dtype == "fp32" else torch.bfloat16
    pages = KVPages.allocate(80, kv, page, dim, DTYPES[dtype], DEV, bounded=True)
    freq = rotary_frequencies(dim)
    g = torch.Generator(DEV).manual_seed(5)
    gains = [1 + 0.1 * torch.randn(dim, generator=g, device=DEV) for _ in range(2)]
    table = torch.randperm(80, generator=torch.Generator().manual_seed(1))[:60].reshape(3, 20).int().to(DEV)
    lengths = torch.zeros(3, dtype=torch.int64, device=DEV)
    seen_k, seen_v = [[] for _ in range(3)], [[] for _ in range(3)]

    def step(counts):
        nonlocal lengths
        T = sum(counts)
        qkv = torch.randn(T, heads + 2 * kv, dim, generator=g, device=DEV).to(x)
        offsets = torch.tensor([0, counts[0], counts[0] + counts[1], T], device=DEV)
        at = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(counts, device=DEV))
        positions = lengths[at] + torch.arange(T, device=DEV) - offsets[at]
        q, k = qk_norm_rope(qkv[:, :heads], qkv[:, heads:heads + kv], positions, freq, eps=1e-6, q_gain=gains[0], k_gain=gains[1])
        v = qkv[:, heads + kv:]
        before = lengths
        lengths = paged_kv_append(pages, k, v, table, lengths, offsets=offsets)
        kv_block_bounds(pages, table, lengths, since=before, max_new=max(counts))
        for b in range(3):
            seen_k[b].append(k[at == b]), seen_v[b].append(v[at == b])
        return q[(offsets[1:] - 1)]

    def values():
        k = pages.k.float() if dtype != "int8" else pages.k.float() * pages.k_scale[..., None]
        v = pages.v.float() if dtype != "int8" else pages.v.float() * pages.v_scale[..., None]
        return k.cpu(), v.cpu()

    def attend(q, count):
        few = paged_block_select(q, pages, table, lengths, count)
        out = paged_attention(q, pages, few.table, few.lengths)
        c = type("", (), {})()
        c.page, c.kv_heads, c.lens, c.table, c.width, c.num, c.gb = page, kv, lengths.tolist(), table.cpu(), 20, 80, pages.bounds
        c.k, c.v = values()
        want, left = expected(c, q, count, 1, 1)
        assert torch.equal(few.table.cpu(), want) and few.lengths.tolist() == left
        by = ByHead.__new__(ByHead)
        by.c, by.table, by.lens = c, want, left
        o, tol, _, _ = by.attention64(q.cpu())
        check(out, o, tol, f"{count} pages")
        return out

    q = step([200, 33, 1])
    attend(q, 4)
    for _ in range(20):
        q = step([1, 1, 1])
    dense = paged_attention(q, pages, table, lengths)
    assert torch.equal(attend(q, 20), dense)  # all pages: the same tiles in the same order
    attend(q, 3)
    # sequence 1 goes on as a fork of sequence 0: its full pages shared, the last one copied
    used = -(-int(lengths[0]) // page)
    spare = sorted(set(range(80)) - set(table.flatten().tolist()))[:1]
    kv_copy_pages(pages, table[0, used - 1:used].contiguous(), torch.tensor(spare, dtype=torch.int32, device=DEV))
    table[1, :used - 1] = table[0, :used - 1]
    table[1, used - 1] = spare[0]
    lengths[1] = lengths[0]
    assert torch.equal(paged_attention(q[[0, 0, 2]], pages, table, lengths)[0], paged_attention(q[[0, 0, 2]], pages, table, lengths)[1])
    for _ in range(3):
        q = step([1, 1, 1])
    attend(q, 5)


def test_captured_and_on_another_stream():
    """Bounds, selection and attention in one graph, replayed on other lengths and values, with eager work in between."""
    from cortex.kernels.paged_kv import kv_block_bounds, kv_copy_pages, paged_attention, paged_block_select

    c = BoundedCache([16 * 30, 16 * 25 + 3, 70], 2, 64, 16, torch.bfloat16, seed=9)
    q = c.query(8).to(DEV)
    src, dst = c.block_table[0, :2].contiguous(), torch.tensor([c.num - 1, c.num - 2], dtype=torch.int32, device=DEV)
    free = sorted(set(range(c.num)) - set(c.table.flatten().tolist()))
    dst = torch.tensor(free[:2], dtype=torch.int32, device=DEV)

    def work():
        kv_copy_pages(c.pages, src, dst)
        kv_block_bounds(c.pages, c.block_table, c.lengths)
        few = paged_block_select(q, c.pages, c.block_table, c.lengths, 6)
        return [*few, paged_attention(q, c.pages, few.table, few.lengths)]

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        first = work()
    with torch.cuda.graph(two):
        second = work()
    lens = [[16 * 30, 16 * 25 + 3, 70], [0, 16 * 30, 100], [5, 16 * 7, 16 * 29 + 1], [16 * 30, 1, 0]]
    c.pages.k.nan_to_num_(), c.pages.v.nan_to_num_()
    for now in lens:
        c.lengths.copy_(torch.tensor(now))
        q.copy_(torch.randn(q.shape))
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in first], [t.clone() for t in second]
        eager = work()
        torch.cuda.synchronize()
        for got in kept:
            assert all(torch.equal(a, b) for a, b in zip(got, eager)), now
        assert torch.equal(c.pages.k[dst.long()], c.pages.k[src.long()])


def test_strided_queries_and_tables():
    from cortex.kernels.paged_kv import kv_block_bounds, paged_block_select

    c = BoundedCache([16 * 30, 16 * 25 + 3, 70], 2, 64, 16, torch.bfloat16, seed=10)
    q = c.query(8)
    wide = torch.full((3, c.width + 6), -5, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + c.width] = c.block_table
    kv_block_bounds(c.pages, wide[:, 2:2 + c.width], c.lengths)
    want = check_selection(c, q, 7)
    joint = torch.zeros(3, 12, 64, dtype=q.dtype, device=DEV)
    joint[:, 3:11] = q.to(DEV)
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    for x in (joint[:, 3:11], odd, q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)):
        got = paged_block_select(x, c.pages, wide[:, 2:2 + c.width], c.lengths, 7)
        assert torch.equal(got.table, want.table) and torch.equal(got.lengths, want.lengths)


def test_refusals():
    from cortex.kernels.paged_kv import KVPages, kv_block_bounds, kv_copy_pages, paged_attention, paged_block_select

    c = BoundedCache([100, 30], 2, 64, 16, torch.bfloat16, tracked=True)
    c.fill_bounds()
    q, table, lengths = c.query(4).to(DEV), c.block_table, c.lengths
    plain = KVPages(c.pages.k, c.pages.v)
    ids = torch.zeros(2, dtype=torch.int32, device=DEV)

    def refused(match, f, *args, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            f(*args, **kw)

    refused("bounds", KVPages, c.pages.k, c.pages.v, bounds=c.gb.float())
    refused("bounds", KVPages, c.pages.k, c.pages.v, bounds=c.gb[:, :1])
    refused("bounds", KVPages, c.pages.k, c.pages.v, bounds=c.gb.transpose(1, 2).contiguous().transpose(1, 2))
    refused("ROCm GPU", KVPages, c.pages.k, c.pages.v, bounds=c.gb.cpu(), error=RuntimeError)
    odd = torch.zeros(c.gb.numel() + 1, dtype=c.gb.dtype, device=DEV)[1:].view(c.gb.shape)
    refused("16-byte", KVPages, c.pages.k, c.pages.v, bounds=odd)
    refused("with bounds", kv_block_bounds, plain, table, lengths)
    refused("since", kv_block_bounds, c.pages, table, lengths, since=lengths[:1])
    refused("since", kv_block_bounds, c.pages, table, lengths, since=lengths.int())
    refused("ROCm GPU", kv_block_bounds, c.pages, table, lengths, since=lengths.cpu(), error=RuntimeError)
    refused("max_new", kv_block_bounds, c.pages, table, lengths, max_new=-1)
    refused("max_length", kv_block_bounds, c.pages, table, lengths, max_length=-1)
    refused("block_table", kv_block_bounds, c.pages, table.long(), lengths)
    refused("block_table", kv_block_bounds, c.pages, table[None], lengths)
    refused("with bounds", paged_block_select, q, plain, table, lengths, 4)
    refused("count", paged_block_select, q, c.pages, table, lengths, 0)
    refused("count", paged_block_select, q, c.pages, table, lengths, 4, first=4)
    refused("count", paged_block_select, q, c.pages, table, lengths, 4, recent=0)
    refused("count", paged_block_select, q, c.pages, table, lengths, 4, first=-1)
    refused("max_length", paged_block_select, q, c.pages, table, lengths, 4, max_length=-1)
    refused("q must be", paged_block_select, q.float(), c.pages, table, lengths, 4)
    refused("q must be", paged_block_select, q[:1], c.pages, table, lengths, 4)
    refused("multiple", paged_block_select, q[:, :3], c.pages, table, lengths, 4)
    refused("no backward", paged_block_select, q.clone().requires_grad_(), c.pages, table, lengths, 4, error=RuntimeError)
    refused("by key heads", paged_attention, q, c.pages, table[:, None].expand(-1, 2, -1), lengths)
    refused("by key heads", paged_attention, q, c.pages, table[:, None].contiguous(), lengths)
    refused("by key heads", paged_attention, q, c.pages, table[:, None].expand(-1, 2, -1).contiguous().long(), lengths)
    refused("int32", kv_copy_pages, c.pages, ids.long(), ids)
    refused("one length", kv_copy_pages, c.pages, ids, ids[:1])
    refused("contiguous", kv_copy_pages, c.pages, torch.zeros(4, dtype=torch.int32, device=DEV)[::2], ids)
    refused("ROCm GPU", kv_copy_pages, c.pages, ids.cpu(), ids, error=RuntimeError)
    refused("both pools", kv_copy_pages, c.pages, ids, ids, into=plain)
    refused("into must", kv_copy_pages, c.pages, ids, ids, into=KVPages.allocate(4, 2, 32, 64))
    refused("into must", kv_copy_pages, c.pages, ids, ids, into=KVPages.allocate(4, 2, 16, 64, torch.float32))
    refused("err_flag", kv_copy_pages, c.pages, ids, ids, err_flag=lengths)
    from cortex._native import NativeLibraryError

    meeting = KVPages(c.pages.k[:1].expand(4, -1, -1, -1), c.pages.v[:4].clone())
    refused("share memory", kv_copy_pages, meeting, ids[:1], ids[:1], error=NativeLibraryError)
