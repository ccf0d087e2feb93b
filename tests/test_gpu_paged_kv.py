"""The paged K/V cache operators against plain computations in 64 bits (tests/_paged.py): append and eviction bit
for bit, attention within bounds derived from its arithmetic."""

from __future__ import annotations

import pytest
import torch

from _paged import DEV, Cache, attention64, codes, evict64

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8}


def check(got, want, tol, what):
    got = got.double().cpu()
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float(off[bad].max())} at "
                           f"{bad.nonzero()[0].tolist()} where {float(tol[bad].min())} is allowed")


def attend(c, q, **kw):
    from cortex.kernels.paged_kv import paged_attention

    return paged_attention(q.to(DEV), c.pages, c.block_table, c.lengths, **kw)


# ------------------------------------------------------------------------------- attention


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 16), (4, 4, 64), (8, 2, 128), (6, 2, 96), (16, 1, 32), (17, 1, 64),
                                                (40, 2, 128), (12, 12, 80), (66, 2, 48), (3, 1, 112)])
def test_attention_heads_and_dims(dtype, heads, kv_heads, dim):
    c = Cache([0, 1, 33, 200, 77], kv_heads, dim, 16, DTYPES[dtype], seed=heads + dim)
    q = c.query(heads)
    want, _, tol, _ = attention64(c, q)
    got = attend(c, q)
    check(got, want, tol, "out")
    assert (got[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 1024])
def test_attention_lengths_around_pages_and_tiles(dtype, page):
    lens = [1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 127, 128, 129, 255, 256, 257, 500, 511, 512, 513]
    c = Cache(lens, 2, 64, page, DTYPES[dtype], seed=page)
    q = c.query(4)
    want, _, tol, _ = attention64(c, q)
    check(attend(c, q), want, tol, "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[20011], [9000, 3, 0, 4097], [5000] * 9 + [1, 0], [0], [0, 0, 0], [2100] * 70,
                                  [1900, 5, 0, 1025] * 40, [2048, 700, 64, 33] * 32],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_attention_long_and_ragged(dtype, lens):
    c = Cache(lens, 2, 64, 32, DTYPES[dtype], seed=len(lens))
    q = c.query(8)
    want, _, tol, _ = attention64(c, q)
    check(attend(c, q), want, tol, "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(17, 1, 64), (32, 1, 128), (66, 2, 96), (80, 2, 48), (34, 2, 128)])
def test_attention_many_heads_on_long_keys(dtype, heads, kv_heads, dim):
    """More query heads to a key head than one product has, on keys that are split: with the weights and without."""
    lens = [3000, 1, 0, 1100, 65]
    c = Cache(lens, kv_heads, dim, 16, DTYPES[dtype], seed=heads, tracked=True)
    q = c.query(heads)
    want, added, tol, wtol = attention64(c, q)
    check(attend(c, q), want, tol, "out")
    check(attend(c, q, accumulate=True), want, tol, "out with weights")
    after = c.pages.weight.cpu()
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        total = c.weight[at].double() + added[b]
        check(after[at], total, wtol[b] + 2.0 ** -24 * total, f"weight {b}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["row", "gap"])
def test_attention_strided_pages_queries_and_outputs(dtype, layout):
    c = Cache([300, 41, 0, 130], 3, 64, 16, DTYPES[dtype], seed=5, layout=layout)
    q = c.query(6)
    want, _, tol, _ = attention64(c, q)
    wide = torch.zeros(4, 3 * 6, 64, dtype=q.dtype, device=DEV)  # the queries of a joint projection
    wide[:, :6] = q.to(DEV)
    out = torch.full((4, 2, 6, 64), 7.0, dtype=q.dtype, device=DEV)
    got = attend(c, wide[:, :6], out=out[:, 1])
    assert got.data_ptr() == out[:, 1].data_ptr()
    check(got, want, tol, "strided")
    assert (out[:, 0] == 7).all()
    odd = torch.zeros(4 * 6 * 64 + 1, dtype=q.dtype, device=DEV)[1:].reshape(4, 6, 64)  # not 16-byte aligned
    odd.copy_(q)
    check(attend(c, odd), want, tol, "unaligned")
    swapped = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    check(attend(c, swapped), want, tol, "heads outside")
    per_batch_table = torch.zeros(4, c.width + 5, dtype=torch.int32, device=DEV)
    per_batch_table[:, 2:2 + c.width] = c.block_table
    from cortex.kernels.paged_kv import paged_attention

    check(paged_attention(q.to(DEV), c.pages, per_batch_table[:, 2:2 + c.width], c.lengths), want, tol, "table slice")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_scale_and_peaked_scores(dtype):
    """One key far above the others, at the first, a middle and the last slot; large negative scores; no scale."""
    c = Cache([700, 700, 700], 1, 64, 16, DTYPES[dtype], seed=8, std=3.0)
    q = c.query(2, std=3.0)
    for b, j in enumerate((0, 333, 699)):
        q[b] = (c.k[c.at(b, torch.tensor([j]))][0, 0].float() * 4).to(q.dtype)
    for scale in (None, 1.0, -0.25, 0.0):
        want, _, tol, _ = attention64(c, q, scale=scale)
        check(attend(c, q, scale=scale), want, tol, f"scale {scale}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,dim", [(40, 64), (300, 128), (5000, 64)])
def test_attention_large_values_without_weight(dtype, n, dim):
    """Keys whose weight is below exp(-200) add nothing, whatever finite values they have."""
    c = Cache([n], 1, dim, 16, DTYPES[dtype], seed=n)
    q = c.query(1)
    for j, value in [(3, 3e38), (17, -3e38), (n - 1, 1e38), (n // 2, -2e37)]:
        at = c.table[0][j // 16].long(), 0, j % 16
        c.k[at] = (-60 * q[0, 0].float()).to(c.k.dtype)
        c.v[at] = value
        for pool, own in ((c.gk, c.k), (c.gv, c.v)):
            pool[at] = own[at].to(DEV)
    want, _, tol, _ = attention64(c, q)
    check(attend(c, q), want, tol, "out")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_infinities(dtype):
    """Values of +-inf and NaN reach the heads and dims that they belong to and no others; a key whose score is
    -inf has no weight; a sequence with only such keys gives 0, as rows without allowed keys do elsewhere."""
    c = Cache([70, 70, 40], 1, 64, 16, DTYPES[dtype], seed=9)
    q = c.query(2).abs() + 0.5
    v = c.v[c.at(0, torch.arange(70))][:, 0].double()
    c.gv[c.table[0][66 // 16], 0, 66 % 16, 3] = float("inf")
    c.gv[c.table[0][5 // 16], 0, 5 % 16, 9] = float("nan")
    c.gk[c.table[1][20 // 16], 0, 20 % 16, 7] = float("-inf")
    c.k[c.table[1][20 // 16], 0, 20 % 16] = -100.0  # (stands for weight 0)
    for j in range(40):
        c.gk[c.table[2][j // 16], 0, j % 16, 1] = float("-inf")
    want, _, tol, _ = attention64(c, q)
    got = attend(c, q).double().cpu()
    assert (got[0, :, 3] == float("inf")).all() and torch.isnan(got[0, :, 9]).all()
    rest = [d for d in range(64) if d not in (3, 9)]
    check(got[0][:, rest], want[0][:, rest], tol[0][:, rest], "beside inf")
    check(got[1], want[1], tol[1], "-inf score")
    assert (got[2] == 0).all() and v.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(8, 2, 64, [5, 0, 130, 64]), (32, 8, 128, [1000, 2500, 31]),
                                                     (20, 1, 96, [300, 33]), (4, 4, 32, [7000]), (8, 2, 64, [1500, 3, 0, 40] * 33)])
def test_accumulated_weights(dtype, heads, kv_heads, dim, lens):
    c = Cache(lens, kv_heads, dim, 16, DTYPES[dtype], seed=11, tracked=True)
    q = c.query(heads)
    want, added, tol, wtol = attention64(c, q)
    before = c.pages.weight.cpu()
    check(attend(c, q, accumulate=True), want, tol, "out")
    after = c.pages.weight.cpu()
    used = torch.zeros_like(before, dtype=torch.bool)
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        used[at] = True
        total = c.weight[at].double() + added[b]
        check(after[at], total, wtol[b] + 2.0 ** -24 * total, f"weight {b}")
    assert torch.isnan(after[~used]).all()  # rows that nobody owns stay as they were
    assert torch.equal(before[used], c.weight[used])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_bad_pages_and_lengths(dtype):
    """A page id outside the pool holds no keys, a length outside the table is cut: both are flagged, once."""
    c = Cache([100, 50, 30, 20], 2, 64, 16, DTYPES[dtype], seed=13, tracked=True)
    q = c.query(4)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    want, _, tol, _ = attention64(c, q)
    check(attend(c, q, err_flag=flag), want, tol, "out")
    assert int(flag) == 0
    c.block_table[0, 2] = c.num
    c.block_table[1, 0] = -1
    c.lengths[3] = -5
    keep = torch.tensor([j for j in range(100) if not 32 <= j < 48])
    saved = c.at
    c.at = lambda b, s: saved(b, keep if b == 0 else torch.arange(16, 50) if b == 1 else s)
    want, added, tol, _ = attention64(c, q, lens=[84, 34, 30, 0])
    before = c.pages.weight.cpu()
    check(attend(c, q, accumulate=True, err_flag=flag), want, tol, "bad pages")
    assert int(flag) == 4
    untouched = c.pages.weight.cpu()[c.table[0, 2].long()]
    assert torch.equal(untouched.nan_to_num(), before[c.table[0, 2].long()].nan_to_num())
    c.at = saved
    flag.zero_()
    c.lengths[3] = c.width * 16 + 1  # one past the table
    attend(c, q, err_flag=flag)
    assert int(flag) == 4


def test_attention_max_length():
    c = Cache([100, 40], 2, 64, 16, torch.bfloat16, seed=14)
    q = c.query(2)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    want, _, tol, _ = attention64(c, q)
    check(attend(c, q, max_length=100, err_flag=flag), want, tol, "bound")
    assert int(flag) == 0
    want, _, tol, _ = attention64(c, q, lens=[64, 40])
    check(attend(c, q, max_length=64, err_flag=flag), want, tol, "cut")
    assert int(flag) == 4
    assert (attend(c, q, max_length=0) == 0).all()


def test_sequences_may_share_pages():
    """Two sequences with a common prefix of pages, of other lengths."""
    c = Cache([100, 100], 2, 64, 16, torch.bfloat16, seed=15)
    q = c.query(4)
    c.block_table[1] = c.block_table[0]
    c.table[1] = c.table[0]
    c.lengths[1] = 70
    want, _, tol, _ = attention64(c, q, lens=[100, 70])
    check(attend(c, q), want, tol, "shared")


# ------------------------------------------------------------------------------- append


def _append_plain(c, k, v, off, pos, dtype):
    """The pools after the append, on the CPU: a dict of tensors."""
    pools = {"k": c.gk.cpu().clone(), "v": c.gv.cpu().clone()}
    for n in ("k_scale", "v_scale", "weight", "position"):
        t = getattr(c.pages, n)
        if t is not None:
            pools[n] = t.cpu().clone()
    for b, n in enumerate(c.lens):
        slots = torch.arange(n, n + off[b + 1] - off[b])
        at = c.at(b, slots)
        for name, x in (("k", k), ("v", v)):
            x = x[off[b]:off[b + 1]]
            if dtype == torch.int8:
                pools[name][at], pools[name + "_scale"][at] = codes(x.float())
            else:
                pools[name][at] = x.to(dtype)
        if "weight" in pools:
            pools["weight"][at] = 0.0
            pools["position"][at] = (slots if pos is None else pos[off[b]:off[b + 1]]).int()[:, None]
    return pools


def _same(c, pools):
    for n, want in pools.items():
        got = (c.gk if n == "k" else c.gv if n == "v" else getattr(c.pages, n)).cpu()
        if got.is_floating_point():
            assert torch.equal(torch.isnan(got), torch.isnan(want)), n
            got, want = got.nan_to_num(), want.nan_to_num()
        assert torch.equal(got, want), n


@pytest.mark.parametrize("x", ["bf16", "fp32"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,dim,page,layout", [(8, 64, 16, "head"), (1, 16, 8, "head"), (3, 96, 32, "row"),
                                                      (17, 128, 16, "gap"), (2, 48, 64, "head"), (40, 112, 8, "row")])
def test_append_a_token_a_sequence(x, dtype, kv_heads, dim, page, layout):
    from cortex.kernels.paged_kv import paged_kv_append

    c = Cache([0, 1, 7, 8, 31, 100, 15, 16], kv_heads, dim, page, DTYPES[dtype], seed=dim, room=1, layout=layout,
              tracked=kv_heads != 3)
    k, v = (torch.randn(8, kv_heads, dim, generator=c.g).to(DTYPES[x]) * 3 for _ in range(2))
    k[2, 0] = 0.0  # a row of zeros: scale 1e-8 / 127
    pools = _append_plain(c, k, v, list(range(9)), None, DTYPES[dtype])
    got = paged_kv_append(c.pages, k.to(DEV), v.to(DEV), c.block_table, c.lengths)
    assert got.tolist() == [n + 1 for n in c.lens] and c.lengths.tolist() == c.lens
    _same(c, pools)
    assert paged_kv_append(c.pages, k.to(DEV), v.to(DEV), c.block_table, c.lengths, new_lengths=c.lengths) is c.lengths
    assert c.lengths.tolist() == [n + 1 for n in c.lens]
    _same(c, pools)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[0, 5, 0, 17, 300, 1, 0], [1] * 300, [0, 0], [1000], [0] * 40 + [9] + [0] * 40],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_append_ragged(dtype, counts):
    from cortex.kernels.paged_kv import paged_kv_append

    lens = [(7 * i) % 40 for i in range(len(counts))]
    c = Cache(lens, 2, 64, 16, DTYPES[dtype], seed=len(counts), room=max(counts), tracked=True)
    off = [0]
    for n in counts:
        off.append(off[-1] + n)
    T = off[-1] + 3  # three rows behind the last sequence
    k, v = (torch.randn(T, 2, 64, generator=c.g).to(torch.bfloat16) for _ in range(2))
    pos = torch.randint(0, 10 ** 6, (T,), generator=c.g)
    pools = _append_plain(c, k, v, off, pos, DTYPES[dtype])
    wide = torch.zeros(T, 6, 64, dtype=torch.bfloat16, device=DEV)  # k and v as parts of a joint projection
    wide[:, :2], wide[:, 2:4] = k.to(DEV), v.to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = (c.pages, wide[:, :2], wide[:, 2:4], c.block_table, c.lengths)
    kw = {"offsets": torch.tensor(off, device=DEV), "positions": pos.to(DEV), "err_flag": flag}
    got = paged_kv_append(*args, **kw)
    assert got.tolist() == [n + m for n, m in zip(lens, counts)] and int(flag) == 0
    _same(c, pools)
    paged_kv_append(*args, **kw, new_lengths=c.lengths)
    assert c.lengths.tolist() == got.tolist()
    _same(c, pools)


@pytest.mark.parametrize("x", ["bf16", "fp32"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,kv_heads,dim", [(4099, 2, 64), (6151, 3, 48), (16801, 8, 128), (133001, 1, 16), (70001, 1, 32)])
def test_append_several_tokens_a_workgroup(x, dtype, tokens, kv_heads, dim):
    """Enough tokens that a workgroup takes several of them (2, 3, 4, 64 and 34 on 256 CUs), the last one fewer, and sequences
    begin and end inside its share."""
    from cortex.kernels.paged_kv import paged_kv_append

    g = torch.Generator().manual_seed(tokens)
    cuts = torch.randint(0, tokens + 1, (40,), generator=g).sort().values.tolist()
    off = [0, 0, *cuts, tokens, tokens]  # (empty sequences at both ends)
    counts = [b - a for a, b in zip(off, off[1:])]
    lens = [(5 * i) % 23 for i in range(len(counts))]
    c = Cache(lens, kv_heads, dim, 32, DTYPES[dtype], seed=tokens, room=max(counts), tracked=True)
    k, v = (torch.randn(tokens + 2, kv_heads, dim, generator=g).to(DTYPES[x]) for _ in range(2))
    pos = torch.randint(0, 10 ** 6, (tokens + 2,), generator=g)
    pools = _append_plain(c, k, v, off, pos, DTYPES[dtype])
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = paged_kv_append(c.pages, k.to(DEV), v.to(DEV), c.block_table, c.lengths, offsets=torch.tensor(off, device=DEV),
                          positions=pos.to(DEV), err_flag=flag)
    assert got.tolist() == [n + m for n, m in zip(lens, counts)] and int(flag) == 0
    _same(c, pools)


@pytest.mark.parametrize("x", ["bf16", "fp32"])
def test_append_int8_rows_without_a_scale(x):
    """Ties round half to even; an infinity or a NaN makes all of its row NaN, and no other row."""
    from cortex.kernels.paged_kv import paged_kv_append

    c = Cache([3, 3, 3, 3], 2, 32, 8, torch.int8, seed=3, room=1)
    k = torch.randn(4, 2, 32, generator=c.g).to(DTYPES[x])
    k[0, 0] = torch.arange(32).to(k.dtype) - 15.5  # halves of the scale 127 / 127
    k[0, 0, 31] = 127.0
    v = k.clone()
    k[1, 1, 5] = float("inf")
    v[2, 0, 31] = float("nan")
    paged_kv_append(c.pages, k.to(DEV), v.to(DEV), c.block_table, c.lengths)
    for b in range(4):
        at = (c.table[b, 0].long(), slice(None), 3)
        for name, t in (("k", k), ("v", v)):
            code, scale = getattr(c.pages, name).cpu()[at], getattr(c.pages, name + "_scale").cpu()[at]
            for h in range(2):
                if not t[b, h].isfinite().all():
                    assert torch.isnan(scale[h])
                    continue
                wc, ws = codes(t[b, h].float())
                assert torch.equal(code[h], wc) and scale[h] == ws


def test_append_without_room_or_page():
    """Nothing is written for a token without a slot or a page; the flag says so, the lengths stay in the table."""
    from cortex.kernels.paged_kv import paged_kv_append

    c = Cache([16, 15, 3, 5, 4], 2, 32, 8, torch.bfloat16, seed=4, tracked=True)
    assert c.width == 2
    k = torch.randn(5, 2, 32, generator=c.g).to(torch.bfloat16)
    c.block_table[2, 0] = c.num
    c.lengths[3] = -1
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = c.gk.clone()
    got = paged_kv_append(c.pages, k.to(DEV), k.to(DEV), c.block_table, c.lengths, err_flag=flag)
    assert got.tolist() == [16, 16, 4, 1, 5] and int(flag) == 4
    changed = (c.gk.nan_to_num(9.0) != before.nan_to_num(9.0)).any(-1).any(1).nonzero().tolist()
    assert sorted(changed) == sorted([[int(c.table[1, 1]), 7], [int(c.table[3, 0]), 0], [int(c.table[4, 0]), 4]])
    # ragged: 20 tokens into 16 slots, the rest of them dropped
    flag.zero_()
    c.lengths.copy_(torch.tensor([4, 16, 0, 0, 0]))
    many = torch.randn(23, 2, 32, generator=c.g).to(torch.bfloat16).to(DEV)
    got = paged_kv_append(c.pages, many, many, c.block_table, c.lengths, err_flag=flag,
                          offsets=torch.tensor([0, 20, 22, 22, 22, 23], device=DEV))
    assert got.tolist() == [16, 16, 0, 0, 1] and int(flag) == 4
    assert torch.equal(c.gk[c.table[0, 1].long(), :, 7], many[11])


def test_append_without_room_page_or_length():
    from cortex.kernels.paged_kv import paged_kv_append

    c = Cache([16, 15, 3, 5, 4], 2, 32, 8, torch.bfloat16, seed=4, tracked=True)
    k = torch.randn(5, 2, 32, generator=c.g).to(torch.bfloat16)
    c.block_table[2, 0] = c.num
    c.lengths[3] = -1
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = c.gk.clone()
    got = paged_kv_append(c.pages, k.to(DEV), k.to(DEV), c.block_table, c.lengths, err_flag=flag)
    assert got.tolist() == [16, 16, 4, -1, 5] and int(flag) == 4
    changed = (c.gk.nan_to_num(9.0) != before.nan_to_num(9.0)).any(-1).any(1).nonzero().tolist()
    assert sorted(changed) == sorted([[int(c.table[1, 1]), 7], [int(c.table[4, 0]), 4]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [None, [3, 2, 0, 4, 1, 40]])
@pytest.mark.parametrize("in_place", [True, False])
def test_append_to_malformed_lengths(dtype, counts, in_place):
    """Step after step the rows of other sequences arrive and those of a malformed length touch nothing; no step makes a
    negative length a valid one."""
    from cortex.kernels.paged_kv import kv_evict_plan, paged_attention, paged_kv_append

    lens = [9, 5, 7, 6, 4, 3]
    c = Cache(lens, 2, 32, 8, DTYPES[dtype], seed=12, room=87, tracked=True)
    most = c.width * 8
    bad = {0: -1, 2: -(1 << 62), 3: most + 1, 5: (1 << 63) - 2}
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([bad.get(b, n) for b, n in enumerate(lens)], device=DEV)
    pools = _append_plain(c, torch.zeros(0, 2, 32), torch.zeros(0, 2, 32), [0] * 7, None, DTYPES[dtype])
    per = counts or [1] * 6
    off = [sum(per[:i]) for i in range(7)]
    want = list(lens)
    for _ in range(2):
        k, v = (torch.randn(off[-1], 2, 32, generator=c.g).to(torch.bfloat16) for _ in range(2))
        lengths = paged_kv_append(c.pages, k.to(DEV), v.to(DEV), c.block_table, lengths, err_flag=flag,
                                  offsets=None if counts is None else torch.tensor(off, device=DEV),
                                  new_lengths=lengths if in_place else None)
        for b in (1, 4):
            slots = torch.arange(want[b], want[b] + per[b])
            at = c.at(b, slots)
            for name, x in (("k", k), ("v", v)):
                x = x[off[b]:off[b + 1]]
                if dtype == "int8":
                    pools[name][at], pools[name + "_scale"][at] = codes(x.float())
                else:
                    pools[name][at] = x.to(DTYPES[dtype])
            pools["weight"][at] = 0.0
            pools["position"][at] = slots[:, None].int()
            want[b] += per[b]
        assert lengths.tolist() == [-1, want[1], -(1 << 62), most, want[4], most] and int(flag) == 4
        _same(c, pools)
    for n in (0, 1):
        assert kv_evict_plan(c.pages, c.block_table, lengths, 2, n).lengths.tolist() == [-1, 2, -(1 << 62), 2, 2, 2]
    out = paged_attention(c.query(4).to(DEV), c.pages, c.block_table, lengths)
    assert (out[[0, 2]] == 0).all()


# ------------------------------------------------------------------------------- eviction


def _evict_plain(c, budget, recent):
    """(dst, src, counts) lists and the pools after the moves."""
    pools = {n: getattr(c.pages, n).cpu().clone() for n in ("k", "v", "k_scale", "v_scale", "weight", "position")
             if getattr(c.pages, n) is not None}
    weight, position = pools["weight"].clone(), pools["position"].clone()
    moves = []
    for b, n in enumerate(c.lens):
        at = c.at(b, torch.arange(n))
        for h in range(c.kv_heads):
            dst, src = evict64(weight[at][:, h], position[at][:, h], n, budget, recent)
            moves.append((dst, src))
            for d, s in zip(dst, src):
                for t in pools.values():
                    t[c.table[b, d // c.page], h, d % c.page] = t[c.table[b, s // c.page], h, s % c.page]
    return moves, pools


def _evict(c, budget, recent, **kw):
    from cortex.kernels.paged_kv import kv_evict_apply, kv_evict_plan

    plan = kv_evict_plan(c.pages, c.block_table, c.lengths, budget, recent, **kw)
    kv_evict_apply(c.pages, c.block_table, plan, **{k: v for k, v in kw.items() if k == "err_flag"})
    return plan


def _check_evict(c, budget, recent, **kw):
    moves, pools = _evict_plain(c, budget, recent)
    plan = _evict(c, budget, recent, **kw)
    room = min(kw.get("max_length", c.width * c.page), c.width * c.page)
    cap = max(0, min(budget, room - budget))
    H = c.kv_heads
    assert plan.dst.shape == plan.src.shape == (len(c.lens), H, cap)
    for i, (dst, src) in enumerate(moves):
        b, h = divmod(i, H)
        assert int(plan.counts[b, h]) == len(dst) == len(src)
        assert plan.dst[b, h].tolist() == dst + [-1] * (cap - len(dst))
        assert plan.src[b, h].tolist() == src + [-1] * (cap - len(src))
    assert plan.lengths.tolist() == [min(n, budget) for n in c.lens]
    _same(c, pools)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,budget,recent", [
    ([100, 64, 63, 65, 0, 1], 64, 16), ([1500, 1100, 3000], 1000, 100), ([50, 20], 1, 0), ([50, 20], 0, 0), ([40], 33, 33),
    ([300], 200, 200), ([4097, 4096, 5000], 4000, 0)])
def test_evict(dtype, lens, budget, recent):
    c = Cache(lens, 2, 64, 16, DTYPES[dtype], seed=budget, tracked=True)
    # positions in no order, as after earlier evictions
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        c.pages.position[at[0].to(DEV), :, at[2].to(DEV)] = torch.stack(
            [torch.randperm(n, generator=c.g) for _ in range(2)], 1).int().to(DEV) + 1000
    _check_evict(c, budget, recent)


def test_evict_equal_positions():
    """More slots at the newest positions than the budget holds: they are equal, the lower ones stay."""
    c = Cache([100], 2, 64, 16, torch.bfloat16, seed=77, tracked=True)
    c.pages.position.fill_(7)
    _check_evict(c, 30, 1)


@pytest.mark.parametrize("lens,budget", [([70000], 30000), ([32768, 32769, 33000], 5000)])
def test_evict_long(lens, budget):
    c = Cache(lens, 1, 16, 64, torch.bfloat16, seed=1, tracked=True)
    moves, _ = _evict_plain(Cache([10], 1, 16, 64, torch.bfloat16, tracked=True), 5, 1)
    plan = _evict(c, budget, 999)
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        dst, src = evict64(c.weight[at][:, 0], c.position[at][:, 0], n, budget, 999)
        assert plan.dst[b, 0, :len(dst)].tolist() == dst and plan.src[b, 0, :len(src)].tolist() == src
        assert int(plan.counts[b, 0]) == len(dst) and (plan.dst[b, 0, len(dst):] == -1).all()
    assert moves


@pytest.mark.parametrize("values", ["random", "ties", "swapped"])
@pytest.mark.parametrize("most", [2048, 2049, 8192, 8193, 16384, 16385, 32768, 32769])
def test_evict_around_the_forms_of_the_plan(values, most):
    """The longest sequence that a form of the plan takes (one, two and four runs of slots a thread, or any number), and one
    more; with every kept slot in the upper half all of the lower half is filled from there."""
    lens, budget = [most, most - 1, most // 2 + 1, most - 9, 3], most // 2
    c = Cache(lens, 2, 16, 64, torch.bfloat16, seed=most, tracked=True)
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        if values == "ties":
            c.weight[at] = torch.randint(0, 3, (n, 2), generator=c.g).float()
        elif values == "swapped":
            c.weight[at] = torch.where(torch.arange(n) < n // 2, 0.0, 1.0)[:, None] + torch.rand(n, 2, generator=c.g) / 2
        c.position[at] = torch.stack([torch.randperm(n, generator=c.g) for _ in range(2)], 1).int()
    c.pages.weight.copy_(c.weight)
    recent = 0 if values == "swapped" else 33
    c.pages.position.copy_(c.position)
    pools = {n: getattr(c.pages, n).cpu() for n in ("k", "v", "weight", "position")}
    plan = _evict(c, budget, recent, max_length=most)
    cap = min(budget, most - budget)
    assert plan.dst.shape == plan.src.shape == (len(lens), 2, cap)
    assert plan.lengths.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        at = c.at(b, torch.arange(n))
        for h in range(2):
            dst, src = evict64(c.weight[at][:, h], c.position[at][:, h], n, budget, recent)
            if values == "swapped" and n == most and most % 2 == 0:
                assert len(dst) == most // 2
            assert int(plan.counts[b, h]) == len(dst) == len(src)
            assert plan.dst[b, h].tolist() == dst + [-1] * (cap - len(dst))
            assert plan.src[b, h].tolist() == src + [-1] * (cap - len(src))
            d, s = torch.tensor(dst, dtype=torch.int64), torch.tensor(src, dtype=torch.int64)
            for t in pools.values():
                t[c.table[b, d // 64].long(), h, d % 64] = t[c.table[b, s // 64].long(), h, s % 64]
    _same(c, pools)


@pytest.mark.parametrize("values", ["ties", "one", "special", "tiny"])
@pytest.mark.parametrize("n,budget", [(90, 37), (2500, 1024)])
def test_evict_equal_and_special_weights(values, n, budget):
    c = Cache([n, n], 2, 32, 8, torch.bfloat16, seed=n, tracked=True)
    if values == "ties":
        w = torch.randint(0, 3, c.weight.shape, generator=c.g).float()
    elif values == "one":
        w = torch.full(c.weight.shape, 0.25)
    elif values == "tiny":  # neighbouring values, subnormal ones among them
        w = (torch.randint(0, 1 << 12, c.weight.shape, generator=c.g).int() + (1 << 22)).view(torch.float32)
    else:
        pick = torch.tensor([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1.0, -1.0, 2.0])
        w = pick[torch.randint(0, 8, c.weight.shape, generator=c.g)]
        w[w.isnan()] = torch.where(torch.rand(int(w.isnan().sum()), generator=c.g) < 0.5, float("nan"), -float("nan"))
    c.pages.weight.copy_(w)
    c.weight = w
    _check_evict(c, budget, 5)


def test_evict_bad_pages_and_max_length():
    c = Cache([100, 90], 2, 32, 8, torch.bfloat16, seed=2, tracked=True)
    _check_evict(c, 60, 8, max_length=100)
    c = Cache([100, 90], 2, 32, 8, torch.bfloat16, seed=2, tracked=True)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.block_table[0, 3] = -7  # slots 24 .. 31 of the first sequence
    plan = _evict(c, 60, 8, err_flag=flag)
    assert int(flag) == 4
    # slots without a page are the first to go: all of them holes, and none of them is filled
    assert all(set(range(24, 32)) <= set(plan.dst[0, h].tolist()) for h in range(2))
    flag.zero_()
    plan = _evict(c, 60, 8, max_length=80, err_flag=flag)  # the lengths are cut to 80
    assert int(flag) == 4 and plan.lengths.tolist() == [60, 60] and int(plan.src.max()) < 80


def test_apply_refuses_moves_outside_the_table():
    from cortex.kernels.paged_kv import EvictPlan, kv_evict_apply

    c = Cache([40], 1, 32, 8, torch.bfloat16, seed=6, tracked=True)
    before = c.gk.clone()
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = torch.tensor([[[-1, 40, 0, 1 << 30]]], dtype=torch.int32, device=DEV)
    plan = EvictPlan(bad, torch.tensor([[[3, 3, -9, 3]]], dtype=torch.int32, device=DEV),
                     torch.tensor([[400]], dtype=torch.int32, device=DEV), c.lengths)  # more moves than there are
    kv_evict_apply(c.pages, c.block_table, plan, err_flag=flag)
    assert int(flag) == 4 and torch.equal(c.gk.nan_to_num(9.0), before.nan_to_num(9.0))


# ------------------------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_steps_under_a_budget(dtype):
    """Append, attend with accumulation, evict, step after step: against the same steps on plain lists of rows.  The plain
    side follows the plan that the kernel made (weights differ by rounding) and checks it against the kernel's own weights."""
    from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    B, H, kv, D, page, budget = 3, 4, 2, 64, 8, 24
    g = torch.Generator().manual_seed(21)
    pages = KVPages.allocate(B * 5 + 1, kv, page, D, DTYPES[dtype], tracked=True)
    table = torch.randperm(B * 5 + 1, generator=g)[:B * 5].reshape(B, 5).int()
    gt = table.to(DEV)
    lengths = torch.zeros(B, dtype=torch.int64, device=DEV)
    rows = [[[] for _ in range(kv)] for _ in range(B)]  # (k, v) of every slot
    for step in range(60):
        k, v = (torch.randn(B, kv, D, generator=g).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(B, H, D, generator=g).to(pages.query_dtype)
        pos = torch.full((B,), step, dtype=torch.int64, device=DEV)
        x = [t.to(torch.float32) if dtype == "fp32" else t for t in (k, v)]
        lengths = paged_kv_append(pages, x[0].to(DEV), x[1].to(DEV), gt, lengths, positions=pos)
        for b in range(B):
            for h in range(kv):
                kept = []
                for t in (k, v):
                    if dtype == "int8":
                        code, s = codes(t[b, h].float())
                        kept.append(code.double() * s.double())
                    else:
                        kept.append(t[b, h].double())
                rows[b][h].append(tuple(kept))
        got = paged_attention(q.to(DEV), pages, gt, lengths, accumulate=True).double().cpu()
        for b in range(B):
            for h in range(H):
                ks, vs = (torch.stack([r[i] for r in rows[b][h // 2]]) for i in range(2))
                p = torch.softmax(ks @ q[b, h].double() / 8, 0)
                # 2^-15 for the probabilities, 2^-8 for the result, fp32 sums below 1e-4
                half = 2.0 ** -8 if dtype != "fp32" else 0.0
                tol = (2.0 ** -15 + 1e-4) * (p @ vs.abs()) + half * (p @ vs).abs()
                assert ((got[b, h] - p @ vs).abs() <= tol).all(), (step, b, h)
        if step % 7 == 6:
            plan = kv_evict_plan(pages, gt, lengths, budget, 6)
            n = int(lengths[0])
            weight, position = pages.weight.cpu(), pages.position.cpu()
            kv_evict_apply(pages, gt, plan)
            for b in range(B):
                slots = torch.arange(n)
                at = table[b][slots // page].long(), slice(None), slots % page
                for h in range(kv):
                    dst, src = evict64(weight[at][:, h], position[at][:, h], n, budget, 6)
                    assert plan.dst[b, h].tolist()[:len(dst)] == dst and plan.src[b, h].tolist()[:len(src)] == src
                    for d, s in zip(dst, src):
                        rows[b][h][d] = rows[b][h][s]
                    del rows[b][h][budget:]
            lengths = plan.lengths
    assert lengths.tolist() == [min(60, budget + 60 % 7)] * B


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeated_calls_and_streams_give_the_same_bits(dtype):
    c = Cache([3000, 100, 5, 900], 2, 128, 16, DTYPES[dtype], seed=31)
    q = c.query(8).to(DEV)
    first = attend(c, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            outs.append(attend(c, q))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_steps(dtype):
    """A decode step captured into a graph (append in place, attention, eviction) and replayed, with eager work and
    synchronisation between the replays, against the same steps run eagerly."""
    from cortex.kernels.paged_kv import kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    def make():
        return Cache([30, 4, 17], 2, 64, 8, DTYPES[dtype], seed=41, room=60, tracked=True)

    a, b = make(), make()
    k, v, q = (torch.zeros(3, h, 64, dtype=a.pages.query_dtype, device=DEV) for h in (2, 2, 8))

    def step(c):
        paged_kv_append(c.pages, k, v, c.block_table, c.lengths, new_lengths=c.lengths)
        out = paged_attention(q, c.pages, c.block_table, c.lengths, accumulate=True)
        plan = kv_evict_plan(c.pages, c.block_table, c.lengths, 40, 4)
        kv_evict_apply(c.pages, c.block_table, plan)
        c.lengths.copy_(plan.lengths)
        return out

    warm = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    g = torch.Generator(DEV).manual_seed(1)
    for i in range(20):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        graph.replay()
        want = step(b)
        if i % 3 == 0:
            torch.cuda.synchronize()
            attend(b, q, accumulate=False)
        assert torch.equal(out, want), i
        assert torch.equal(a.lengths, b.lengths)
    for n in ("k", "v", "weight", "position"):
        x, y = getattr(a.pages, n), getattr(b.pages, n)
        assert torch.equal(x.float().nan_to_num(9.0), y.float().nan_to_num(9.0)), n


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_graphs_at_once(dtype):
    """Two graphs over the same pages (long enough for a join), replayed at once on two streams: each has its workspace."""
    c = Cache([5000, 1300, 0, 40], 2, 64, 16, DTYPES[dtype], seed=51)
    qs = [c.query(8).to(DEV), c.query(8).to(DEV)]
    want = [attend(c, q) for q in qs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attend(c, q))
        graphs.append(graph)
    torch.cuda.synchronize()
    for i in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = attend(c, qs[i % 2])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[i % 2])
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), i


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_past_four_gib(dtype):
    """The same rows in pages at the end of a pool of more than 4 GiB and in a small one: the same bits."""
    from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    dt = DTYPES[dtype]
    es = torch.empty(0, dtype=dt).element_size()
    big = (9 << 29) // (2 * 64 * 128 * es)  # pages of 4.5 GiB
    g = torch.Generator().manual_seed(61)
    k, v = (torch.randn(900, 2, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn(3, 8, 128, generator=g).to(torch.float32 if dtype == "fp32" else torch.bfloat16).to(DEV)
    off = torch.tensor([0, 500, 500, 900], device=DEV)
    got = []
    for num in (30, big):
        pages = KVPages.allocate(num, 2, 64, 128, dt, tracked=True)
        table = (num - 1 - torch.randperm(30, generator=torch.Generator().manual_seed(1))).reshape(3, 10).int().to(DEV)
        n = paged_kv_append(pages, k, v, table, torch.zeros(3, dtype=torch.int64, device=DEV), offsets=off)
        out = [n, paged_attention(q, pages, table, n, accumulate=True)]
        plan = kv_evict_plan(pages, table, n, 200, 50)
        kv_evict_apply(pages, table, plan)
        out += [*plan, paged_attention(q, pages, table, plan.lengths), pages.weight[table.long()], pages.position[table.long()],
                pages.k[table.long()]]
        got.append([t.cpu() for t in out])
        del pages
        torch.cuda.empty_cache()
    assert int(got[0][4].min()) == 0 and int(got[0][4].max()) > 0  # (an empty sequence and ones that were cut)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_empty_batches_and_caches():
    from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    pages = KVPages.allocate(2, 2, 8, 32, tracked=True)
    none = torch.empty(0, 3, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV)
    rows = torch.empty(0, 2, 32, dtype=torch.bfloat16, device=DEV)
    assert paged_attention(rows, pages, *none).shape == (0, 2, 32)
    assert paged_kv_append(pages, rows, rows, *none).shape == (0,)
    plan = kv_evict_plan(pages, *none, 4, 1)
    kv_evict_apply(pages, none[0], plan)
    table, lengths = torch.empty(3, 0, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    q = torch.ones(3, 4, 32, dtype=torch.bfloat16, device=DEV)
    assert (paged_attention(q, pages, table, lengths) == 0).all()
    assert kv_evict_plan(pages, table, lengths, 4, 1).lengths.tolist() == [0, 0, 0]


# ------------------------------------------------------------------------------- refusals


def test_refused_tensors():
    from cortex.kernels.paged_kv import KVPages, paged_attention, paged_kv_append

    c = Cache([40, 9], 2, 64, 16, torch.bfloat16, tracked=True)
    q = c.query(4).to(DEV)
    for out in (torch.empty(1, 4, 64, device=DEV, dtype=q.dtype).expand(2, 4, 64),
                torch.empty(2, 1, 64, device=DEV, dtype=q.dtype).expand(2, 4, 64),
                torch.empty(512, device=DEV, dtype=q.dtype).as_strided((2, 4, 64), (192, 64, 1)),
                torch.empty(512, device=DEV, dtype=q.dtype).as_strided((2, 4, 64), (64, 32, 1))):
        with pytest.raises(ValueError, match="overlap itself"):
            paged_attention(q, c.pages, c.block_table, c.lengths, out=out)
    heads_first = torch.empty(4, 2, 64, device=DEV, dtype=q.dtype).transpose(0, 1)
    want = paged_attention(q, c.pages, c.block_table, c.lengths)
    assert torch.equal(paged_attention(q, c.pages, c.block_table, c.lengths, out=heads_first), want)
    with pytest.raises(RuntimeError, match="backward"):
        paged_attention(q, c.pages, c.block_table, c.lengths, out=torch.empty_like(q, requires_grad=True))
    off = torch.zeros(c.weight.numel() + 1, device=DEV)[1:].view(c.weight.shape)
    with pytest.raises(ValueError, match="16-byte"):
        KVPages(c.gk, c.gv, weight=off)
    with pytest.raises(ValueError, match="gradients"):
        KVPages(c.gk, c.gv, weight=c.weight.to(DEV).requires_grad_())
    buf = torch.tensor([20, 5, 7], device=DEV)
    rows = torch.zeros(2, 2, 64, device=DEV, dtype=q.dtype)
    with pytest.raises(Exception, match="overlaps"):
        paged_kv_append(c.pages, rows, rows, c.block_table, buf[:2], new_lengths=buf[1:])
    assert buf.tolist() == [20, 5, 7]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["planes", "columns", "halves", "every other", "heads", "rows outside"])
def test_keys_and_values_in_one_buffer(dtype, layout):
    """Views of one allocation are written like pools of their own."""
    from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_kv_append

    def z(*shape):
        return torch.zeros(*shape, dtype=DTYPES[dtype], device=DEV)

    n, H, S, D = 6, 2, 8, 32
    if layout == "planes":
        both = z(n, 2, H, S, D)
        k, v = both[:, 1], both[:, 0]
    elif layout == "columns":
        both = z(n, H, S, 2 * D)
        k, v = both[..., :D], both[..., D:]
    elif layout == "halves":
        both = z(2 * n, H, S, D)
        k, v = both[:n], both[n:]
    elif layout == "every other":
        both = z(2 * n, H, S, D)
        k, v = both[1::2], both[::2]
    elif layout == "heads":
        both = z(n, S, 2 * H, D)
        k, v = both[:, :, :H].transpose(1, 2), both[:, :, H:].transpose(1, 2)
    else:
        both = z(2, S, n, H, D)
        k, v = (both[i].permute(1, 2, 0, 3) for i in (0, 1))
    scales = {"k_scale": torch.zeros(n, H, S, device=DEV), "v_scale": torch.zeros(n, H, S, device=DEV)} if dtype == "int8" else {}
    tracked = [{"weight": torch.zeros(n, H, S, device=DEV), "position": torch.zeros(n, H, S, dtype=torch.int32, device=DEV)}
               for _ in range(2)]
    one = KVPages(k, v, **scales, **tracked[0])
    two = KVPages(z(n, H, S, D), z(n, H, S, D), **{a: t.clone() for a, t in scales.items()}, **tracked[1])
    g = torch.Generator(DEV).manual_seed(1)
    rows = [torch.randn(37, H, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
    table = torch.tensor([[3, 0, 5], [1, 4, 2]], dtype=torch.int32, device=DEV)
    for p in (one, two):
        lengths = paged_kv_append(p, *rows, table, torch.zeros(2, dtype=torch.int64, device=DEV),
                                  offsets=torch.tensor([0, 20, 37], device=DEV))
        kv_evict_apply(p, table, kv_evict_plan(p, table, lengths, 9, 4))
    for a in ("k", "v", "k_scale", "v_scale", "position"):
        if getattr(one, a) is not None:
            assert torch.equal(getattr(one, a), getattr(two, a)), a
    assert not torch.equal(one.k, one.v)


def test_pools_whose_rows_share_memory():
    """They are read like others, and not written."""
    from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    c = Cache([40, 9], 1, 64, 16, torch.bfloat16, tracked=True)
    q = c.query(4)
    want, _, tol, _ = attention64(c, q)
    more = {n: getattr(c.pages, n).expand(-1, 2, -1).contiguous() for n in ("weight", "position")}
    wide = KVPages(c.gk.expand(-1, 2, -1, -1), c.gv.expand(-1, 2, -1, -1), **more)
    check(paged_attention(q.to(DEV), wide, c.block_table, c.lengths), want, tol, "expanded")
    tied = KVPages(c.gk, c.gk, weight=c.pages.weight, position=c.pages.position)
    before = c.gk.clone()
    for pages, heads in ((wide, 2), (tied, 1)):
        rows = torch.ones(2, heads, 64, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(Exception, match="share memory"):
            paged_kv_append(pages, rows, rows, c.block_table, c.lengths)
        with pytest.raises(Exception, match="share memory"):
            kv_evict_apply(pages, c.block_table, kv_evict_plan(pages, c.block_table, c.lengths, 8, 2))
    assert torch.equal(c.gk.nan_to_num(9.0), before.nan_to_num(9.0))


def test_refused_tangents():
    """The tangent of a forward-mode dual tensor would be lost."""
    from torch.autograd import forward_ad

    from cortex.kernels.paged_kv import KVPages, paged_attention, paged_kv_append

    c = Cache([40, 9], 2, 64, 16, torch.bfloat16, room=1, tracked=True)
    q, rows = c.query(4).to(DEV), torch.ones(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    want = paged_attention(q, c.pages, c.block_table, c.lengths)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        before = c.gk.clone()
        for k, v in [(dual(rows), rows), (rows, dual(rows))]:
            with pytest.raises(RuntimeError, match="tangent"):
                paged_kv_append(c.pages, k, v, c.block_table, c.lengths)
        assert torch.equal(c.gk.nan_to_num(9.0), before.nan_to_num(9.0))
        for bad in [dual(q), dual(q)[:], dual(q).transpose(0, 1).contiguous().transpose(0, 1)]:
            for grad in (True, False):
                with pytest.raises(RuntimeError, match="tangent"), torch.set_grad_enabled(grad):
                    paged_attention(bad, c.pages, c.block_table, c.lengths)
        with pytest.raises(RuntimeError, match="tangent"):
            paged_attention(q, c.pages, c.block_table, c.lengths, out=dual(q))
        with pytest.raises(RuntimeError, match="tangent"):
            KVPages(c.gk, dual(c.gv))
        assert torch.equal(paged_attention(forward_ad.unpack_dual(dual(q)).primal, c.pages, c.block_table, c.lengths), want)
        paged_kv_append(c.pages, rows, rows, c.block_table, c.lengths)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: paged_attention(x, c.pages, c.block_table, c.lengths), (q,), (torch.ones_like(q),))


def test_refusals():
    from cortex.kernels.paged_kv import EvictPlan, KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append

    def pool(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=DEV)

    k = pool(4, 2, 16, 64)
    scale = pool(4, 2, 16, dtype=torch.float32)
    for bad in [(k, pool(4, 2, 16, 48), {}), (k, pool(4, 2, 16, 64, dtype=torch.float32), {}), (k[0], k[0], {}),
                (k.half(), k.half(), {}), (k, k, {"k_scale": scale, "v_scale": scale}), (k.char(), k.char(), {}),
                (k.char(), k.char(), {"k_scale": scale}), (pool(4, 2, 24, 64), pool(4, 2, 24, 64), {}),
                (pool(4, 2, 4, 64), pool(4, 2, 4, 64), {}), (pool(4, 2, 16, 24), pool(4, 2, 16, 24), {}),
                (pool(4, 2, 16, 144), pool(4, 2, 16, 144), {}), (pool(4, 2, 64, 16).transpose(2, 3),) * 2 + ({},),
                (pool(4, 2, 16, 68)[..., 4:], k, {}), (k, k, {"weight": scale[:3]}), (k, k, {"position": scale}),
                (k, k, {"weight": scale.transpose(0, 1)})]:
        with pytest.raises(ValueError):
            KVPages(bad[0], bad[1], **bad[2])
    with pytest.raises(RuntimeError):
        KVPages(k.cpu(), k.cpu())
    pages = KVPages(k, k.clone())
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(2, dtype=torch.int64, device=DEV)
    q = pool(2, 4, 64)
    good = (q, pages, table, lengths)
    assert paged_attention(*good).shape == (2, 4, 64)
    for i, bad in [(0, pool(2, 3, 64)), (0, pool(3, 4, 64)), (0, pool(2, 4, 48)), (0, q.float()), (0, q[0]), (2, table.long()),
                   (2, table[0]), (2, torch.zeros(3, 2, dtype=torch.int32, device=DEV).t()), (3, lengths.int()),
                   (3, torch.zeros(3, dtype=torch.int64, device=DEV)), (3, lengths[None])]:
        with pytest.raises(ValueError):
            paged_attention(*good[:i], bad, *good[i + 1:])
    for kw in [{"accumulate": True}, {"max_length": -1}, {"out": q}, {"out": pool(2, 4, 32)}, {"out": q.float()},
               {"err_flag": lengths}]:
        with pytest.raises(ValueError):
            paged_attention(*good, **kw)
    buf = pool(2, 12, 64)  # queries and outputs in one buffer
    for ok, out in [(True, buf[:, 4:8]), (True, buf[:, 8:]), (False, buf[:, 2:6]), (False, buf[:, :4])]:
        if ok:
            paged_attention(buf[:, :4], *good[1:], out=out)
        else:
            with pytest.raises(ValueError, match="overlap"):
                paged_attention(buf[:, :4], *good[1:], out=out)
    flat = pool(3, 4, 64)
    with pytest.raises(ValueError, match="overlap"):
        paged_attention(flat[:2], *good[1:], out=flat[1:])
    with pytest.raises(RuntimeError):
        paged_attention(q.cpu(), *good[1:])
    with pytest.raises(RuntimeError, match="backward"):
        paged_attention(q.clone().requires_grad_(), *good[1:])
    with torch.no_grad():
        paged_attention(q.clone().requires_grad_(), *good[1:])
    rows = pool(2, 2, 64)
    good = (pages, rows, rows, table, lengths)
    paged_kv_append(*good)
    for i, bad in [(1, pool(3, 2, 64)), (1, pool(2, 3, 64)), (1, pool(2, 2, 48)), (1, rows.float()), (2, rows.half())]:
        with pytest.raises(ValueError):
            paged_kv_append(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError):
        paged_kv_append(pages, pool(3, 2, 64), pool(3, 2, 64), table, lengths)
    with pytest.raises(ValueError):
        paged_kv_append(pages, rows.half(), rows.half(), table, lengths)
    for kw in [{"offsets": lengths}, {"positions": torch.zeros(3, dtype=torch.int64, device=DEV)},
               {"new_lengths": lengths.int()}]:
        with pytest.raises(ValueError):
            paged_kv_append(*good, **kw)
    with pytest.raises(ValueError):
        kv_evict_plan(pages, table, lengths, 4, 1)
    tracked = KVPages.allocate(4, 2, 16, 64, tracked=True)
    for budget, recent, kw in [(-1, 0, {}), (1, -1, {}), (200, 500, {}), (1, 1, {"max_length": -2})]:
        with pytest.raises(ValueError):
            kv_evict_plan(tracked, table, lengths, budget, recent, **kw)
    plan = kv_evict_plan(tracked, table, lengths, 4, 1)
    for bad in [EvictPlan(plan.dst[:1], *plan[1:]), EvictPlan(plan.dst.long(), *plan[1:]),
                EvictPlan(plan.dst, plan.src, plan.counts[:, :1], plan.lengths)]:
        with pytest.raises(ValueError):
            kv_evict_apply(tracked, table, bad)
