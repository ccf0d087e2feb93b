"""Refusals of the entry points for rotation, copies, bounds and selections, which return before any device work (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cortex import _native as nat

# the pointers are made up: where there is a GPU, a call that should have been refused and was not would follow them
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: only where nothing can be launched")

P = 16  # a pointer that no check may follow
V = 1 << 20


def pages(**kw):
    d = {"num_pages": 4, "kv_heads": 2, "page_size": 16, "head_dim": 64, "dtype": nat.BF16, "k_page": 2048, "k_head": 1024,
         "k_slot": 64, "v_page": 2048, "v_head": 1024, "v_slot": 64, "k": P, "v": V, "bounds": P}
    d.update(kw)
    return nat.KvPagesStruct(**d)


def ref(p):
    return p and ctypes.byref(p)


def copy(p, to=None, n=2, src=P, dst=P):
    return "cortex_kv_copy_pages", ref(p), ref(to or p), n, src, dst, None, None


def bounds(p, B=2, table=P, ld=3, width=3, lengths=P, most=48, since=None, new=-1):
    return "cortex_kv_block_bounds", ref(p), B, table, ld, width, lengths, most, since, new, None, None


def select(p, B=2, heads=4, q=P, sb=256, sh=64, table=P, ld=300, width=300, lengths=P, most=4800, count=8, first=1, recent=1,
           out=4 * V, after=2 * V, ws=P, ws_bytes=1 << 40):
    return ("cortex_kv_select", ref(p), B, heads, q, sb, sh, table, ld, width, lengths, most, count, first, recent, out, after,
            ws, ws_bytes, None, None)


def tables(p, B=2, heads=4, q=P, table=P, ld=600, sh=300, width=300, lengths=P, most=4800, out=P, ws=P, ws_bytes=1 << 40):
    return ("cortex_paged_attention_tables", ref(p), B, heads, q, 256, 64, table, ld, sh, width, lengths, most,
            ctypes.c_float(0.125), 0, out, 256, 64, ws, ws_bytes, None, None)


def rope(T=4, heads=2, kv=1, dim=64, dtype=nat.BF16, q=P, st=192, sh=64, k=P, positions=P, n_axes=1, pairs=32, freq=P, norm=1,
         eps=1e-6, gain=P, gain_dtype=nat.F32, out=P):
    return ("cortex_qk_norm_rope", T, heads, kv, dim, dtype, q, st, sh, k, st, sh, positions, 1, 0, n_axes, pairs, freq, None,
            0, norm, ctypes.c_float(eps), gain, gain, gain_dtype, out, st, sh, out, st, sh, None, None)


def refused(call, part, rc=-1):
    lib = nat.load()
    assert getattr(lib, call[0])(*call[1:]) == rc
    assert part.encode() in lib.cortex_last_error(), lib.cortex_last_error()


def accepted(call):
    assert getattr(nat.load(), call[0])(*call[1:]) == 0


@pytest.mark.parametrize("call", [copy, bounds, select, tables], ids=lambda f: f.__name__)
def test_pages_that_no_operator_takes(call):
    for kw, part in [({"dtype": nat.F16}, "dtype"), ({"num_pages": 0}, "page count"), ({"kv_heads": 0}, "head count"),
                     ({"page_size": 24}, "power of two"), ({"head_dim": 72}, "head dim"), ({"k": None}, "null k or v"),
                     ({"k_scale": P}, "int8 pages"), ({"dtype": nat.I8}, "int8 pages"), ({"k": 8}, "16-byte"),
                     ({"k_slot": 32}, "overlap")]:
        refused(call(pages(**kw)), part)
    refused(call(None, **({"to": pages()} if call is copy else {})), "null pages")


@pytest.mark.parametrize("call", [bounds, select, tables], ids=lambda f: f.__name__)
def test_tables_and_lengths(call):
    refused(call(pages(), B=-1), "negative shape")
    refused(call(pages(), table=None), "block table")
    refused(call(pages(), lengths=None), "null")
    refused(call(pages(), ld=2), "overlap")
    accepted(call(pages(), B=0))


def test_refused_copies():
    for kw in ({"kv_heads": 1}, {"page_size": 8}, {"head_dim": 48}, {"dtype": nat.F32, "k_slot": 64}):
        refused(copy(pages(), pages(**kw)), "different shapes")
    for name in ("weight", "position", "bounds"):
        refused(copy(pages(bounds=None, **{name: P}) if name != "bounds" else pages(), pages(bounds=None)), "both pools")
    refused(copy(pages(bounds=8)), "16-byte")
    refused(copy(pages(), n=-1), "negative")
    refused(copy(pages(), src=None), "null pointer")
    refused(copy(pages(), dst=None), "null pointer")
    refused(copy(pages(), n=1 << 30), "too many")
    accepted(copy(pages(), n=0, src=None, dst=None))
    for kw in ({"k_head": 0}, {"v_page": 0}, {"v": P}, {"k_page": 1024}):
        refused(copy(pages(), pages(**kw)), "share memory")
        refused(copy(pages(**kw)), "share memory")


def test_refused_bounds():
    refused(bounds(pages(bounds=None)), "aligned bounds")
    refused(bounds(pages(bounds=8)), "aligned bounds")
    refused(bounds(pages(kv_heads=65535), B=1 << 24, ld=1, width=1), "too many")
    accepted(bounds(pages(), B=0, most=0))


def test_refused_selections():
    refused(select(pages(bounds=None)), "aligned bounds")
    refused(select(pages(), heads=3), "multiple")
    refused(select(pages(), heads=0), "multiple")
    refused(select(pages(), heads=4096), "multiple")
    for kw in ({"count": 0}, {"count": 1}, {"first": -1}, {"recent": 0}, {"first": 8}, {"recent": 8},
               {"first": (1 << 63) - 1, "recent": 2}):
        refused(select(pages(), **kw), "has to hold")
    refused(select(pages(), q=None), "null pointer")
    refused(select(pages(), after=None), "null pointer")
    refused(select(pages(), out=None), "null table")
    for after in (P, P + 8, P - 8):
        refused(select(pages(), after=after), "overlap")
    refused(select(pages(), out=P + 2396), "overlap")
    refused(select(pages(), out=2 * V, table=2 * V + 4), "overlap")
    refused(select(pages(), q=8), "16-byte")
    refused(select(pages(), sb=252), "16-byte")
    refused(select(pages(), ws=None), "workspace")
    refused(select(pages(), ws=8), "workspace")
    refused(select(pages(), ws_bytes=64), "needed", rc=-4)
    refused(select(pages(kv_heads=65535, head_dim=64), heads=65535, B=1 << 12, out=1 << 60), "too much")
    lib = nat.load()
    size = lib.cortex_kv_select_workspace_bytes
    assert size(ref(pages()), 2, 4800, 8) == 2 * 2 * 304 * 4
    assert size(ref(pages()), 2, 4800, 300) == 0 and size(ref(pages()), 2, 128, 8) == 0
    assert size(None, 2, 4800, 8) == 0 and size(ref(pages()), -1, 4800, 8) == 0 and size(ref(pages()), 2, -1, 8) == 0


def test_selections_whose_tensors_meet():
    """Workgroups write while others still read: an output or the workspace that overlaps what is read, or another of them,
    is refused, at its first byte and at its last one."""
    # 4 pages of 2 heads x 64 in bf16, 2 sequences of up to 300 blocks, 4 query heads, 8 blocks kept
    size = {"q": 2 * (256 + 3 * 64 + 64), "table": 4 * 600, "lengths": 16, "bounds": 4 * 2 * 2 * 64 * 2, "out": 4 * 2 * 2 * 8,
            "after": 16, "ws": 4 * 2 * 2 * 304}
    places = {name: (i + 2) * V for i, name in enumerate(size)}

    def with_places(**kw):
        at = {**places, **kw}
        bounds = at.pop("bounds")
        return select(pages(bounds=bounds), **at)

    for written in ("after", "out", "ws"):
        for other in size:
            if other == written:
                continue
            for at in (places[other], places[other] + size[other] - 16, places[other] - size[written] + 16):
                refused(with_places(**{written: at}), "overlap")
    # the sizes that this goes by do not wrap around
    refused(with_places(B=1 << 40, ld=1 << 40), "too much")
    # rows far apart: each of them, from either end, and what lies between them is nobody's
    far = 1 << 40
    for place in (places["table"], places["table"] + far):
        refused(with_places(ld=far // 4, after=place), "overlap the block table")
    refused(with_places(ld=1 << 62, after=places["table"] + 1184), "overlap the block table")
    for sb, sh in ((far // 2, 64), (64, far // 2), (-far // 2, 64), (64, -far // 2), (-far // 2, -64)):
        refused(with_places(q=1 << 44, sb=sb, sh=sh, after=(1 << 44) + 2 * (sb + sh)), "overlap the queries")
    refused(with_places(sb=64, sh=1 << 61, q=1 << 44, after=(1 << 44) + 2 * 64), "overlap the queries")
    refused(with_places(sb=64, sh=-(1 << 61), q=1 << 44, after=(1 << 44) + 2 * 64), "overlap the queries")
    for kw in ({"ld": far // 4, "after": places["table"] + far // 2}, {"sb": far // 2, "after": places["q"] + far // 2}):
        refused(with_places(ws=None, **kw), "workspace")  # (past the outputs, to what is refused next)


def test_refused_tables_by_key_head():
    refused(tables(pages(), sh=299), "overlap")
    refused(tables(pages(), sh=-1), "overlap")
    refused(tables(pages(), heads=3), "multiple")
    refused(tables(pages(), ws=None), "workspace")


def test_refused_rotations():
    refused(rope(T=-1), "tokens")
    refused(rope(heads=-1), "heads")
    refused(rope(heads=65535, kv=1), "heads")
    for dim in (0, 4, 12, 264):
        refused(rope(dim=dim, pairs=0), "head dim")
    for pairs in (-8, 4, 12, 40):
        refused(rope(pairs=pairs), "pairs")
    refused(rope(dtype=nat.F16), "f32 or bf16")
    refused(rope(norm=0), "gains")
    refused(rope(gain_dtype=nat.I8), "gains")
    refused(rope(eps=-1.0), "negative eps")
    refused(rope(eps=float("nan")), "negative eps")
    refused(rope(n_axes=0), "axes")
    for name in ("q", "k", "positions", "freq", "out"):
        refused(rope(**{name: None}), "null pointer")
    refused(rope(q=8), "16-byte")
    refused(rope(st=196), "16-byte")
    refused(rope(gain=8), "gains must")
    accepted(rope(T=0))
    accepted(rope(heads=0, kv=0))
    # the tensors themselves have to be on the GPU
    from cortex.kernels.rotary import qk_norm_rope, rotary_frequencies

    q = torch.zeros(4, 2, 64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        qk_norm_rope(q, q, torch.arange(4), rotary_frequencies(64, device="cpu"))


def test_a_table_by_key_heads_of_the_right_size_only():
    from types import SimpleNamespace

    from cortex.kernels import paged_kv

    pages_like = SimpleNamespace(index=-1, kv_heads=2)
    lengths = torch.zeros(3, dtype=torch.int64)
    table = torch.zeros(3, 2, 5, dtype=torch.int32)
    assert paged_kv._common("x", pages_like, table, lengths, None, True) == (3, 10, 5)
    for bad in (table[:, :1].contiguous(), table[:, :, :4], table.long(), table[:2]):
        with pytest.raises(ValueError):
            paged_kv._common("x", pages_like, bad, lengths, None, True)
