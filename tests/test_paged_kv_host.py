"""Refusals of the paged K/V cache entry points, which return before any device work (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cortex import _native as nat

# the pointers are made up: where there is a GPU, a call that should have been refused and was not would follow them
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers: only where nothing can be launched")

P = 16  # a pointer that no check may follow


def pages(**kw):
    d = {"num_pages": 4, "kv_heads": 2, "page_size": 16, "head_dim": 64, "dtype": nat.BF16, "k_page": 2048, "k_head": 1024,
         "k_slot": 64, "v_page": 2048, "v_head": 1024, "v_slot": 64, "k": P, "v": P}
    d.update(kw)
    return nat.KvPagesStruct(**d)


def append(p, B=2, T=2, x=nat.BF16, k=P, st=128, sh=64, table=P, ld=3, width=3, offsets=None, lengths=P, out=P):
    return ("cortex_kv_append", p and ctypes.byref(p), B, T, x, k, st, sh, k, st, sh, table, ld, width, offsets, lengths,
            None, out, None, None)


def attention(p, B=2, heads=4, q=P, table=P, ld=300, width=300, lengths=P, most=4800, accumulate=0, out=P, ws=P, ws_bytes=1 << 40):
    return ("cortex_paged_attention", p and ctypes.byref(p), B, heads, q, 256, 64, table, ld, width, lengths, most,
            ctypes.c_float(0.125), accumulate, out, 256, 64, ws, ws_bytes, None, None)


def plan(p, B=2, table=P, ld=3, width=3, lengths=P, most=48, budget=8, recent=2, moves=P, counts=P, after=2 * P):
    return ("cortex_kv_evict_plan", p and ctypes.byref(p), B, table, ld, width, lengths, most, budget, recent, moves, moves,
            counts, after, None, None)


def apply(p, B=2, table=P, ld=3, width=3, moves=P, cap=8, counts=P):
    return ("cortex_kv_evict_apply", p and ctypes.byref(p), B, table, ld, width, moves, moves, cap, counts, None, None)


def refused(call, part, rc=-1):
    lib = nat.load()
    assert getattr(lib, call[0])(*call[1:]) == rc
    assert part.encode() in lib.cortex_last_error(), lib.cortex_last_error()


def tracked(**kw):
    return pages(weight=P, position=P, **kw)


@pytest.mark.parametrize("call", [append, attention, plan, apply], ids=lambda f: f.__name__)
def test_pages_that_no_operator_takes(call):
    for kw, part in [({"dtype": nat.F16}, "dtype"), ({"num_pages": 0}, "page count"), ({"num_pages": 1 << 31}, "page count"),
                     ({"kv_heads": 0}, "head count"), ({"page_size": 24}, "power of two"), ({"page_size": 4}, "power of two"),
                     ({"page_size": 1 << 17}, "power of two"), ({"page_size": -16}, "power of two"),
                     ({"head_dim": 0}, "head dim"), ({"head_dim": 72}, "head dim"), ({"head_dim": 256}, "head dim"),
                     ({"k": None}, "null k or v"), ({"v": None}, "null k or v"), ({"k_scale": P}, "int8 pages"),
                     ({"dtype": nat.I8}, "int8 pages"), ({"dtype": nat.I8, "k_scale": P}, "int8 pages"),
                     ({"k": 8}, "16-byte"), ({"v_slot": 68}, "16-byte"), ({"k_page": -2048}, "16-byte"),
                     ({"k_slot": 32}, "overlap")]:
        refused(call(tracked(**kw)), part)
    refused(call(None), "null pages")
    refused(call(tracked(), B=-1), "negative shape")
    refused(call(tracked(), width=-1), "negative shape")
    refused(call(tracked(), table=None), "block table")
    refused(call(tracked(), ld=2, width=3), "overlap")
    refused(call(tracked(page_size=65536), width=20000, ld=20000), "2^30")


def test_refused_appends():
    refused(append(pages(), T=3), "one token a sequence")
    refused(append(pages(), T=-1), "tokens")
    refused(append(pages(), x=nat.F16), "f32 or bf16")
    refused(append(pages(), lengths=None), "null lengths")
    refused(append(pages(), k=None), "null k or v")
    refused(append(pages(), k=8), "16-byte")
    refused(append(pages(), st=132), "16-byte")
    assert append(pages(), B=0, T=0) and getattr(nat.load(), "cortex_kv_append")(*append(pages(), B=0, T=0)[1:]) == 0


def test_per_row_arrays_off_their_alignment():
    for name in ("weight", "position"):
        for call in (append, attention, plan, apply):
            refused(call(pages(**{"weight": P, "position": P, name: 4})), "16-byte")
    for name in ("k_scale", "v_scale"):
        refused(attention(pages(dtype=nat.I8, **{"k_scale": P, "v_scale": P, name: 24})), "16-byte")


def test_new_lengths_that_overlap_an_input():
    n = 1 << 20
    for out in (n + 8, n - 8):
        refused(append(pages(), lengths=n, out=out), "overlaps")
        refused(plan(tracked(), lengths=n, after=out), "may not be lengths")
    for out in (n, n + 16, n - 8):  # offsets are one more than the sequences
        refused(append(pages(), lengths=2 * n, offsets=n, out=out), "overlaps")
    call = list(append(pages(), lengths=2 * n, out=n + 8))
    call[-4] = n  # positions
    refused(tuple(call), "overlaps")


def test_launches_of_too_many_threads():
    refused(plan(tracked(kv_heads=65535), B=65), "too many heads")
    refused(apply(pages(kv_heads=65535), B=257), "too many heads")
    refused(attention(pages(kv_heads=65535), B=129, heads=65535, most=32), "too much for one call")
    refused(attention(pages(kv_heads=1024, head_dim=64), B=16, heads=1 << 20, most=16, width=1, ld=1), "too much")
    refused(append(pages(kv_heads=65535), B=1 << 24, T=1 << 24), "too many for one call")


def test_refused_attention():
    refused(attention(pages(), heads=3), "multiple")
    refused(attention(pages(), heads=0), "multiple")
    refused(attention(pages(), B=4097), "at most 4096")
    refused(attention(pages(), B=4096, heads=1024, width=1 << 20, ld=1 << 20, most=-1), "too much for one call")
    refused(attention(pages(), ws=None), "workspace")
    refused(attention(pages(), ws=8), "workspace")
    refused(attention(pages(), ws_bytes=64), "needed", rc=-4)
    refused(attention(pages(), q=8), "16-byte")
    refused(attention(pages(), accumulate=1), "weight")
    refused(attention(pages(), q=None), "null q")
    refused(attention(pages(), lengths=None), "null q")
    assert nat.load().cortex_paged_attention(*attention(pages(), B=0)[1:]) == 0


def test_refused_evictions():
    refused(plan(pages()), "weight and position")
    refused(plan(tracked(), budget=-1), "negative budget")
    refused(plan(tracked(), budget=1, recent=2), "exceeds the budget")
    refused(plan(tracked(), moves=None), "null pointer")
    refused(plan(tracked(), after=P), "may not be lengths")
    refused(apply(pages(), cap=-1), "negative cap")
    refused(apply(pages(), counts=None), "null pointer")
    lib = nat.load()
    assert lib.cortex_kv_evict_plan(*plan(tracked(), B=0)[1:]) == 0 and lib.cortex_kv_evict_apply(*apply(pages(), cap=0)[1:]) == 0


def test_pools_whose_rows_share_memory_are_not_written():
    n = 1 << 20
    for kw in [{"k_head": 0}, {"v_head": 0}, {"k_page": 0}, {"k_page": 1024}, {"v_page": 2032}, {"k_head": 512}, {"k_slot": 80}]:
        for call in (append, apply):
            refused(call(pages(v=n, **kw)), "share memory")
    for shift in (0, 32, 64, 1024, 2048, 4096, 8192 - 64):  # k and v in one buffer, `shift` elements apart
        for call in (append, apply):
            refused(call(pages(k=n, v=n + 2 * shift)), "share memory")
            refused(call(pages(k=n + 2 * shift, v=n)), "share memory")
