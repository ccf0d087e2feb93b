"""Paged K/V cache on gfx950: append, attention of one new token, eviction by accumulated weight.

The keys and values of a sequence live in pages of a shared pool: slot ``j`` of sequence ``b`` is row
``j % page_size`` of page ``block_table[b, j // page_size]``.  ``KVPages`` holds the pools; the operators take
them with a ``block_table`` (B, max_pages) int32 and ``lengths`` (B,) int64 on the device and launch on torch's
current stream, never synchronising:

    pages = KVPages.allocate(num_pages, kv_heads, page_size, head_dim, torch.bfloat16, "cuda", tracked=True)
    lengths = paged_kv_append(pages, k, v, block_table, lengths)            # a token a sequence, or CSR prompts
    out = paged_attention(q, pages, block_table, lengths, accumulate=True)  # (B, heads, head_dim)
    plan = kv_evict_plan(pages, block_table, lengths, budget=4096, recent=512)
    kv_evict_apply(pages, block_table, plan)                                # then plan.lengths slots are in use

``cortex.cache.PagedKVCache`` keeps pages, tables and lengths for named sessions.  No reference counterpart:
its StreamingKVCache (cortex/cache/streaming.py:79-236) pages embedding rows and attends to none of them.
Inference only: inputs that require a gradient or carry a forward-mode tangent are refused.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from cortex import _native as nat

_PER_ROW = ("k_scale", "v_scale", "weight", "position")


class KVPages:
    """Pools of pages: ``k`` and ``v`` (num_pages, kv_heads, page_size, head_dim) in bf16, fp32 or int8 (any
    strides, head_dim contiguous, rows 16-byte aligned, none that share memory where append or eviction write them;
    ``page_size`` a power of two from 8, ``head_dim`` a multiple of 16 up to 128) and contiguous (num_pages, kv_heads,
    page_size) arrays: ``k_scale``, ``v_scale`` fp32 (int8 pages: a row is ``code * scale``), ``weight`` fp32 (softmax weight
    received so far) and ``position`` int32 (where the token stood in its sequence), the last two optional.  The tensors of
    an object do not change."""

    __slots__ = ("k", "v", *_PER_ROW, "num_pages", "kv_heads", "page_size", "head_dim", "device", "index", "query_dtype",
                 "_struct", "ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                 position: torch.Tensor | None = None) -> None:
        self.device = nat.require_gpu(k, v, k_scale, v_scale, weight, position, what="KVPages")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError(f"k and v must be (num_pages, kv_heads, page_size, head_dim) of one dtype, got "
                             f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        if k.dtype not in (torch.bfloat16, torch.float32, torch.int8):
            raise ValueError(f"pages of dtype {k.dtype} are not supported (bfloat16, float32 or int8)")
        if (k.dtype == torch.int8) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("int8 pages need k_scale and v_scale, float pages take none")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("k and v need a contiguous last (head) dim")
        if any(t is not None and t.requires_grad for t in (k, v, k_scale, v_scale, weight)):
            raise ValueError("pages hold values without gradients")
        if forward_ad._current_level >= 0:
            _no_tangent("KVPages", k, v, k_scale, v_scale, weight)
        self.index = k.get_device()
        # of queries and outputs: the pages' own, bfloat16 for int8 pages
        self.query_dtype = torch.bfloat16 if k.dtype == torch.int8 else k.dtype
        self.k, self.v, self.k_scale, self.v_scale, self.weight, self.position = k, v, k_scale, v_scale, weight, position
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        for name in _PER_ROW:
            t = getattr(self, name)
            want = torch.int32 if name == "position" else torch.float32
            if t is not None and (t.shape != k.shape[:3] or t.dtype != want or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous {want} tensor of shape {tuple(k.shape[:3])}")
        if self.page_size < 8 or self.page_size > 65536 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size must be a power of two from 8 to 65536, got {self.page_size}")
        if self.head_dim % 16 or not 16 <= self.head_dim <= 128:
            raise ValueError(f"head_dim must be a multiple of 16 up to 128, got {self.head_dim}")
        es = k.element_size()
        if any(x % 16 for t in (k, v) for x in (t.data_ptr(), *(s * es for s in t.stride()[:3]))):
            raise ValueError("page rows must be 16-byte aligned")
        if any(t is not None and t.data_ptr() % 16 for t in (k_scale, v_scale, weight, position)):
            raise ValueError("k_scale, v_scale, weight and position must be 16-byte aligned")
        self._struct = nat.KvPagesStruct(*k.shape, nat.code(k.dtype), *k.stride()[:3], *v.stride()[:3], nat.ptr(k),
                                         nat.ptr(v), *(nat.ptr(getattr(self, n)) for n in _PER_ROW))
        self.ref = ctypes.addressof(self._struct)

    @classmethod
    def allocate(cls, num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda", *, tracked: bool = False) -> KVPages:
        """Zeroed pools; ``tracked`` adds ``weight`` and ``position`` (eviction needs them)."""
        shape = (num_pages, kv_heads, page_size)
        k, v = (torch.zeros(*shape, head_dim, dtype=dtype, device=device) for _ in range(2))
        more = {}
        if dtype == torch.int8:
            more = {n: torch.zeros(shape, device=device) for n in ("k_scale", "v_scale")}
        if tracked:
            more["weight"] = torch.zeros(shape, device=device)
            more["position"] = torch.zeros(shape, dtype=torch.int32, device=device)
        return cls(k, v, **more)


class EvictPlan(NamedTuple):
    """What ``kv_evict_plan`` found: slot ``src[b, h, i]`` moves to ``dst[b, h, i]`` for ``i < counts[b, h]`` (-1
    behind), and ``lengths`` slots are in use afterwards."""

    dst: torch.Tensor
    src: torch.Tensor
    counts: torch.Tensor
    lengths: torch.Tensor


_get_device = torch._C._cuda_getDevice  # what torch.cuda.current_device() asks, without its initialisation check


def _i64(t: torch.Tensor, n: int, name: str, what: str) -> None:
    if t.dtype is not torch.int64 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous int64 tensor of {n} values, got {tuple(t.shape)} {t.dtype}")


def _common(what: str, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor,
            err_flag) -> tuple[int, int, int]:
    """Checks what every operator takes; the block table's rows, row stride and columns."""
    idx = pages.index
    if (block_table.get_device() != idx or lengths.get_device() != idx
            or (err_flag is not None and err_flag.get_device() != idx)):
        _elsewhere(what, pages, block_table, lengths, err_flag)
    shape = block_table.shape
    if len(shape) != 2 or block_table.dtype is not torch.int32:
        raise ValueError(f"{what}: block_table must be a (B, max_pages) int32 tensor")
    B, width = shape
    if block_table.is_contiguous():
        ld = width
    else:
        ld, unit = block_table.stride()
        if width > 1 and unit != 1:
            raise ValueError(f"{what}: the rows of block_table must be contiguous")
        if B < 2:
            ld = width
    if lengths.dtype is not torch.int64 or lengths.shape != (B,) or not lengths.is_contiguous():
        _i64(lengths, B, "lengths", what)
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        raise ValueError(f"{what}: err_flag must be one int32")
    return B, ld, width


def _elsewhere(what: str, pages: KVPages, *tensors) -> None:
    dev = nat.require_gpu(*tensors, what=what)
    raise RuntimeError(f"{what}: tensors on different devices ({dev} vs {pages.device})")


def _no_grad(what: str) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")


def _no_tangent(what: str, *tensors: torch.Tensor | None) -> None:
    """Within a level of forward-mode differentiation (the callers ask for that, which is cheaper)."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it on tensors without tangents")


def _rows(t: torch.Tensor, pages: KVPages, es: int) -> tuple[torch.Tensor, int, int]:
    """(n, heads, head_dim) rows that vector loads take, as given or copied, and their strides."""
    if t.is_contiguous():
        if t.data_ptr() & 15:
            t = t.clone()
        return t, t.shape[1] * pages.head_dim, pages.head_dim
    s0, s1, s2 = t.stride()
    if s2 != 1 or (t.data_ptr() | s0 * es | s1 * es) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, _ = t.stride()
    return t, s0, s1


def _own_overlap(t: torch.Tensor) -> bool:
    """Whether rows of a (n, heads, head_dim) tensor may share memory."""
    n, m, d = t.shape
    s, r = t.stride(0), t.stride(1)
    if r > s and n > 1:  # (heads outside)
        n, m, s, r = m, n, r, s
    return (m > 1 and r < d) or (n > 1 and s < (m - 1) * r + d)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (n, heads, head_dim) tensors may share memory (parts of one buffer that lie in each other's gaps, such as
    the columns of a joint projection, do not)."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    es = a.element_size()

    def span(t):  # bytes from the first to past the last value of the tensor, and of a row of it
        row = ((t.shape[1] - 1) * t.stride(1) + t.shape[2]) * es
        return (t.shape[0] - 1) * t.stride(0) * es + row, row

    (na, ra), (nb, rb) = span(a), span(b)
    if a0 + na <= b0 or b0 + nb <= a0:
        return False
    pitch = a.stride(0) * es
    if a.stride(0) != b.stride(0) or not 0 < max(ra, rb) <= pitch:
        return True
    d = (b0 - a0) % pitch
    return d < ra or d + rb > pitch


def paged_kv_append(pages: KVPages, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, offsets: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, new_lengths: torch.Tensor | None = None,
                    err_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Writes the rows of new tokens behind the ``lengths`` of their sequences and returns the new lengths (B,).

    ``k``, ``v`` (T, kv_heads, head_dim) bf16 or fp32: token b of sequence b, or with ``offsets`` (B + 1,) int64 the
    tokens ``[offsets[b], offsets[b + 1])`` of sequence b (no two tokens may share a slot).   Int8 pages take each row at
    scale ``max(max|x|, 1e-8) / 127``, rounded half to even; a row with an infinity or a NaN becomes NaN.  Tracked
    pages get weight 0 and the token's position: ``positions`` (T,) int64 (kept in 32 bits), by default its slot number.
    ``new_lengths`` may be ``lengths`` itself and overlaps no other input.  A token without a slot or a page, or of a sequence
    whose length is negative or past the table, is dropped and sets bit 2 of ``err_flag`` (int32, never cleared here); a
    negative length stays negative."""
    idx = pages.index
    if idx != _get_device():
        with torch.cuda.device(idx):
            return paged_kv_append(pages, k, v, block_table, lengths, offsets=offsets, positions=positions,
                                   new_lengths=new_lengths, err_flag=err_flag)
    B, ld, width = _common("paged_kv_append", pages, block_table, lengths, err_flag)
    if (k.get_device() != idx or v.get_device() != idx or (offsets is not None and offsets.get_device() != idx)
            or (positions is not None and positions.get_device() != idx)
            or (new_lengths is not None and new_lengths.get_device() != idx)):
        _elsewhere("paged_kv_append", pages, k, v, offsets, positions, new_lengths)
    if k.requires_grad or v.requires_grad:
        _no_grad("paged_kv_append")
    if forward_ad._current_level >= 0:
        _no_tangent("paged_kv_append", k, v)
    shape, dtype = k.shape, k.dtype
    if shape != v.shape or len(shape) != 3 or shape[1:] != (pages.kv_heads, pages.head_dim) or dtype is not v.dtype:
        raise ValueError(f"k and v must be (T, {pages.kv_heads}, {pages.head_dim}) of one dtype, got {tuple(k.shape)} "
                         f"{k.dtype} and {tuple(v.shape)} {v.dtype}")
    if dtype is torch.bfloat16:
        code, es = nat.BF16, 2
    elif dtype is torch.float32:
        code, es = nat.F32, 4
    else:
        raise ValueError(f"rows of dtype {dtype} are not supported (bfloat16 or float32)")
    T = shape[0]
    if offsets is not None:
        _i64(offsets, B + 1, "offsets", "paged_kv_append")
    elif T != B:
        raise ValueError(f"{T} tokens for {B} sequences: without offsets there is one token a sequence")
    if positions is not None:
        _i64(positions, T, "positions", "paged_kv_append")
    if new_lengths is None:
        new_lengths = torch.empty_like(lengths)
    else:
        _i64(new_lengths, B, "new_lengths", "paged_kv_append")
    k, kt, kh = _rows(k, pages, es)
    v, vt, vh = _rows(v, pages, es)
    nat.call("cortex_kv_append", pages.ref, B, T, code, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
             block_table.data_ptr(), ld, width, nat.ptr(offsets), lengths.data_ptr(), nat.ptr(positions),
             new_lengths.data_ptr(), nat.ptr(err_flag), nat.stream_of(pages.device))
    return new_lengths


def paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: float | None = None, accumulate: bool = False, max_length: int | None = None,
                    out: torch.Tensor | None = None, err_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax_{j < lengths[b]}(scale * q . k_j) v_j`` of one query a sequence: ``q`` (B, heads, head_dim) in
    ``pages.query_dtype`` with ``heads`` a multiple of the key heads (query head h reads key head
    ``h // (heads // kv_heads)``), ``scale`` ``head_dim ** -0.5`` by default.  A sequence of length 0 gives 0.

    ``accumulate`` adds to ``pages.weight`` the softmax weight that each key received, summed over the query heads
    of its key head; no two sequences of the call may then share a page.  ``out`` may not overlap ``q`` or itself.
    ``max_length``: a bound of the lengths known on the host (default: the table's width), which sizes the launch and
    the workspace; longer sequences are cut to it and set bit 2 of ``err_flag``, as lengths outside the table and page
    ids outside the pool do (such pages hold no keys).  With ``accumulate`` the workspace holds ``B * heads * max_length`` fp32
    scores beside the parts, whatever the lengths are: give the bound where tables are wide.  Up to 4096 sequences and 1024
    query heads a key head.  Values are summed in fp32 before they are divided: ``lengths[b] * max|v|`` is to stay below 2^120."""
    if pages.index != _get_device():
        with torch.cuda.device(pages.index):
            return paged_attention(q, pages, block_table, lengths, scale=scale, accumulate=accumulate,
                                   max_length=max_length, out=out, err_flag=err_flag)
    B, ld, width = _common("paged_attention", pages, block_table, lengths, err_flag)
    if q.get_device() != pages.index or (out is not None and out.get_device() != pages.index):
        _elsewhere("paged_attention", pages, q, out)
    if q.requires_grad or (out is not None and out.requires_grad):
        _no_grad("paged_attention")
    if forward_ad._current_level >= 0:
        _no_tangent("paged_attention", q, out)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or shape[0] != B or shape[2] != pages.head_dim or dtype is not pages.query_dtype:
        raise ValueError(f"q must be ({B}, heads, {pages.head_dim}) in {pages.query_dtype}, got {tuple(shape)} {dtype}")
    heads = shape[1]
    if heads < 1 or heads % pages.kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {pages.kv_heads} key heads")
    if accumulate and pages.weight is None:
        raise ValueError("accumulate needs pages with weight")
    if max_length is None:
        max_length = width * pages.page_size
    elif max_length < 0:
        raise ValueError(f"max_length must not be negative, got {max_length}")
    else:
        max_length = min(max_length, width * pages.page_size)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype is not dtype or out.stride(2) != 1:
        raise ValueError(f"out must be a {tuple(shape)} {dtype} tensor with a contiguous last dim")
    elif _own_overlap(out):
        raise ValueError("out may not overlap itself (an expanded tensor)")
    elif _overlap(out, q):
        raise ValueError("out may not overlap q")
    q, qb, qh = _rows(q, pages, 4 if dtype is torch.float32 else 2)
    ws_bytes = nat.load().cortex_paged_attention_workspace_bytes(pages.ref, B, heads, max_length, accumulate)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=pages.device) if ws_bytes else None
    ob, oh, _ = out.stride()
    nat.call("cortex_paged_attention", pages.ref, B, heads, q.data_ptr(), qb, qh, block_table.data_ptr(), ld, width,
             lengths.data_ptr(), max_length, pages.head_dim ** -0.5 if scale is None else scale, accumulate,
             out.data_ptr(), ob, oh, nat.ptr(ws), ws_bytes, nat.ptr(err_flag), nat.stream_of(pages.device))
    return out


def kv_evict_plan(pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, budget: int, recent: int, *,
                  max_length: int | None = None, err_flag: torch.Tensor | None = None) -> EvictPlan:
    """Which slots each key head keeps where a sequence holds more than ``budget``: those of the last ``recent``
    positions first (``recent <= budget``), then the ones with the largest ``pages.weight`` (a NaN before every number,
    equal weights by the lower slot).  Kept slots at or past the budget are to fill the slots below it that are given up
    (``EvictPlan``); shorter sequences stay as they are.  Slots that no query has attended to with ``accumulate`` have weight
    0, all of a new prompt among them: of those the newest stay, then the first ones.  Reads ``pages.weight`` and
    ``pages.position`` and writes neither; a negative length stays negative in ``EvictPlan.lengths``.  ``max_length`` and ``err_flag`` as for ``paged_attention``."""
    if pages.index != _get_device():
        with torch.cuda.device(pages.index):
            return kv_evict_plan(pages, block_table, lengths, budget, recent, max_length=max_length, err_flag=err_flag)
    B, ld, width = _common("kv_evict_plan", pages, block_table, lengths, err_flag)
    if pages.weight is None or pages.position is None:
        raise ValueError("eviction needs pages with weight and position (tracked=True)")
    if budget < 0 or recent < 0 or (max_length is not None and max_length < 0):
        raise ValueError(f"budget, recent and max_length must not be negative, got {budget}, {recent}, {max_length}")
    if recent > budget:
        raise ValueError(f"recent ({recent}) exceeds the budget ({budget})")
    budget, recent = min(budget, 1 << 40), min(recent, 1 << 40)  # (as far as a C integer goes)
    room = width * pages.page_size
    most = room if max_length is None else min(max_length, room)
    cap = max(0, min(budget, most - budget))
    dst = block_table.new_empty((B, pages.kv_heads, cap))
    src = torch.empty_like(dst)
    counts = block_table.new_empty((B, pages.kv_heads))
    after = torch.empty_like(lengths)
    nat.call("cortex_kv_evict_plan", pages.ref, B, block_table.data_ptr(), ld, width, lengths.data_ptr(), most, budget,
             recent, dst.data_ptr(), src.data_ptr(), counts.data_ptr(), after.data_ptr(), nat.ptr(err_flag),
             nat.stream_of(pages.device))
    return EvictPlan(dst, src, counts, after)


def kv_evict_apply(pages: KVPages, block_table: torch.Tensor, plan: EvictPlan, *,
                   err_flag: torch.Tensor | None = None) -> None:
    """Moves the rows of a plan in place: keys, values and, where the pages have them, scales, weight and position.
    Slots at or past the budget keep what they held.  Sequences of the call may not share pages."""
    if pages.index != _get_device():
        with torch.cuda.device(pages.index):
            return kv_evict_apply(pages, block_table, plan, err_flag=err_flag)
    dst, src, counts, after = plan
    B, ld, width = _common("kv_evict_apply", pages, block_table, after, err_flag)
    if dst.get_device() != pages.index or src.get_device() != pages.index or counts.get_device() != pages.index:
        _elsewhere("kv_evict_apply", pages, dst, src, counts)
    shape = dst.shape
    if (len(shape) != 3 or shape[:2] != (B, pages.kv_heads) or src.shape != shape or counts.shape != shape[:2]
            or not dst.dtype is src.dtype is counts.dtype is torch.int32
            or not (dst.is_contiguous() and src.is_contiguous() and counts.is_contiguous())):
        raise ValueError(f"the plan must hold contiguous int32 moves of ({B}, {pages.kv_heads}) heads")
    nat.call("cortex_kv_evict_apply", pages.ref, B, block_table.data_ptr(), ld, width, dst.data_ptr(), src.data_ptr(),
             shape[2], counts.data_ptr(), nat.ptr(err_flag), nat.stream_of(pages.device))


__all__ = ["EvictPlan", "KVPages", "kv_evict_apply", "kv_evict_plan", "paged_attention", "paged_kv_append"]
