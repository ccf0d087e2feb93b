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
Inference only: inputs that require a gradient are refused.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from cortex import _native as nat

_PER_ROW = ("k_scale", "v_scale", "weight", "position")


class KVPages:
    """Pools of pages: ``k`` and ``v`` (num_pages, kv_heads, page_size, head_dim) in bf16, fp32 or int8 (any
    strides, head_dim contiguous, rows 16-byte aligned; ``page_size`` a power of two from 8, ``head_dim`` a multiple of
    16 up to 128) and contiguous (num_pages, kv_heads, page_size) arrays: ``k_scale``, ``v_scale`` fp32 (int8 pages:
    a row is ``code * scale``), ``weight`` fp32 (softmax weight received so far) and ``position`` int32 (where the
    token stood in its sequence), the last two optional.  The tensors of an object do not change."""

    __slots__ = ("k", "v", *_PER_ROW, "num_pages", "kv_heads", "page_size", "head_dim", "device", "_struct", "ref")

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
        if any(t is not None and t.requires_grad for t in (k, v)):
            raise ValueError("pages hold values without gradients")
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

    @property
    def query_dtype(self) -> torch.dtype:
        """The dtype of queries and outputs: the pages' own, bfloat16 for int8 pages."""
        return torch.bfloat16 if self.k.dtype == torch.int8 else self.k.dtype


class EvictPlan(NamedTuple):
    """What ``kv_evict_plan`` found: slot ``src[b, h, i]`` moves to ``dst[b, h, i]`` for ``i < counts[b, h]`` (-1
    behind), and ``lengths`` slots are in use afterwards."""

    dst: torch.Tensor
    src: torch.Tensor
    counts: torch.Tensor
    lengths: torch.Tensor


def _i64(t: torch.Tensor, n: int, name: str, what: str) -> None:
    if t.dtype != torch.int64 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous int64 tensor of {n} values, got {tuple(t.shape)} {t.dtype}")


def _common(what: str, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, err_flag, *more) -> int:
    """Checks what every operator takes; the number of sequences."""
    dev = nat.require_gpu(block_table, lengths, err_flag, *more, what=what)
    if dev != pages.device:
        raise RuntimeError(f"{what}: tensors on different devices ({dev} vs {pages.device})")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"{what}: block_table must be a (B, max_pages) int32 tensor with contiguous rows")
    B = block_table.shape[0]
    _i64(lengths, B, "lengths", what)
    if err_flag is not None and (err_flag.dtype != torch.int32 or err_flag.numel() != 1):
        raise ValueError(f"{what}: err_flag must be one int32")
    return B


def _launch(name: str, device: torch.device, *args) -> None:
    """``nat.call`` on the current stream of ``device``, whichever device is current."""
    if device.index == torch.cuda.current_device():
        nat.call(name, *args, nat.stream_of(device))
    else:
        with torch.cuda.device(device):
            nat.call(name, *args, nat.stream_of(device))


def _ld(block_table: torch.Tensor) -> int:
    return block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]


def _no_grad(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(n, heads, head_dim) rows that vector loads take: as given, or a contiguous copy."""
    es = t.element_size()
    s0, s1, s2 = t.stride()
    if s2 != 1 or t.data_ptr() % 16 or (s0 * es) % 16 or (s1 * es) % 16:
        return t.clone(memory_format=torch.contiguous_format)  # (contiguous() keeps rows that only start off)
    return t


def paged_kv_append(pages: KVPages, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, offsets: torch.Tensor | None = None,
                    positions: torch.Tensor | None = None, new_lengths: torch.Tensor | None = None,
                    err_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Writes the rows of new tokens behind the ``lengths`` of their sequences and returns the new lengths (B,).

    ``k``, ``v`` (T, kv_heads, head_dim) bf16 or fp32: token b of sequence b, or with ``offsets`` (B + 1,) int64 the
    tokens ``[offsets[b], offsets[b + 1])`` of sequence b (no two tokens may share a slot).  Int8 pages take each row at scale
    ``max(max|x|, 1e-8) / 127``, rounded half to even.  Tracked pages get weight 0 and the token's position:
    ``positions`` (T,) int64, by default its slot number.  ``new_lengths`` may be ``lengths`` itself.  A token without
    a slot or a page is dropped and sets bit 2 of ``err_flag`` (int32, never cleared here)."""
    B = _common("paged_kv_append", pages, block_table, lengths, err_flag, k, v, offsets, positions, new_lengths)
    _no_grad("paged_kv_append", k, v)
    T = k.shape[0]
    if k.shape != v.shape or k.dim() != 3 or k.shape[1:] != (pages.kv_heads, pages.head_dim) or k.dtype != v.dtype:
        raise ValueError(f"k and v must be (T, {pages.kv_heads}, {pages.head_dim}) of one dtype, got {tuple(k.shape)} "
                         f"{k.dtype} and {tuple(v.shape)} {v.dtype}")
    if k.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"rows of dtype {k.dtype} are not supported (bfloat16 or float32)")
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
    k, v = _rows(k), _rows(v)
    (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
    _launch("cortex_kv_append", pages.device, pages.ref, B, T, nat.code(k.dtype), k.data_ptr(), kt, kh, v.data_ptr(),
            vt, vh, block_table.data_ptr(), _ld(block_table), block_table.shape[1], nat.ptr(offsets),
            lengths.data_ptr(), nat.ptr(positions), new_lengths.data_ptr(), nat.ptr(err_flag))
    return new_lengths


def paged_attention(q: torch.Tensor, pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: float | None = None, accumulate: bool = False, max_length: int | None = None,
                    out: torch.Tensor | None = None, err_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax_{j < lengths[b]}(scale * q . k_j) v_j`` of one query a sequence: ``q`` (B, heads, head_dim) in
    ``pages.query_dtype`` with ``heads`` a multiple of the key heads (query head h reads key head
    ``h // (heads // kv_heads)``), ``scale`` ``head_dim ** -0.5`` by default.  A sequence of length 0 gives 0.

    ``accumulate`` adds to ``pages.weight`` the softmax weight that each key received, summed over the query heads
    of its key head; no two sequences of the call may then share a page.  ``max_length``: a bound of the lengths
    known on the host (default: the table's width), which sizes the launch and the workspace; longer sequences are cut
    to it and set bit 2 of ``err_flag``, as lengths outside the table and page ids outside the pool do (such pages hold no keys)."""
    B = _common("paged_attention", pages, block_table, lengths, err_flag, q, out)
    _no_grad("paged_attention", q)
    if q.dim() != 3 or q.shape[0] != B or q.shape[2] != pages.head_dim or q.dtype != pages.query_dtype:
        raise ValueError(f"q must be ({B}, heads, {pages.head_dim}) in {pages.query_dtype}, got {tuple(q.shape)} {q.dtype}")
    heads = q.shape[1]
    if heads < 1 or heads % pages.kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {pages.kv_heads} key heads")
    if accumulate and pages.weight is None:
        raise ValueError("accumulate needs pages with weight")
    if max_length is not None and max_length < 0:
        raise ValueError(f"max_length must not be negative, got {max_length}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.data_ptr() == q.data_ptr():
        raise ValueError(f"out must be a {tuple(q.shape)} {q.dtype} tensor of its own with a contiguous last dim")
    if B == 0:
        return out
    most = block_table.shape[1] * pages.page_size if max_length is None else max_length
    q = _rows(q)
    ws_bytes = nat.load().cortex_paged_attention_workspace_bytes(pages.ref, B, heads, most, int(accumulate))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=pages.device) if ws_bytes else None
    _launch("cortex_paged_attention", pages.device, pages.ref, B, heads, q.data_ptr(), q.stride(0), q.stride(1),
            block_table.data_ptr(), _ld(block_table), block_table.shape[1], lengths.data_ptr(), most,
            float(scale) if scale is not None else pages.head_dim ** -0.5, int(accumulate), out.data_ptr(),
            out.stride(0), out.stride(1), nat.ptr(ws), ws_bytes, nat.ptr(err_flag))
    return out


def kv_evict_plan(pages: KVPages, block_table: torch.Tensor, lengths: torch.Tensor, budget: int, recent: int, *,
                  max_length: int | None = None, err_flag: torch.Tensor | None = None) -> EvictPlan:
    """Which slots each key head keeps where a sequence holds more than ``budget``: those of the last ``recent``
    positions first (``recent <= budget``), then the ones with the largest ``pages.weight`` (a NaN before every number,
    equal weights by the lower slot).  Kept slots at or past the budget are to fill the slots below it that are given up (``EvictPlan``);
    shorter sequences stay as they are.  Reads ``pages.weight`` and ``pages.position`` and writes neither.
    ``max_length`` and ``err_flag`` as for ``paged_attention``."""
    B = _common("kv_evict_plan", pages, block_table, lengths, err_flag)
    if pages.weight is None or pages.position is None:
        raise ValueError("eviction needs pages with weight and position (tracked=True)")
    if budget < 0 or recent < 0 or (max_length is not None and max_length < 0):
        raise ValueError(f"budget, recent and max_length must not be negative, got {budget}, {recent}, {max_length}")
    if recent > budget:
        raise ValueError(f"recent ({recent}) exceeds the budget ({budget})")
    room = block_table.shape[1] * pages.page_size
    most = room if max_length is None else min(max_length, room)
    cap = max(0, min(budget, most - budget))
    H = pages.kv_heads
    moves = torch.empty((2, B, H, cap), dtype=torch.int32, device=pages.device)
    counts = torch.empty((B, H), dtype=torch.int32, device=pages.device)
    after = torch.empty_like(lengths)
    plan = EvictPlan(moves[0], moves[1], counts, after)
    if B == 0:
        return plan
    _launch("cortex_kv_evict_plan", pages.device, pages.ref, B, block_table.data_ptr(), _ld(block_table),
            block_table.shape[1], lengths.data_ptr(), most, int(budget), int(recent), plan.dst.data_ptr(),
            plan.src.data_ptr(), counts.data_ptr(), after.data_ptr(), nat.ptr(err_flag))
    return plan


def kv_evict_apply(pages: KVPages, block_table: torch.Tensor, plan: EvictPlan, *,
                   err_flag: torch.Tensor | None = None) -> None:
    """Moves the rows of a plan in place: keys, values and, where the pages have them, scales, weight and position.
    Slots at or past the budget keep what they held.  Sequences of the call may not share pages."""
    B = _common("kv_evict_apply", pages, block_table, plan.lengths, err_flag, plan.dst, plan.src, plan.counts)
    shape = plan.dst.shape
    if (len(shape) != 3 or shape[:2] != (B, pages.kv_heads) or plan.src.shape != shape or plan.counts.shape != shape[:2]
            or any(t.dtype != torch.int32 or not t.is_contiguous() for t in plan[:3])):
        raise ValueError(f"the plan must hold contiguous int32 moves of ({B}, {pages.kv_heads}) heads")
    if B == 0 or shape[2] == 0:
        return
    _launch("cortex_kv_evict_apply", pages.device, pages.ref, B, block_table.data_ptr(), _ld(block_table),
            block_table.shape[1], plan.dst.data_ptr(), plan.src.data_ptr(), shape[2], plan.counts.data_ptr(),
            nat.ptr(err_flag))


__all__ = ["EvictPlan", "KVPages", "kv_evict_apply", "kv_evict_plan", "paged_attention", "paged_kv_append"]
