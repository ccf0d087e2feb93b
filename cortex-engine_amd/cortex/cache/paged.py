"""Paged K/V cache of named sessions, over the operators of ``cortex.kernels.paged_kv``.

``PagedKVCache`` keeps what a server keeps beside the pools: which pages a session owns, how many slots of them are in
use, and where in its sequence it stands.  All of that is on the host, so nothing is read back from the device; a step
uploads its block table, lengths and positions as one pinned copy:

    cache = PagedKVCache(num_pages=4096, kv_heads=8, head_dim=128, layers=12, tracked=True)
    batch = cache.extend(["a", "b"], counts=[900, 12])      # slots for prompts
    cache.append(batch, k, v, layer=0)                      # (912, 8, 128) rows, session after session
    batch = cache.extend(["a", "b"])                        # slots for a token each
    cache.append(batch, k, v, layer=0)
    out = cache.attend(batch, q, layer=0)                   # (2, heads, 128)
    cache.evict(["a", "b"], budget=512, recent=64)          # keep what drew attention

As in the reference's paged cache (cortex/cache/streaming.py:203-233) pages come from a free list and, when that is
empty, from what was used least recently: here whole sessions, since a sequence with a gap is of no use.

Not thread-safe: like the other caches it is meant for the single inference executor thread.  The operators run on
torch's current stream; a call on another stream than the one before (the first: than the one that the cache was made
on) first waits, on the device, for that one.  A graph cannot follow its steps, each of which has a table of its own: in a
capture ``extend`` is refused, and so is a call on another stream than the one before (``cortex.kernels.paged_kv`` on tables
that the program keeps can be captured).
"""

from __future__ import annotations

from collections import OrderedDict
from typing import NamedTuple

import numpy as np
import torch

from cortex.kernels.paged_kv import KVPages, kv_evict_apply, kv_evict_plan, paged_attention, paged_kv_append


class KVBatch(NamedTuple):
    """Sessions of a step as the operators take them (device tensors): ``block_table`` (B, pages) int32, the slots in use
    before the step's tokens (``before``) and with them (``lengths``), ``offsets`` (B + 1,) of the tokens (None: one a
    session), their ``positions``, and on the host ``tokens`` and ``max_length``.  It holds until one of its sessions is
    cut or dropped; ``append`` and ``attend`` refuse it from then on.  ``filled``: the layers that have its tokens' rows;
    ``needs``: the same of every batch whose rows some layer lacked when this one was made, its own among them."""

    sessions: tuple[str, ...]
    block_table: torch.Tensor
    before: torch.Tensor
    lengths: torch.Tensor
    offsets: torch.Tensor | None
    positions: torch.Tensor
    tokens: int
    max_length: int
    held: tuple  # the sessions' records and the versions that the batch was made of
    versions: tuple[int, ...]
    epoch: int
    stream: torch.cuda.Stream  # that its tensors were made on
    filled: set[int]
    needs: tuple[set[int], ...]


class _Session:
    __slots__ = ("pages", "used", "length", "seen", "version", "pending")

    def __init__(self) -> None:
        self.pages = np.empty(8, dtype=np.int32)
        self.used = 0  # pages owned: pages[:used]
        self.length = 0  # slots in use
        self.seen = 0  # tokens ever appended: the position of the next
        self.version = 0  # counts what makes batches of this session out of date
        self.pending: list[set[int]] = []  # ``filled`` of the batches whose rows some layer may lack


class PagedKVCache:
    """Pages of keys and values for named sessions, ``layers`` pools that share one block table."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, layers: int = 1, tracked: bool = False,
                 device: str | torch.device = "cuda") -> None:
        if num_pages < 1 or layers < 1:
            raise ValueError("num_pages and layers must be >= 1")
        self.num_pages, self.page_size, self.tracked = num_pages, page_size, tracked
        self.layers = [KVPages.allocate(num_pages, kv_heads, page_size, head_dim, dtype, device, tracked=tracked)
                       for _ in range(layers)]
        self.device = self.layers[0].device
        self._free = list(range(num_pages - 1, -1, -1))
        self._sessions: OrderedDict[str, _Session] = OrderedDict()  # least recently used first
        self._stage = torch.empty(1 << 12, dtype=torch.int64).pin_memory()
        self._staged = torch.cuda.Event()
        self._stream = torch.cuda.current_stream(self.device)  # of the last call: here, of the pools' zero fills
        self._epoch = 0  # counts the changes of any session's version

    @property
    def pages_used(self) -> int:
        return self.num_pages - len(self._free)

    @property
    def sessions(self) -> list[str]:
        """Session names, least recently used first."""
        return list(self._sessions)

    def length(self, session_id: str) -> int:
        """Slots of a session that are in use (0: unknown session)."""
        s = self._sessions.get(session_id)
        return s.length if s is not None else 0

    def evict_session(self, session_id: str) -> int:
        """Free every page of ``session_id``; returns how many were freed."""
        s = self._sessions.pop(session_id, None)
        if s is None:
            return 0
        return self._release(s, 0)

    def extend(self, session_ids, counts=None) -> KVBatch:
        """Slots for ``counts[i]`` new tokens of session i (one each by default), new sessions among them, and the batch
        that ``append`` and ``attend`` take.  Sessions that are not in the call give way, least recently used first, when
        the free pages do not do; MemoryError, and nothing changed, when that is not enough either."""
        names = self._names(session_ids)
        if counts is None:
            new = np.ones(len(names), dtype=np.int64)
        else:
            new = np.asarray(counts, dtype=np.int64).reshape(-1)
            if new.shape[0] != len(names) or (new < 0).any():
                raise ValueError(f"counts must be {len(names)} numbers >= 0")
        held = [self._sessions.get(n) or _Session() for n in names]
        need = [max(0, -(-(s.length + int(c)) // self.page_size) - s.used) for s, c in zip(held, new)]
        total = sum(need)
        missing, victims = total - len(self._free), []
        if missing > 0:
            keep = set(names)
            for name, s in self._sessions.items():
                if missing <= 0:
                    break
                if name not in keep and s.used:
                    victims.append(name)
                    missing -= s.used
            if missing > 0:
                raise MemoryError(f"{missing} pages short of {total} (of {self.num_pages} in all)")
        # the end of the free list as it is once the victims are gone, the last one first
        taken = [p for name in victims for p in self._sessions[name].pages[:self._sessions[name].used].tolist()][::-1]
        taken = taken[:total] + self._free[len(self._free) - max(0, total - len(taken)):][::-1]
        B, width = len(names), max((s.used + n for s, n in zip(held, need)), default=0)
        table = np.full((B, width), -1, dtype=np.int32)
        before = np.empty(B, dtype=np.int64)
        positions = np.empty(int(new.sum()), dtype=np.int64)
        at = row = 0
        for i, (s, n, c) in enumerate(zip(held, need, new.tolist())):
            table[i, :s.used] = s.pages[:s.used]
            if n:
                table[i, s.used:s.used + n] = taken[at:at + n]
                at += n
            before[i] = s.length
            if c == 1:
                positions[row] = s.seen
            else:
                positions[row:row + c] = np.arange(s.seen, s.seen + c)
            row += c
        ragged = not (new == 1).all()
        offsets = np.concatenate([[0], np.cumsum(new)]) if ragged else np.empty(0, dtype=np.int64)
        flat = np.zeros(-(-table.size // 2) * 2, dtype=np.int32)
        flat[:table.size] = table.reshape(-1)
        parts = self._upload([before, before + new, positions, offsets.astype(np.int64, copy=False), flat.view(np.int64)])

        # nothing that may fail comes after this
        for name in victims:
            self.evict_session(name)
        del self._free[len(self._free) - total:]
        filled: set[int] = set()
        for name, s, n, c, pages in zip(names, held, need, new.tolist(), table):
            self._sessions[name] = s
            self._sessions.move_to_end(name)
            if n:
                if s.used + n > s.pages.shape[0]:
                    s.pages = np.concatenate([s.pages[:s.used], np.empty(s.used + 2 * n, dtype=np.int32)])
                s.pages[s.used:s.used + n] = pages[s.used:s.used + n]
                s.used += n
            s.length += c
            s.seen += c
            if s.pending:
                s.pending = [f for f in s.pending if len(f) < len(self.layers)]
            if c:
                s.pending.append(filled)
        return KVBatch(names, parts[4].view(torch.int32)[:table.size].view(B, width), parts[0], parts[1],
                       parts[3] if ragged else None, parts[2], positions.shape[0],
                       int((before + new).max()) if B else 0, tuple(held), tuple(s.version for s in held), self._epoch,
                       self._stream, filled, tuple({id(f): f for s in held for f in s.pending}.values()))

    def batch(self, session_ids) -> KVBatch:
        """The sessions as they stand, without new tokens (KeyError: an unknown one)."""
        names = self._names(session_ids)
        for n in names:
            if n not in self._sessions:
                raise KeyError(f"unknown session {n!r}")
        return self.extend(names, [0] * len(names))

    def append(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
        """The rows (tokens, kv_heads, head_dim) of a batch's new tokens into ``layer``'s pages, session after session."""
        if k.shape[0] != batch.tokens:
            raise ValueError(f"{k.shape[0]} rows for {batch.tokens} new tokens")
        self._enter(batch)
        paged_kv_append(self.layers[layer], k, v, batch.block_table, batch.before, offsets=batch.offsets,
                        positions=batch.positions)
        batch.filled.add(layer % len(self.layers))

    def attend(self, batch: KVBatch, q: torch.Tensor, layer: int = 0, *, scale: float | None = None,
               accumulate: bool | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """``paged_attention`` of one query (B, heads, head_dim) a session over its slots, the batch's new tokens among
        them: ``layer`` must have the rows of all of them by then (``append``), also of batches before this one (where
        one of those is given up, its sessions have to be dropped).  ``accumulate``: by default where the pages are
        tracked."""
        if any(layer % len(self.layers) not in filled for filled in batch.needs):
            raise RuntimeError(f"some slots of the batch's sessions have no rows in layer {layer}: append them first")
        self._enter(batch)
        return paged_attention(q, self.layers[layer], batch.block_table, batch.lengths, scale=scale, out=out,
                               accumulate=self.tracked if accumulate is None else accumulate, max_length=batch.max_length)

    def evict(self, session_ids, budget: int, recent: int) -> int:
        """Cuts sessions of more than ``budget`` slots down to it in every layer, each key head keeping its ``recent``
        newest slots and then those with the most weight (``kv_evict_plan``); returns the pages freed.  Every layer
        must have the rows of the sessions' tokens.  Batches made before no longer hold for these sessions."""
        if not self.tracked:
            raise ValueError("eviction by weight needs tracked=True")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"budget must be >= 1 and recent between 0 and it, got {budget} and {recent}")
        names = self._names(session_ids)
        for n in names:
            if n not in self._sessions:
                raise KeyError(f"unknown session {n!r}")
        names = [n for n in names if self._sessions[n].length > budget]
        if not names:
            return 0
        for n in names:
            if any(len(f) < len(self.layers) for f in self._sessions[n].pending):
                raise RuntimeError(f"session {n!r} has slots without rows in some layer: append them first")
        b = self.batch(names)
        # all plans, which need memory, before the first row moves: a session is cut in every layer or in none
        plans = [kv_evict_plan(pages, b.block_table, b.lengths, budget, recent, max_length=b.max_length)
                 for pages in self.layers]
        for pages, plan in zip(self.layers, plans):
            kv_evict_apply(pages, b.block_table, plan)
        freed = 0
        for n in names:
            s = self._sessions[n]
            s.length = budget
            freed += self._release(s, -(-budget // self.page_size))
        return freed

    # ---------------------------------------------------------------------------

    def _names(self, session_ids) -> tuple[str, ...]:
        names = tuple(session_ids)
        if isinstance(session_ids, str) or len(set(names)) != len(names):
            raise ValueError("session_ids must be distinct names")
        return names

    def _release(self, s: _Session, keep: int) -> int:
        """Pages of a session past the first ``keep`` go back to the free list (the last one first out)."""
        s.version += 1
        self._epoch += 1
        freed = s.used - keep
        self._free.extend(s.pages[keep:s.used].tolist())
        s.used = keep
        return freed

    def _enter(self, batch: KVBatch | None = None) -> None:
        """Before an operator: the batch still holds, and what another stream was given here comes first."""
        if batch is not None and batch.epoch != self._epoch:
            for name, s, version in zip(batch.sessions, batch.held, batch.versions):
                if s.version != version:
                    raise RuntimeError(f"the batch is out of date: session {name!r} was cut or dropped since")
        stream = torch.cuda.current_stream(self.device)
        if self._stream != stream:
            self._not_captured()
            done = torch.cuda.Event()
            done.record(self._stream)
            stream.wait_event(done)
            for p in self.layers:
                for t in (p.k, p.v, p.k_scale, p.v_scale, p.weight, p.position):
                    if t is not None:
                        t.record_stream(stream)
        if batch is not None and batch.stream != stream:
            batch.lengths.record_stream(stream)  # (all of a batch is one allocation)
        self._stream = stream

    def _not_captured(self) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the steps of a PagedKVCache are not captured: a graph takes the operators of "
                               "cortex.kernels.paged_kv on tables and lengths that its program keeps")

    def _upload(self, cols: list[np.ndarray]) -> list[torch.Tensor]:
        """int64 arrays on the device, parts of one allocation and one pinned copy."""
        need = sum(c.shape[0] for c in cols)
        self._not_captured()
        self._enter()
        self._staged.synchronize()  # the copy before has left the pinned buffer
        if self._stage.numel() < need:
            self._stage = torch.empty(max(need, 2 * self._stage.numel()), dtype=torch.int64).pin_memory()
        np.concatenate(cols, out=self._stage.numpy()[:need])
        dev = torch.empty(need, dtype=torch.int64, device=self.device)
        dev.copy_(self._stage[:need], non_blocking=True)
        self._staged.record(torch.cuda.current_stream(self.device))
        return dev.split([c.shape[0] for c in cols])
