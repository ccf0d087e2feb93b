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
    cache.fork("a", ["a/1", "a/2"])                         # two more that go on from here

With ``bounded=True`` a step may attend to the pages alone that its largest scores may be in: ``attend(..., blocks=64)``.

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

from cortex.kernels.paged_kv import (KVPages, kv_block_bounds, kv_copy_pages, kv_evict_apply, kv_evict_plan, paged_attention,
                                     paged_block_select, paged_kv_append)


# Rows of a call of kv_copy_pages.  A workgroup takes 32 rows or more and a page 8 or more, so that these are at most
# 2^21 + 2^23 workgroups; a launch has fewer than 2^24.
_COPY_ROWS = 1 << 26


class KVBatch(NamedTuple):
    """Sessions of a step as the operators take them (device tensors): ``block_table`` (B, pages) int32, the slots in use
    before the step's tokens (``before``) and with them (``lengths``), ``offsets`` (B + 1,) of the tokens (None: one a
    session), their ``positions``, and on the host ``tokens``, ``max_length`` and ``max_new``, the most tokens of a session.
    It holds until one of its sessions is cut, dropped, forked or moved; ``append`` and ``attend`` refuse it from then on.
    ``filled``: the layers that have its tokens' rows; ``needs``: the same of every batch whose rows some layer lacked when
    this one was made, its own among them."""

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
    max_new: int


class _Session:
    __slots__ = ("pages", "used", "length", "seen", "version", "pending")

    def __init__(self) -> None:
        self.pages = np.empty(8, dtype=np.int32)
        self.used = 0  # pages owned: pages[:used]
        self.length = 0  # slots in use
        self.seen = 0  # tokens ever appended: the position of the next
        self.version = 0  # counts what makes batches of this session out of date
        self.pending: list[set[int]] = []  # ``filled`` of the batches whose rows some layer may lack


class _NoRoom(MemoryError, torch.OutOfMemoryError):
    """What ``resize`` raises where the device has no room: its own promise, and the kind of every other allocation."""


class PagedKVCache:
    """Pages of keys and values for named sessions, ``layers`` pools that share one block table."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, layers: int = 1, tracked: bool = False, bounded: bool = False,
                 device: str | torch.device = "cuda") -> None:
        if num_pages < 1 or layers < 1:
            raise ValueError("num_pages and layers must be >= 1")
        self.num_pages, self.page_size, self.tracked, self.bounded = num_pages, page_size, tracked, bounded
        shape, self._kind = (kv_heads, page_size, head_dim, dtype), {"tracked": tracked}
        if bounded:
            self._kind["bounded"] = True
        self.layers = [KVPages.allocate(num_pages, *shape, device, **self._kind) for _ in range(layers)]
        self.device = self.layers[0].device
        self._shape = (*shape, self.device)  # ("cuda" alone is whatever device is current)
        self._free = list(range(num_pages - 1, -1, -1))
        self._users = np.zeros(num_pages, dtype=np.int32)  # sessions that have a page
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
        victims, taken = self._room(total, set(names))
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
        self._take(victims, total)
        self._users[taken] = 1
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
                       self._stream, filled, tuple({id(f): f for s in held for f in s.pending}.values()),
                       int(new.max()) if B else 0)

    def batch(self, session_ids) -> KVBatch:
        """The sessions as they stand, without new tokens (KeyError: an unknown one)."""
        names = self._names(session_ids)
        for n in names:
            if n not in self._sessions:
                raise KeyError(f"unknown session {n!r}")
        return self.extend(names, [0] * len(names))

    def append(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
        """The rows (tokens, kv_heads, head_dim) of a batch's new tokens into ``layer``'s pages, session after session.  In
        a bounded cache the batches of a session in their order, and each once a layer: the bounds are those of the keys up to
        the batch's own."""
        if k.shape[0] != batch.tokens:
            raise ValueError(f"{k.shape[0]} rows for {batch.tokens} new tokens")
        at = layer % len(self.layers)
        if self.bounded:
            if at in batch.filled:
                raise RuntimeError(f"the batch's rows are in layer {layer} already")
            if any(at not in filled for filled in batch.needs if filled is not batch.filled):
                raise RuntimeError(f"an earlier batch of these sessions has no rows in layer {layer}: append them first")
        self._enter(batch)
        pages = self.layers[layer]
        paged_kv_append(pages, k, v, batch.block_table, batch.before, offsets=batch.offsets, positions=batch.positions)
        if self.bounded:
            kv_block_bounds(pages, batch.block_table, batch.lengths, since=batch.before, max_new=batch.max_new,
                            max_length=batch.max_length)
        batch.filled.add(at)

    def attend(self, batch: KVBatch, q: torch.Tensor, layer: int = 0, *, scale: float | None = None,
               accumulate: bool | None = None, blocks: int | None = None, first: int = 1, recent: int = 1,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """``paged_attention`` of one query (B, heads, head_dim) a session over its slots, the batch's new tokens among
        them: ``layer`` must have the rows of all of them by then (``append``), also of batches before this one (where
        one of those is given up, its sessions have to be dropped).  ``accumulate``: by default where the pages are
        tracked.  ``blocks``: attend to that many pages of a session at most, of each key head those that the largest scores
        may be in, the first ``first`` and the last ``recent`` among them (``paged_block_select``; a bounded cache, and a
        ``scale`` above 0)."""
        if blocks is not None and not self.bounded:
            raise ValueError("a selection of pages needs bounded=True")
        if blocks is not None and scale is not None and not scale > 0:
            raise ValueError(f"a selection of pages, which goes by the largest q . k, needs a scale above 0, got {scale}")
        if any(layer % len(self.layers) not in filled for filled in batch.needs):
            raise RuntimeError(f"some slots of the batch's sessions have no rows in layer {layer}: append them first")
        self._enter(batch)
        pages, table, lengths, most = self.layers[layer], batch.block_table, batch.lengths, batch.max_length
        if blocks is not None:
            table, lengths = paged_block_select(q, pages, table, lengths, blocks, first=first, recent=recent, max_length=most)
            most = min(most, blocks * self.page_size)
        return paged_attention(q, pages, table, lengths, scale=scale, out=out,
                               accumulate=self.tracked if accumulate is None else accumulate, max_length=most)

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
        self._filled(names)
        b = self.batch(names)
        # all plans, which need memory, before the first row moves: a session is cut in every layer or in none
        plans = [kv_evict_plan(pages, b.block_table, b.lengths, budget, recent, max_length=b.max_length)
                 for pages in self.layers]
        for pages, plan in zip(self.layers, plans):
            kv_evict_apply(pages, b.block_table, plan)
            if self.bounded:
                kv_block_bounds(pages, b.block_table, plan.lengths, max_length=budget)
        freed = 0
        for n in names:
            s = self._sessions[n]
            s.length = budget
            freed += self._release(s, -(-budget // self.page_size))
        return freed

    def fork(self, session_id: str, names) -> None:
        """New sessions ``names`` that go on from where ``session_id`` stands.  They share its full pages, and each gets a
        copy of the last one where it is in use in part; in a tracked cache, whose attention and eviction write to pages,
        each gets copies of all.  Every layer must have the rows of the session's tokens.  Sessions that are not in the call
        give way as for ``extend``; MemoryError, and nothing changed, when that is not enough.  Batches made before no
        longer hold for ``session_id``."""
        new = self._names(names)
        s = self._sessions.get(session_id)
        if s is None:
            raise KeyError(f"unknown session {session_id!r}")
        for n in new:
            if n in self._sessions:
                raise ValueError(f"there is a session {n!r} already")
        if not new:
            return
        self._filled((session_id,))
        shared = 0 if self.tracked else s.length // self.page_size
        own = s.used - shared
        total = own * len(new)
        victims, taken = self._room(total, {session_id})
        at = self._ids(np.tile(s.pages[shared:s.used], len(new)), np.array(taken, dtype=np.int32)) if total else ()

        # nothing that may fail comes after this
        self._take(victims, total)
        self._users[s.pages[:shared]] += len(new)
        self._users[taken] = 1
        s.version += 1
        self._epoch += 1
        self._sessions.move_to_end(session_id)
        for i, n in enumerate(new):
            f = self._sessions[n] = _Session()
            f.pages = np.concatenate([s.pages[:shared], np.array(taken[i * own:(i + 1) * own], dtype=np.int32)])
            f.used, f.length, f.seen = s.used, s.length, s.seen
        if at:
            for pages in self.layers:
                self._copy(pages, *at)

    def compact(self) -> int:
        """Moves pages so that those in use are the first ``pages_used`` of the pools; returns how many moved.  Every layer
        must have the rows of the tokens of sessions that move; batches made before no longer hold for these."""
        used = int((self._users > 0).sum())
        src = np.flatnonzero(self._users[used:] > 0).astype(np.int32) + used
        if src.shape[0] == 0:
            return 0
        place = np.arange(self.num_pages, dtype=np.int32)
        place[src] = np.flatnonzero(self._users[:used] == 0)
        moved = self._moved(place)
        at = self._ids(src, place[src])
        self._rename(place, moved, self.num_pages)
        for pages in self.layers:
            self._copy(pages, *at)
        return src.shape[0]

    def resize(self, num_pages: int) -> int:
        """Pools of ``num_pages`` pages instead (``layers`` are other objects then); returns how many pages got another
        place, those past the end of smaller pools.  MemoryError, and nothing changed, where the pages in use are more, or
        where the device has no room for the new pools beside the old ones (a torch.OutOfMemoryError too, then).  Every layer
        must have the rows of the tokens of sessions that move; batches made before no longer hold for these."""
        if num_pages < 1:
            raise ValueError("num_pages must be >= 1")
        src = np.flatnonzero(self._users > 0).astype(np.int32)
        if src.shape[0] > num_pages:
            raise MemoryError(f"{src.shape[0]} pages in use are more than {num_pages}")
        place = np.arange(self.num_pages, dtype=np.int32)
        past = src[src >= num_pages]
        place[past] = np.flatnonzero(self._users[:num_pages] == 0)[:past.shape[0]]
        moved = self._moved(place)
        self._not_captured()
        self._enter()
        layers = []
        try:
            layers = [KVPages.allocate(num_pages, *self._shape, **self._kind) for _ in self.layers]
            at = self._ids(src, place[src]) if src.shape[0] else ()
        except torch.OutOfMemoryError as e:
            layers.clear()  # (what was allocated does not live as long as the error)
            raise _NoRoom(f"no room on {self.device} for {num_pages} pages beside the {self.num_pages} there are: "
                          f"{e}") from e.with_traceback(None)
        self._rename(place, moved, num_pages)
        for old, new in zip(self.layers, layers):
            if at:
                self._copy(old, *at, into=new)
        self.layers = layers
        return past.shape[0]

    # ---------------------------------------------------------------------------

    def _room(self, total: int, keep: set[str]) -> tuple[list[str], list[int]]:
        """Sessions outside ``keep`` that have to give way for ``total`` pages, least recently used first, and the pages:
        the end of the free list as it is once they are gone, the last one first."""
        missing, victims, back = total - len(self._free), [], []
        if missing > 0:
            gone, users = [], self._users
            try:  # the counts as they are once these are gone, and back again: a copy would be one of all pages
                for name, s in self._sessions.items():
                    if len(back) >= missing:
                        break
                    if name not in keep and s.used:
                        pages = s.pages[:s.used]
                        gone.append((name, pages))
                        users[pages] -= 1
                        back += pages[users[pages] == 0].tolist()
                # (not those whose pages others keep)
                victims = [name for name, pages in gone if (users[pages] == 0).any()]
            finally:
                for _, pages in gone:
                    users[pages] += 1
            if len(back) < missing:
                raise MemoryError(f"{missing - len(back)} pages short of {total} (of {self.num_pages} in all)")
        taken = back[::-1][:total]
        return victims, taken + self._free[len(self._free) - (total - len(taken)):][::-1]

    def _take(self, victims: list[str], total: int) -> None:
        for name in victims:
            self.evict_session(name)
        del self._free[len(self._free) - total:]

    def _ids(self, *ids: np.ndarray) -> list[torch.Tensor]:
        """int32 arrays of one length on the device."""
        n = ids[0].shape[0]
        flat = np.zeros((len(ids), -(-n // 2) * 2), dtype=np.int32)
        flat[:, :n] = ids
        (dev,) = self._upload([flat.reshape(-1).view(np.int64)])
        return [t[:n] for t in dev.view(torch.int32).view(flat.shape)]

    def _copy(self, pages: KVPages, src: torch.Tensor, dst: torch.Tensor, into: KVPages | None = None) -> None:
        n = max(1, _COPY_ROWS // (self._shape[0] * self.page_size))
        for i in range(0, src.shape[0], n):
            kv_copy_pages(pages, src[i:i + n], dst[i:i + n], into=into)

    def _filled(self, names) -> None:
        for n in names:
            if any(len(f) < len(self.layers) for f in self._sessions[n].pending):
                raise RuntimeError(f"session {n!r} has slots without rows in some layer: append them first")

    def _moved(self, place: np.ndarray) -> list[str]:
        """Sessions that have a page whose place changes; refused where one lacks rows."""
        names = [n for n, s in self._sessions.items() if (place[s.pages[:s.used]] != s.pages[:s.used]).any()]
        self._filled(names)
        return names

    def _rename(self, place: np.ndarray, moved: list[str], num_pages: int) -> None:
        """Page p is page ``place[p]`` from now on, of ``num_pages``."""
        users = np.zeros(num_pages, dtype=np.int32)
        old = np.flatnonzero(self._users > 0)
        users[place[old]] = self._users[old]
        for n in moved:
            s = self._sessions[n]
            s.pages[:s.used] = place[s.pages[:s.used]]
            s.version += 1
        if moved:
            self._epoch += 1
        self._users, self.num_pages = users, num_pages
        self._free = np.flatnonzero(users == 0)[::-1].tolist()

    def _names(self, session_ids) -> tuple[str, ...]:
        names = tuple(session_ids)
        if isinstance(session_ids, str) or len(set(names)) != len(names):
            raise ValueError("session_ids must be distinct names")
        return names

    def _release(self, s: _Session, keep: int) -> int:
        """Pages of a session past the first ``keep`` go back to the free list (the last one first out)."""
        s.version += 1
        self._epoch += 1
        pages = s.pages[keep:s.used]
        self._users[pages] -= 1
        free = pages[self._users[pages] == 0].tolist()
        self._free.extend(free)
        s.used = keep
        return len(free)

    def _enter(self, batch: KVBatch | None = None) -> None:
        """Before an operator: the batch still holds, and what another stream was given here comes first."""
        if batch is not None and batch.epoch != self._epoch:
            for name, s, version in zip(batch.sessions, batch.held, batch.versions):
                if s.version != version:
                    raise RuntimeError(f"the batch is out of date: session {name!r} was cut, dropped, forked or moved since")
        stream = torch.cuda.current_stream(self.device)
        if self._stream != stream:
            self._not_captured()
            done = torch.cuda.Event()
            done.record(self._stream)
            stream.wait_event(done)
            for p in self.layers:
                for t in (p.k, p.v, p.k_scale, p.v_scale, p.weight, p.position, p.bounds if self.bounded else None):
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
