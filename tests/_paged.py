"""Paged caches for the tests, and the operators on them in 64 bits on the CPU."""

from __future__ import annotations

import numpy as np
import torch

DEV = "cuda"


def codes(x: torch.Tensor):
    """Rows as int8 codes and fp32 scales, the quantisation of the package's weights per row."""
    s = x.abs().amax(-1).clamp_min(1e-8) / x.new_full((), 127.0)
    return (x / s[..., None]).round().clamp_(-127, 127).to(torch.int8), s


class Cache:
    """Pages on the GPU that hold known rows, and NaN (int8: the largest codes at scale NaN) wherever no row is."""

    def __init__(self, lens, kv_heads, dim, page, dtype, *, seed=0, room=0, tracked=False, layout="head", std=1.0,
                 extra=2):
        from cortex.kernels.paged_kv import KVPages

        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.page, self.kv_heads, self.dim = g, list(lens), page, kv_heads, dim
        B = len(self.lens)
        self.width = max(1, max(-(-(n + room) // page) for n in self.lens)) if B else 1
        self.num = B * self.width + extra
        self.table = torch.randperm(self.num, generator=g)[:B * self.width].reshape(B, self.width).int()
        shape = (self.num, kv_heads, page)
        self.k, self.v = (torch.full((*shape, dim), float("nan")) for _ in range(2))
        self.weight = torch.full(shape, float("nan"))
        self.position = torch.full(shape, 2 ** 30, dtype=torch.int32)
        for b, n in enumerate(self.lens):
            at = self.at(b, torch.arange(n))
            self.k[at] = torch.randn(n, kv_heads, dim, generator=g) * std
            self.v[at] = torch.randn(n, kv_heads, dim, generator=g)
            self.weight[at] = torch.rand(n, kv_heads, generator=g)
            self.position[at] = torch.arange(n, dtype=torch.int32)[:, None]
        self.k_scale = self.v_scale = None
        if dtype == torch.int8:
            (kc, self.k_scale), (vc, self.v_scale) = codes(self.k), codes(self.v)
            kc[torch.isnan(self.k_scale)] = 127
            vc[torch.isnan(self.v_scale)] = -127
            self.k_codes, self.v_codes = kc, vc
            self.k, self.v = (c.float() * s[..., None] for c, s in ((kc, self.k_scale), (vc, self.v_scale)))
            pools = [kc, vc]
        else:
            self.k, self.v = self.k.to(dtype), self.v.to(dtype)
            pools = [self.k, self.v]
        self.gk, self.gv = (self._place(t, layout) for t in pools)
        more = {}
        if self.k_scale is not None:
            more = {"k_scale": self.k_scale.to(DEV), "v_scale": self.v_scale.to(DEV)}
        if tracked:
            more |= {"weight": self.weight.to(DEV), "position": self.position.to(DEV)}
        self.pages = KVPages(self.gk, self.gv, **more)
        self.block_table = self.table.to(DEV)
        self.lengths = torch.tensor(self.lens, dtype=torch.int64, device=DEV)

    def _place(self, t, layout):
        if layout == "head":  # (page, head, row, dim)
            return t.to(DEV).contiguous()
        if layout == "row":  # stored as (page, row, head, dim)
            return t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        big = torch.full((t.shape[0], 2, t.shape[1], t.shape[2], t.shape[3] + 32), 77).to(t.dtype).to(DEV)
        big[:, 1, :, :, 16:16 + t.shape[3]] = t.to(DEV)  # one plane of a larger pool, rows with a gap
        return big[:, 1, :, :, 16:16 + t.shape[3]]

    def at(self, b, slots):
        """Index of (len(slots), kv_heads) rows of sequence b in the pools."""
        return self.table[b][slots // self.page].long(), slice(None), slots % self.page

    def query(self, heads, *, std=1.0):
        dtype = self.pages.query_dtype
        return (torch.randn(len(self.lens), heads, self.dim, generator=self.g) * std).to(dtype)


def attention64(c: Cache, q: torch.Tensor, scale=None, lens=None):
    """``(out, weight added per sequence, bound of out, bound of the weight)``, all in 64 bits.

    The bounds are what the arithmetic may be off by, with u = 2^-24 (half a step of fp32):
      * a score is a sum of Dh products in fp32, then a product with the scale and, int8, one with the row's scale:
        |ds| <= (Dh + 4) u * scale * sum_d |q_d k_d|; exp of it is off by a factor within exp(+-|ds|) and its own error;
      * the running sums over n keys and their joins add (n + 64) u each to numerator and denominator;
      * bf16 and int8: the probabilities enter the second product as two bf16 values, the upper half of the bits (less than a
        step, 2^-7, below) and the rest rounded (half a step of it): 2^-15 of each; the result is rounded to bf16
        (2^-8 of it); fp32: u."""
    n_seq, heads, dim = q.shape
    group = heads // c.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    u = 2.0 ** -24
    half = u if q.dtype == torch.float32 else 2.0 ** -8
    out = torch.zeros(n_seq, heads, dim, dtype=torch.float64)
    tol = torch.zeros_like(out)
    added, added_tol = [], []
    for b, n in enumerate(lens or c.lens):
        at = c.at(b, torch.arange(n))
        k, v = c.k[at].double(), c.v[at].double()
        w = torch.zeros(n, c.kv_heads, dtype=torch.float64)
        wt = torch.zeros_like(w)
        for h in range(heads if n else 0):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[b, h].double()
            s = kh @ qh * scale
            p = torch.softmax(s, 0)
            ds = float(((dim + 4) * u * abs(scale) * (kh.abs() @ qh.abs())).max()) + 8 * u * (1 + float(s.abs().max()))
            rel = 2 * ds + 2 * (n + 64) * u
            out[b, h] = p @ vh
            mass = p @ vh.abs()
            tol[b, h] = 1.01 * (rel * mass + (2.0 ** -15 * mass if half > u else 0) + half * out[b, h].abs()) + 1e-37
            w[:, h // group] += p
            wt[:, h // group] += p * (rel + group * u)
        added.append(w)
        added_tol.append(1.01 * wt)
    return out, added, tol, added_tol


def evict64(weight, position, n, budget, recent):
    """``(dst, src)`` of one head: slots given up below the budget and kept ones past it, ascending."""
    if n <= budget:
        return [], []
    w, pos = weight[:n].double().numpy().copy(), position[:n].numpy().astype(np.int64)
    young = pos > pos.max() - recent
    w[young] = 0.0  # equal among themselves
    nan = np.isnan(w)
    order = np.lexsort((np.arange(n), -np.where(nan, 0, w), ~nan, ~young))
    keep = np.zeros(n, dtype=bool)
    keep[order[:budget]] = True
    return [i for i in range(budget) if not keep[i]], [i for i in range(budget, n) if keep[i]]
