"""Bounds of pages, their selection and the rotation by position in plain form, in 64 bits on the CPU."""

from __future__ import annotations

import numpy as np
import torch

from _paged import DEV, Cache


class BoundedCache(Cache):
    """A ``Cache`` whose pages have bounds: 7 everywhere until they are computed."""

    def __init__(self, *args, **kw):
        from cortex.kernels.paged_kv import KVPages

        super().__init__(*args, **kw)
        p = self.pages
        kind = torch.float32 if p.k.dtype == torch.int8 else p.k.dtype
        self.gb = torch.full((self.num, self.kv_heads, 2, self.dim), 7.0, dtype=kind, device=DEV)
        self.pages = KVPages(p.k, p.v, k_scale=p.k_scale, v_scale=p.v_scale, weight=p.weight, position=p.position,
                             bounds=self.gb)

    def bounds64(self, b, block, n=None):
        """(kv_heads, 2, dim): largest and smallest value of the keys of a block that are in use."""
        n = self.lens[b] if n is None else n
        rows = self.k[int(self.table[b][block]), :, :min(self.page, n - block * self.page)].double()
        return torch.stack([rows.amax(1), rows.amin(1)], 1)

    def fill_bounds(self):
        want = torch.full(self.gb.shape, 7.0, dtype=torch.float64)
        for b, n in enumerate(self.lens):
            for i in range(-(-n // self.page)):
                want[int(self.table[b][i])] = self.bounds64(b, i)
        self.gb.copy_(want.to(self.gb.dtype))
        return want


def select64(table, bounds, q, n, page, count, first, recent, num_pages):
    """Blocks kept of one sequence and key head.  ``bounds`` (num_pages, 2, dim) of that head and ``q`` (group, dim), both
    fp64 numpy: products and sums of numbers of at most 24 bits in 64 bits, then one rounding."""
    blocks = -(-n // page)
    if blocks <= count:
        return list(range(blocks))
    ids = np.asarray(table[:blocks], dtype=np.int64)
    there = (ids >= 0) & (ids < num_pages)
    rows = bounds[np.where(there, ids, 0)]
    with np.errstate(invalid="ignore", over="ignore"):
        up, down = np.where(q < 0, 0.0, q), np.where(q < 0, q, 0.0)
        each = np.stack([(u * rows[:, 0] + d * rows[:, 1]).sum(-1) for u, d in zip(up, down)], 1).astype(np.float32)
    lost = np.isnan(each).any(1)
    score = np.where(lost, 0.0, np.where(np.isnan(each), 0.0, each).max(1))
    rank = [(2 if n else 1, float(x)) if t else (0, 0.0) for t, n, x in zip(there.tolist(), lost.tolist(), score.tolist())]
    always = [i < first or i >= blocks - recent for i in range(blocks)]
    order = sorted(range(blocks), key=lambda i: (not always[i], -rank[i][0], -rank[i][1], i))
    return sorted(order[:count])


def rope64(x, positions, inv_freq, axes, interleaved, eps, gain):
    """``(y, |x'_i| |cos| + |x'_j| |sin|, |x'_i| + |x'_j|)``: the rotated rows and what the bounds of their error need."""
    T, heads, dim = x.shape
    x = x.double()
    if eps is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        if gain is not None:
            x = x * gain.double()
    pairs = inv_freq.shape[0]
    pos = positions.reshape(T, -1).double()
    y, a, b = x.clone(), x.abs(), x.abs()
    for p in range(pairs):
        axis = 0 if axes is None else int(axes[p])
        if not 0 <= axis < pos.shape[1]:
            continue
        angle = pos[:, axis] * inv_freq[p].double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        a[..., i] = x[..., i].abs() * c.abs() + x[..., j].abs() * s.abs()
        a[..., j] = x[..., j].abs() * c.abs() + x[..., i].abs() * s.abs()
        b[..., i] = b[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, a, b


def rope_bound(y, a, b, dim, normed, dtype):
    """What the arithmetic of a rotated row may be off by, with u = 2^-24 (half a step of fp32):
      * the mean of dim squares: (dim + 2) u of it, with eps one more; the root halves that; root, quotient and the two
        products of x' add u each: (dim / 2 + 6) u of x'; rows that are only rotated are exact;
      * the two products and the sum of a rotation: 3 u of |x'_i cos| + |x'_j sin|;
      * sine and cosine: their argument, at most pi/4, rounded to fp32 (u), and two steps (4 u) of the functions
        themselves: 5 u of |x'_i| + |x'_j|;
      * one rounding to the rows' type."""
    u = 2.0 ** -24
    half = u if dtype == torch.float32 else 2.0 ** -8
    t = ((dim / 2 + 6) * u if normed else 0.0) * a + 3 * u * a + 5 * u * b
    return 1.01 * (t + half * (y.abs() + t)) + 1e-37
