"""Norms of queries and keys per head and their rotation by position, in one pass on gfx950.

What stands between a projection to queries and keys and the cache that the keys go to (``cortex.kernels.paged_kv``):

    inv_freq = rotary_frequencies(head_dim, device="cuda")
    q, k = qk_norm_rope(q, k, positions, inv_freq, eps=1e-6, q_gain=wq, k_gain=wk)   # (T, heads, head_dim) each
    lengths = paged_kv_append(pages, k, v, block_table, lengths, offsets=offsets)

Images and video have several positions a token (time, height, width): ``positions`` (T, axes), and ``axes`` says which of
them turns a pair.  No reference counterpart: its model adds learned position rows (cortex/models/tokenizer.py:46-48).
Inference only: inputs that require a gradient or carry a forward-mode tangent are refused.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from cortex import _native as nat
from cortex.kernels.paged_kv import _get_device, _no_grad, _no_tangent, _overlap, _own_overlap

_WHAT = "qk_norm_rope"


def rotary_frequencies(dims: int, *, base: float = 10000.0, device: str | torch.device = "cuda") -> torch.Tensor:
    """``base ** (-2 p / dims)`` for the ``dims // 2`` pairs of ``dims`` rotated dims, fp32."""
    if dims < 2 or dims % 2:
        raise ValueError(f"dims must be even and positive, got {dims}")
    p = torch.arange(dims // 2, dtype=torch.float64)
    return (base ** (-2.0 * p / dims)).to(device=device, dtype=torch.float32)


def _rows(t: torch.Tensor, es: int) -> tuple[torch.Tensor, int, int]:
    """Rows that vector loads take, as given or copied, and the strides of their tokens and heads."""
    if t.is_contiguous():
        if t.data_ptr() & 15:
            t = t.clone()
        _, heads, dim = t.shape
        return t, heads * dim, dim
    st, sh, unit = t.stride()
    if unit != 1 or (t.data_ptr() | st * es | sh * es) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, _ = t.stride()
    return t, st, sh


def _check_out(out: tuple[torch.Tensor, torch.Tensor], q: torch.Tensor, k: torch.Tensor, es: int) -> None:
    for i, (y, own, x) in enumerate(((out[0], q, k), (out[1], k, q))):
        if y.shape != own.shape or y.dtype is not own.dtype:
            raise ValueError(f"out[{i}] must be a {tuple(own.shape)} {own.dtype} tensor, got {tuple(y.shape)} {y.dtype}")
        if y.numel() == 0:
            continue
        st, sh, unit = y.stride()
        if unit != 1 or (y.data_ptr() | st * es | sh * es) & 15:
            raise ValueError(f"the rows of out[{i}] must be contiguous and 16-byte aligned")
        if _own_overlap(y):
            raise ValueError(f"out[{i}] may not overlap itself (an expanded tensor)")
        same = y.data_ptr() == own.data_ptr() and y.stride() == own.stride()
        if (not same and _overlap(y, own)) or (x.numel() and _overlap(y, x)):
            raise ValueError("a result may be its own input, and overlaps no other")
    if out[0].numel() and out[1].numel() and _overlap(*out):
        raise ValueError("the results may not overlap each other")


def _gain(t: torch.Tensor | None, dim: int, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.shape != (dim,) or t.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name} must be ({dim},) in float32 or bfloat16, got {tuple(t.shape)} {t.dtype}")
    if not t.is_contiguous() or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 axes: torch.Tensor | None = None, interleaved: bool = False, eps: float | None = None,
                 q_gain: torch.Tensor | None = None, k_gain: torch.Tensor | None = None,
                 out: tuple[torch.Tensor, torch.Tensor] | None = None,
                 err_flag: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The queries and keys, each row (one head of one token) divided by its root mean square and rotated.

    ``q`` (T, heads, head_dim), ``k`` (T, kv_heads, head_dim) bf16 or fp32, any strides (views of a joint projection);
    ``head_dim`` a multiple of 8 up to 256.  With ``eps`` a row becomes ``x / sqrt(mean(x ** 2) + eps)``, times
    ``q_gain`` / ``k_gain`` (head_dim,) where given; without it rows are only rotated.  Squares are summed in fp32:
    ``sum(x ** 2)`` is to stay below 2^127, and ``mean(x ** 2) + eps`` from 2^-110 up (a row of zeros without eps is NaN).

    Pair p turns by ``positions[t, axes[p]] * inv_freq[p]`` (fp32 frequencies, the product rounded to 64 bits: exact up to
    positions of 2^29, further out off by at most 2^-53 of the angle, 2.4e-7 rad at 2^31 and 1.2e-4 at 2^40 where the
    frequency is 1): dims p and p + pairs, or 2p and 2p + 1 where ``interleaved``.  ``inv_freq`` (pairs,) with pairs a
    multiple of 8; the dims past 2 * pairs are not turned.  ``positions`` (T,) or (T, n) int64 of any strides, below 2^53 in
    amount; ``axes`` (pairs,) int32, by default axis 0 for every pair.  A pair whose axis is not there is not turned and
    sets bit 3 of ``err_flag`` (int32, never cleared here).  ``out``: where the results go; each may be its own input (in
    place) and overlaps no other tensor of the call."""
    idx = q.get_device()
    given = ()
    if axes is not None or eps is not None or err_flag is not None or out is not None:
        given = [t for t in (axes, q_gain, k_gain, err_flag) if t is not None]
        if out is not None:
            given += out
    elsewhere = idx < 0 or k.get_device() != idx or positions.get_device() != idx or inv_freq.get_device() != idx
    wants_grad = q.requires_grad or k.requires_grad or inv_freq.requires_grad
    for t in given:
        elsewhere = elsewhere or t.get_device() != idx
        wants_grad = wants_grad or t.requires_grad
    if elsewhere:
        nat.require_gpu(q, k, positions, inv_freq, *given, what=_WHAT)
    if idx != _get_device():
        with torch.cuda.device(idx):
            return qk_norm_rope(q, k, positions, inv_freq, axes=axes, interleaved=interleaved, eps=eps, q_gain=q_gain,
                                k_gain=k_gain, out=out, err_flag=err_flag)
    if wants_grad:
        _no_grad(_WHAT)
    if forward_ad._current_level >= 0:
        _no_tangent(_WHAT, q, k, inv_freq, *given)
    shape, k_shape, dtype = q.shape, k.shape, q.dtype
    if len(shape) != 3 or len(k_shape) != 3 or shape[0] != k_shape[0] or shape[2] != k_shape[2] or k.dtype is not dtype:
        raise ValueError(f"q and k must be (T, heads, head_dim) of one dtype, got {tuple(shape)} {dtype} and "
                         f"{tuple(k_shape)} {k.dtype}")
    if dtype is torch.bfloat16:
        code, es = nat.BF16, 2
    elif dtype is torch.float32:
        code, es = nat.F32, 4
    else:
        raise ValueError(f"rows of dtype {dtype} are not supported (bfloat16 or float32)")
    T, heads, dim = shape
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {dim}")
    if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float32 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous (pairs,) float32 tensor")
    pairs = inv_freq.shape[0]
    if pairs % 8 or 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs: a multiple of 8 up to half of the head_dim {dim} is needed")
    at = positions.shape
    if positions.dtype is not torch.int64 or len(at) not in (1, 2) or at[0] != T:
        raise ValueError(f"positions must be ({T},) or ({T}, axes) int64, got {tuple(at)} {positions.dtype}")
    if len(at) == 1:
        p_st, p_sa, n_axes = positions.stride(0), 0, 1
    else:
        (p_st, p_sa), n_axes = positions.stride(), at[1]
        if n_axes < 1:
            raise ValueError("positions need one axis at least")
    if axes is not None and (axes.dtype is not torch.int32 or axes.shape != (pairs,) or not axes.is_contiguous()):
        raise ValueError(f"axes must be a contiguous ({pairs},) int32 tensor")
    gain_code = nat.F32
    if eps is None:
        if q_gain is not None or k_gain is not None:
            raise ValueError("gains belong to the norm: give eps")
    elif not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    elif q_gain is not None or k_gain is not None:
        q_gain, k_gain = _gain(q_gain, dim, "q_gain"), _gain(k_gain, dim, "k_gain")
        if q_gain is not None and k_gain is not None and q_gain.dtype is not k_gain.dtype:
            raise ValueError(f"q_gain and k_gain of different dtypes: {q_gain.dtype} and {k_gain.dtype}")
        gain_code = nat.code((k_gain if q_gain is None else q_gain).dtype)
    if err_flag is not None and (err_flag.dtype is not torch.int32 or err_flag.numel() != 1):
        raise ValueError("err_flag must be one int32")
    if out is None:
        q_out, k_out = q.new_empty(shape), k.new_empty(k_shape)
        yt, yh, zt, zh = heads * dim, dim, k_shape[1] * dim, dim
    else:
        _check_out(out, q, k, es)
        q_out, k_out = out
        (yt, yh, _), (zt, zh, _) = q_out.stride(), k_out.stride()
    q, st, sh = _rows(q, es)
    k, kt, kh = _rows(k, es)
    nat.call("cortex_qk_norm_rope", T, heads, k_shape[1], dim, code, q.data_ptr(), st, sh, k.data_ptr(), kt, kh,
             positions.data_ptr(), p_st, p_sa, n_axes, pairs, inv_freq.data_ptr(), nat.ptr(axes), interleaved,
             eps is not None, 0.0 if eps is None else eps, nat.ptr(q_gain), nat.ptr(k_gain), gain_code, q_out.data_ptr(), yt,
             yh, k_out.data_ptr(), zt, zh, nat.ptr(err_flag), nat.stream_of(q_out.device))
    return q_out, k_out


__all__ = ["qk_norm_rope", "rotary_frequencies"]
