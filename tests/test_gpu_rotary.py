"""``qk_norm_rope`` against a plain computation in 64 bits (tests/_blocks.py), within bounds derived from its arithmetic."""

from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from _blocks import rope64, rope_bound
from _paged import DEV

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


class Case:
    def __init__(self, T, heads, kv_heads, dim, pairs, dtype, *, axes=1, far=1000, seed=0, gains=True, gain_dtype=None):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dim = dtype, dim
        self.q = torch.randn(T, heads, dim, generator=g).to(dtype)
        self.k = (torch.randn(T, kv_heads, dim, generator=g) * 3).to(dtype)
        self.positions = torch.randint(-far, far, (T, axes), generator=g)
        self.inv_freq = (10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).float()
        self.axes = torch.randint(0, axes, (pairs,), generator=g).int() if axes > 1 else None
        self.gains = [None, None]
        if gains:
            self.gains = [(1 + 0.3 * torch.randn(dim, generator=g)).to(gain_dtype or dtype) for _ in range(2)]

    def run(self, *, eps=1e-6, interleaved=False, q=None, k=None, positions=None, **kw):
        from cortex.kernels.rotary import qk_norm_rope

        up = lambda t: None if t is None else t.to(DEV)
        if eps is not None:
            kw |= {"q_gain": up(self.gains[0]), "k_gain": up(self.gains[1])}
        return qk_norm_rope(up(self.q) if q is None else q, up(self.k) if k is None else k,
                            up(self.positions) if positions is None else positions, up(self.inv_freq), axes=up(self.axes),
                            interleaved=interleaved, eps=eps, **kw)

    def check(self, got, *, eps=1e-6, interleaved=False):
        for name, x, gain, y in zip(("q", "k"), (self.q, self.k), self.gains, got):
            want, a, b = rope64(x, self.positions, self.inv_freq, self.axes, interleaved, eps, gain)
            tol = rope_bound(want, a, b, self.dim, eps is not None, self.dtype)
            assert y.shape == x.shape and y.dtype == x.dtype
            off = (y.double().cpu() - want).abs()
            bad = ~(off <= tol)
            assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max())} times "
                                   f"what is allowed, first at {bad.nonzero()[0].tolist()}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("heads,kv_heads,dim,pairs", [
    (1, 1, 8, 0), (1, 1, 16, 8), (8, 8, 64, 32), (12, 12, 64, 16), (4, 2, 96, 48), (3, 1, 80, 8), (32, 8, 128, 64),
    (5, 1, 120, 56), (7, 0, 32, 16), (0, 3, 32, 16), (2, 2, 256, 128), (9, 3, 192, 72), (40, 40, 128, 32), (1, 1, 248, 120)])
def test_heads_dims_and_pairs(dtype, interleaved, heads, kv_heads, dim, pairs):
    for eps in (None, 1e-6):
        c = Case(37, heads, kv_heads, dim, pairs, DTYPES[dtype], seed=dim + pairs)
        c.check(c.run(eps=eps, interleaved=interleaved), eps=eps, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 63, 64, 65, 1000, 2049, 5003, 20011])
def test_lengths(dtype, T):
    c = Case(T, 3, 1, 64, 32, DTYPES[dtype], seed=T)
    c.check(c.run())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("axes", [2, 3, 5])
def test_several_axes(dtype, axes):
    c = Case(301, 4, 2, 64, 32, DTYPES[dtype], axes=axes, seed=axes)
    for interleaved in (False, True):
        c.check(c.run(interleaved=interleaved), interleaved=interleaved)
    # positions kept by axis
    c.check(c.run(positions=c.positions.t().contiguous().to(DEV).t()))
    # every pair by the first axis where no axes are given
    c.axes = None
    c.check(c.run())


@pytest.mark.parametrize("far", [1, 1 << 20, 1 << 31, 1 << 40, 1 << 52])
def test_far_positions(far):
    """Angles of far positions, in both directions: the product and its reduction are in 64 bits."""
    c = Case(400, 2, 2, 64, 32, torch.float32, far=far, seed=3)
    c.positions[:4, 0] = torch.tensor([0, far, -far, far - 1])
    for eps in (None, 1e-5):
        c.check(c.run(eps=eps), eps=eps)


PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


@pytest.mark.parametrize("far", [1 << 20, 1 << 29, 1 << 31, 1 << 40, (1 << 53) - 1])
def test_far_positions_by_exact_angles(far):
    """Angles as fractions, without the rounding of the product: up to 2^29 (29 bits times 24) there is none, further out
    the angle is off by half a unit of the 64-bit product, at most 2^-53 of it, times |x_i| + |x_j| in the result."""
    c = Case(40, 1, 1, 64, 32, torch.float32, far=far, seed=6, gains=False)
    c.positions[:4, 0] = torch.tensor([far, -far, far - 1, far // 3])
    angle = [[int(p) * Fraction(float(f)) for f in c.inv_freq] for p in c.positions[:, 0]]
    product = c.positions.double() * c.inv_freq.double()
    apart = [[float(abs(a - Fraction(float(x)))) for a, x in zip(r, s)] for r, s in zip(angle, product)]
    off = torch.tensor(apart, dtype=torch.float64)
    assert (off == 0).all() if far <= 1 << 29 else (off <= 2.0 ** -53 * product.abs()).all() and off.any()
    small = torch.tensor([[float(a - round(a / (2 * PI)) * 2 * PI) for a in r] for r in angle], dtype=torch.float64)[:, None]
    for x, y in zip((c.q, c.k), c.run(eps=None)):
        u, v = x.double()[..., :32], x.double()[..., 32:]
        cos, sin = small.cos(), small.sin()
        want = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
        near = torch.cat([u.abs() * cos.abs() + v.abs() * sin.abs(), v.abs() * cos.abs() + u.abs() * sin.abs()], -1)
        size = torch.cat([u.abs() + v.abs()] * 2, -1)
        # (2^-50: the reduced angle and its functions in 64 bits here)
        tol = rope_bound(want, near, size, 64, False, torch.float32) + (torch.cat([off, off], -1)[:, None] + 2.0 ** -50) * size
        assert ((y.double().cpu() - want).abs() <= tol).all(), far


@pytest.mark.parametrize("dtype", DTYPES)
def test_gains(dtype):
    c = Case(50, 4, 2, 64, 32, DTYPES[dtype], gains=False)
    c.check(c.run())
    for kind in (torch.float32, torch.bfloat16):
        c = Case(50, 4, 2, 64, 32, DTYPES[dtype], gain_dtype=kind)
        c.check(c.run())
        both = list(c.gains)
        for which in (0, 1):
            c.gains = [g if i == which else None for i, g in enumerate(both)]
            c.check(c.run())
    odd = torch.zeros(65, dtype=torch.float32, device=DEV)[1:]  # not 16-byte aligned
    odd.copy_(both[0])
    from cortex.kernels.rotary import qk_norm_rope

    got = qk_norm_rope(c.q.to(DEV), c.k.to(DEV), c.positions.to(DEV), c.inv_freq.to(DEV), eps=1e-6, q_gain=odd)
    c.gains = [odd.cpu(), None]
    c.check(got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_places(dtype):
    c = Case(77, 6, 2, 64, 32, DTYPES[dtype], seed=1)
    joint = torch.full((77, 11, 64), 9.0, dtype=c.dtype, device=DEV)  # of a joint projection
    q, k = joint[:, :6], joint[:, 7:9]
    q.copy_(c.q), k.copy_(c.k)
    before = joint.clone()
    want = c.run(q=q, k=k)
    c.check(want)
    assert torch.equal(joint, before)
    # heads outside, and a tensor off its alignment
    c.check(c.run(q=c.q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)))
    odd = torch.zeros(c.q.numel() + 1, dtype=c.dtype, device=DEV)[1:].view(c.q.shape)
    odd.copy_(c.q)
    c.check(c.run(q=odd))
    wide = torch.zeros(77, 6, 128, dtype=c.dtype, device=DEV)[:, :, ::2]  # head_dim not contiguous
    wide.copy_(c.q)
    c.check(c.run(q=wide))
    # one token for all (queries read only)
    c2 = Case(77, 6, 2, 64, 32, DTYPES[dtype], seed=1)
    c2.q = c2.q[:1].expand(77, 6, 64)
    c2.check(c2.run(q=c2.q[:1].to(DEV).expand(77, 6, 64)))
    # into given places, and in place
    place = torch.full((77, 11, 64), 9.0, dtype=c.dtype, device=DEV)
    got = c.run(q=q, k=k, out=(place[:, 1:7], place[:, 9:11]))
    assert got[0].data_ptr() == place[:, 1:7].data_ptr()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (place[:, 0] == 9).all() and (place[:, 7:9] == 9).all()
    c.run(q=q, k=k, out=(q, k))
    assert torch.equal(joint[:, :6], want[0]) and torch.equal(joint[:, 7:9], want[1])
    assert torch.equal(joint[:, [6, 9, 10]], before[:, [6, 9, 10]])


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_ends(dtype):
    """Rows of zeros, infinities and NaN stay in their rows; large and small numbers; eps 0."""
    c = Case(40, 2, 1, 64, 32, DTYPES[dtype], seed=2)
    c.q[3, 0] = 0.0
    c.q[4] *= 1e15
    c.q[5] *= 1e-15
    c.check(c.run())
    c.check(c.run(eps=1e-30), eps=1e-30)
    plain = c.run()[0]
    for value in (float("inf"), float("-inf"), float("nan")):
        c.q[7, 1, 5] = value
        got = c.run()[0]
        others = torch.ones(40, 2, dtype=torch.bool)
        others[7, 1] = False
        assert torch.equal(got.cpu()[others], plain.cpu()[others])
        assert got[7, 1, 5].isnan()
        got = c.run(eps=None)[0]  # without the norm the pair alone
        assert not got[7, 1, 5].isfinite() and not got[7, 1, 37].isfinite()
        keep = [d for d in range(64) if d not in (5, 37)]
        assert got[7, 1, keep].isfinite().all()
    c.q[7, 1] = 0.0
    got = c.run(eps=0.0)[0]
    assert got[7, 1].isnan().all() and got[8].isfinite().all()  # 0 / 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -53, 1.0, 2.0 ** 59])
def test_rows_at_either_end_without_eps(dtype, size):
    """Squares are summed in fp32: a mean from 2^-110 up loses nothing to numbers below the normal ones (256 squares that
    are off by 2^-150 each: 2^-40 of their sum), and sums below 2^127 have room."""
    c = Case(30, 2, 2, 256, 32, DTYPES[dtype], seed=11)
    c.q, c.k = (x / x.double().square().mean(-1, keepdim=True).sqrt() * size for x in (c.q, c.k))
    c.q, c.k = c.q.to(c.dtype), c.k.to(c.dtype)
    c.check(c.run(eps=0.0), eps=0.0)


def test_axes_that_are_not_there():
    """Such pairs are not turned, and the flag says so."""
    c = Case(20, 2, 2, 64, 32, torch.float32, axes=3)
    c.axes[4], c.axes[9], c.axes[31] = 3, -1, 2 ** 31 - 1
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.check(c.run(err_flag=flag))
    assert flag.item() == 8
    c.check(c.run())
    c.axes.clamp_(0, 2)
    flag.zero_()
    c.check(c.run(err_flag=flag))
    assert flag.item() == 0


def test_nothing_to_do():
    c = Case(0, 4, 2, 64, 32, torch.bfloat16)
    q, k = c.run()
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    c = Case(5, 0, 0, 64, 32, torch.bfloat16)
    q, k = c.run()
    assert q.shape == k.shape == (5, 0, 64)


def test_refusals():
    from cortex.kernels.rotary import qk_norm_rope, rotary_frequencies

    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(4, 1, 64, dtype=torch.bfloat16, device=DEV)
    pos, freq = torch.arange(4, device=DEV), rotary_frequencies(64)
    gain = torch.ones(64, device=DEV)

    def refused(match, q=q, k=k, pos=pos, freq=freq, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            qk_norm_rope(q, k, pos, freq, **kw)

    refused("one dtype", k=k.float())
    refused("one dtype", k=k[:3])
    refused("one dtype", k=k[..., :32])
    refused("one dtype", q=q[0], k=k[0])
    refused("not supported", q=q.half(), k=k.half())
    refused("head_dim", q=q[..., :60], k=k[..., :60])
    refused("head_dim", q=q.repeat(1, 1, 5), k=k.repeat(1, 1, 5))
    refused("inv_freq", freq=freq.double())
    refused("inv_freq", freq=freq[::2])
    refused("inv_freq", freq=freq[None])
    refused("pairs", freq=freq[:12])
    refused("pairs", freq=rotary_frequencies(128))
    refused("positions", pos=pos.int())
    refused("positions", pos=pos[:3])
    refused("positions", pos=pos[:, None, None])
    refused("one axis", pos=pos[:, None][:, :0])
    refused("axes", axes=torch.zeros(32, dtype=torch.int64, device=DEV))
    refused("axes", axes=torch.zeros(16, dtype=torch.int32, device=DEV))
    refused("eps", q_gain=gain)
    refused("eps", eps=-1e-6)
    refused("eps", eps=float("nan"))
    refused("q_gain", eps=1e-6, q_gain=gain[:32])
    refused("k_gain", eps=1e-6, k_gain=gain.half())
    refused("different dtypes", eps=1e-6, q_gain=gain, k_gain=gain.bfloat16())
    refused("err_flag", err_flag=torch.zeros(2, dtype=torch.int32, device=DEV))
    refused("ROCm GPU", pos=pos.cpu(), error=RuntimeError)
    refused("ROCm GPU", q=q.cpu(), error=RuntimeError)
    refused(r"out\[0\]", out=(q.float(), k))
    refused(r"out\[1\]", out=(q, q))
    refused("overlap itself", out=(q[:1].expand(4, 2, 64), k))
    refused("contiguous", out=(torch.zeros(4, 2, 128, dtype=q.dtype, device=DEV)[..., ::2], k))
    both = torch.zeros(4, 4, 64, dtype=q.dtype, device=DEV)
    refused("own input", q=both[:, :2], out=(both[:, 1:3], k))
    refused("own input", q=both[:, :2], out=(torch.empty_like(q), both[:, :1]))
    refused("each other", out=(both[:, :2], both[:, 1:2]))
    refused("no backward", q=q.clone().requires_grad_(), error=RuntimeError)
    refused("no backward", eps=1e-6, q_gain=gain.clone().requires_grad_(), error=RuntimeError)
    with torch.no_grad():
        qk_norm_rope(q.clone().requires_grad_(), k, pos, freq)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        refused("tangents", q=fwd.make_dual(q, torch.ones_like(q)), error=RuntimeError)
    for dims in (0, 7, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(dims)


def test_frequencies():
    from cortex.kernels.rotary import rotary_frequencies

    got = rotary_frequencies(64, base=500000.0).cpu().double()
    want = torch.tensor([500000.0 ** (-2 * p / 64) for p in range(32)], dtype=torch.float64)
    assert ((got - want).abs() <= 2.0 ** -24 * want * 1.01).all()


def test_other_streams_and_graphs():
    c = Case(130, 4, 2, 64, 32, torch.bfloat16, seed=4)
    want = c.run()
    q, k = c.q.to(DEV), c.k.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(q=q, k=k)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pos, freq = c.positions.to(DEV), c.inv_freq.to(DEV)
    gains = [g.to(DEV) for g in c.gains]
    from cortex.kernels.rotary import qk_norm_rope

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = qk_norm_rope(q, k, pos, freq, eps=1e-6, q_gain=gains[0], k_gain=gains[1])
    for step in range(4):
        other = Case(130, 4, 2, 64, 32, torch.bfloat16, seed=10 + step)
        q.copy_(other.q), k.copy_(other.k), pos.copy_(other.positions)
        graph.replay()
        other.gains = c.gains
        eager = other.run()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
