"""What the operators around a paged K/V decode step are measured on, and what their results have to be.

  rope        ``qk_norm_rope``: the norms of queries and keys per head and the rotation by position, in one pass
  copy        ``kv_copy_pages``: pages of a pool into others (a fork, a compaction)
  bounds      ``kv_block_bounds``: the largest and smallest value of a page's keys in every dim
  select      ``paged_block_select``: the pages that a query may find its largest scores in
  sparse      ``paged_block_select`` and ``paged_attention`` over what it selected

``listed`` gives the fixed cases and ``draw`` further ones of the same ranges; ``prepare`` makes what a
program holds before the call, ``run`` is one pass, ``work`` what it cannot do without, ``exact`` its
results in 64 bits.  With ``own`` false ``run`` computes the operators from elementary torch operations.

Slot j of sequence b lives in page ``table[b, j // page]``, row ``j % page``; the pools are
(pages, kv heads, page, head dim), the bounds (pages, kv heads, 2, head dim): largest, then smallest.
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "cortex-engine_amd")
_TOKENS = 1 << 17  # cached tokens of the largest cases


def listed():
    return [
        # one token of one stream at the middle configuration's heads, rotated only: the smallest call, all latency
        {"name": "rope_b1", "kind": "rope", "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 64, "rotary": 64, "axes": 1,
         "interleaved": False, "norm": False, "far": 600, "dtype": "bfloat16"},
        # ragged prompts, queries and keys as columns of one joint projection, far positions
        {"name": "rope_prompts", "kind": "rope", "tokens": 16801, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "axes": 1, "interleaved": False, "norm": True, "far": 1 << 20, "dtype": "bfloat16"},
        # patches of a video at the largest configuration's heads in fp32: time, height and width, half of a head rotated
        {"name": "rope_axes_fp32", "kind": "rope", "tokens": 4999, "heads": 12, "kv_heads": 12, "dim": 64, "rotary": 32,
         "axes": 3, "interleaved": True, "norm": True, "far": 4096, "dtype": "float32"},
        # one stream forked: the page that both would write to
        {"name": "copy_b1", "kind": "copy", "pages": 1, "kv_heads": 8, "dim": 64, "page": 16, "pool": "bfloat16",
         "tracked": False},
        # long prompts forked whole, with the weight and the positions of their rows
        {"name": "copy_prompts", "kind": "copy", "pages": 2053, "kv_heads": 8, "dim": 128, "page": 16,
         "pool": "bfloat16", "tracked": True},
        # a decode step of 32 sequences: the bounds of the pages that their tokens went to
        {"name": "bounds_step_b32", "kind": "bounds", "batch": 32, "lo": 150, "hi": 8003, "new": 1, "kv_heads": 8,
         "dim": 128, "page": 16, "pool": "bfloat16"},
        # after prompts into an int8 cache: the bounds of all of its pages
        {"name": "bounds_prompts_int8", "kind": "bounds", "batch": 16, "lo": 1000, "hi": 15001, "new": 0, "kv_heads": 4,
         "dim": 128, "page": 32, "pool": "int8"},
        # one short stream, a key head for every query head: latency
        {"name": "select_b1_short", "kind": "select", "batch": 1, "lo": 600, "hi": 600, "heads": 8, "kv_heads": 8,
         "dim": 64, "page": 16, "pool": "bfloat16", "count": 16},
        # a serving batch of ragged lengths on small pages: many blocks
        {"name": "select_b32_ragged", "kind": "select", "batch": 32, "lo": 150, "hi": 8003, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "pool": "bfloat16", "count": 64},
        # one sequence with a very long cache, an eighth of it attended to
        {"name": "sparse_b1_long", "kind": "sparse", "batch": 1, "lo": 131072, "hi": 131072, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "pool": "bfloat16", "count": 256},
        # the same batch of ragged lengths, each down to 2048 keys at most
        {"name": "sparse_b32_ragged", "kind": "sparse", "batch": 32, "lo": 150, "hi": 8003, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "pool": "bfloat16", "count": 64},
        # the fp32 mode at the largest configuration's twelve heads
        {"name": "sparse_b8_fp32", "kind": "sparse", "batch": 8, "lo": 101, "hi": 2049, "heads": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "pool": "float32", "count": 24},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("rope", "copy", "bounds", "select", "sparse"))
    dim = rng.choice((32, 64, 96, 128))
    if kind == "rope":
        kv = rng.choice((1, 2, 4, 8, 12))
        return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "heads": kv * rng.choice((1, 2, 3, 4)), "kv_heads": kv,
                "dim": dim, "rotary": rng.choice([r for r in (16, 32, 48, 64, 96, 128) if r <= dim]),
                "axes": rng.choice((1, 1, 2, 3)), "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.7,
                "far": _log_int(rng, 16, 1 << 24), "dtype": rng.choice(("bfloat16", "float32"))}
    case = {"kind": kind, "kv_heads": rng.choice((1, 2, 4, 8, 12)), "dim": dim,
            "page": rng.choice((8, 16, 32, 64, 128))}
    if kind == "copy":
        pool = rng.choice(("bfloat16", "bfloat16", "float32"))
        most = 32768 * 1024 // (case["kv_heads"] * dim * case["page"] * _bytes_of(pool) // 2)
        return {**case, "pages": _log_int(rng, 1, most), "pool": pool, "tracked": rng.random() < 0.5}
    case["pool"] = rng.choice(("bfloat16", "bfloat16", "int8", "float32"))
    case["batch"] = batch = _log_int(rng, 1, 64)
    # (cached values of a case: what 2^17 tokens of four heads in bf16 are)
    hi = _log_int(rng, 1, min(32768, _TOKENS * 8 // (batch * case["kv_heads"] * _bytes_of(case["pool"]))))
    case["lo"], case["hi"] = (rng.randint(0, hi) if rng.random() < 0.7 else hi), hi
    if kind == "bounds":
        return {**case, "new": rng.choice((0, 1))}
    blocks = -(-hi // case["page"])
    return {**case, "heads": case["kv_heads"] * rng.choice((1, 2, 3, 4, 8, 16)),
            "count": max(2, _log_int(rng, 1, max(2, blocks)))}


# ------------------------------------------------------------------------------- inputs


def _bytes_of(name):
    return {"int8": 1, "bfloat16": 2, "float32": 4}[name]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 7919 + 31)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _even(batch, lo, hi):
    """Whole numbers spread evenly over [lo, hi]."""
    return torch.linspace(lo, hi, batch, dtype=torch.float64).round().long()


def _codes(x):
    """Rows as int8 codes and their scales, max|x| / 127."""
    scale = x.abs().amax(-1).clamp_min(1e-8) / x.new_full((), 127.0)
    return (x / scale[..., None]).round().clamp_(-127, 127).to(torch.int8), scale


def _pool(g, case, pages):
    """(pages, kv heads, page, dim) rows and, for int8, their scales.  What stands close together is alike: the rows of
    a page have a part in common."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = _randn(g, *shape) + _randn(g, *shape[:2], 1, shape[3])
    if case["pool"] == "int8":
        return _codes(x)
    return x.to(getattr(torch, case["pool"])), None


def _values(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "rope":
        return _prepare_rope(case, g, s)
    if case["kind"] == "copy":
        n = case["pages"]
        pages = 2 * n + 3
        order = torch.randperm(pages, generator=g, device="cuda").int()
        s["src"], s["dst"] = order[:n].clone(), order[n:2 * n].clone()
    else:
        batch, page = case["batch"], case["page"]
        s["lengths"] = _even(batch, case["lo"], case["hi"]).cuda()[torch.randperm(batch, generator=g, device="cuda")]
        width = max(1, -(-case["hi"] // page))
        pages = batch * width + 3  # a few that belong to nobody
        # the pages of a sequence lie anywhere in the pool
        s["table"] = torch.randperm(pages, generator=g, device="cuda")[:batch * width].reshape(batch, width).int()
    s["k"], s["k_scale"] = _pool(g, case, pages)
    s["v"], s["v_scale"] = _pool(g, case, pages)
    slots = (pages, case["kv_heads"], case["page"])
    if case.get("tracked"):
        s["weight"] = torch.exp(_randn(g, *slots, std=2.0))
        s["position"] = torch.randint(0, 1 << 20, slots, generator=g, device="cuda", dtype=torch.int32)
    if case["kind"] != "copy":
        exact_type = torch.float32 if case["pool"] == "int8" else s["k"].dtype
        rows = _values(s["k"], s["k_scale"])
        s["bounds"] = torch.stack([rows.amax(2), rows.amin(2)], 2).to(exact_type)
        if case["kind"] == "bounds":
            s["bounds"].zero_()
            s["since"] = (s["lengths"] - case["new"]).clamp_min(0) if case["new"] else None
        else:
            x = torch.bfloat16 if case["pool"] == "int8" else s["k"].dtype
            s["q"] = _randn(g, batch, case["heads"], case["dim"]).to(x)
    if own:
        _use_package()
        from cortex.kernels.paged_kv import KVPages

        s["pages"] = KVPages(s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], weight=s.get("weight"),
                             position=s.get("position"), bounds=s.get("bounds"))
    return s


def _prepare_rope(case, g, s):
    n, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    joint = _randn(g, n, h + 2 * kv, d).to(dtype)  # a projection to queries, keys and values
    s["q"], s["k"] = joint[:, :h], joint[:, h:h + kv]
    pairs, axes = case["rotary"] // 2, case["axes"]
    s["positions"] = torch.randint(0, case["far"], (n, axes), generator=g, device="cuda")
    s["inv_freq"] = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    s["inv_freq"] = s["inv_freq"].float()
    # neighbouring pairs turn with the same axis, the first with the first
    s["axes"] = (torch.arange(pairs, device="cuda") * axes // pairs).int() if axes > 1 else None
    if axes == 1:
        s["positions"] = s["positions"][:, 0].contiguous()
    if case["norm"]:
        s["q_gain"], s["k_gain"] = ((1.0 + _randn(g, d, std=0.2)).to(dtype) for _ in range(2))
    if own:
        _use_package()
    return s


def _use_package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)


# ------------------------------------------------------------------------------- one pass


def run(state):
    return {"rope": _rope, "copy": _copy, "bounds": _bounds, "select": _select, "sparse": _sparse}[
        state["case"]["kind"]](state)


def _rope(s):
    case = s["case"]
    eps = 1e-6 if case["norm"] else None
    if own:
        from cortex.kernels.rotary import qk_norm_rope

        return qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], axes=s["axes"],
                            interleaved=case["interleaved"], eps=eps, q_gain=s.get("q_gain"), k_gain=s.get("k_gain"))
    pairs = case["rotary"] // 2
    at = s["positions"][:, None].expand(-1, pairs) if s["axes"] is None else s["positions"][:, s["axes"].long()]
    angle = at.double() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for name in ("q", "k"):
        x = s[name].float()
        if eps is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * s[name + "_gain"].float()
        if case["interleaved"]:
            a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :pairs], x[..., pairs:2 * pairs]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, x[..., 2 * pairs:]], -1).to(s[name].dtype))
    return out


def _copy(s):
    names = ["k", "v"] + [n for n in ("weight", "position") if n in s]
    if own:
        from cortex.kernels.paged_kv import kv_copy_pages

        kv_copy_pages(s["pages"], s["src"], s["dst"])
    else:
        src, dst = s["src"].long(), s["dst"].long()
        for n in names:
            s[n][dst] = s[n][src]
    return [s[n] for n in names]


def _bounds(s):
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import kv_block_bounds

        kv_block_bounds(s["pages"], s["table"], s["lengths"], since=s["since"], max_new=case["new"] or None)
        return [s["bounds"]]
    page = case["page"]
    if case["new"]:  # one block a sequence
        blocks = ((s["lengths"] - 1).clamp_min(0) // page)[:, None]
    else:
        blocks = torch.arange(s["table"].shape[1], device="cuda")[None].expand(case["batch"], -1)
    used = s["lengths"][:, None] - blocks * page
    b, i = (used > 0).nonzero(as_tuple=True)
    at = s["table"][b, blocks[b, i]].long()
    rows = _values(s["k"][at], None if s["k_scale"] is None else s["k_scale"][at])
    there = (torch.arange(page, device="cuda") < used[b, i][:, None])[:, None, :, None]
    most = rows.masked_fill(~there, float("-inf")).amax(2)
    least = rows.masked_fill(~there, float("inf")).amin(2)
    s["bounds"][at] = torch.stack([most, least], 2).to(s["bounds"].dtype)
    return [s["bounds"]]


_FIRST, _RECENT = 1, 1  # blocks that are always selected


def _select(s):
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import paged_block_select

        return list(paged_block_select(s["q"], s["pages"], s["table"], s["lengths"], case["count"], first=_FIRST,
                                       recent=_RECENT))
    batch, kv, d, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    width = s["table"].shape[1]
    keep = min(case["count"], width)
    rows = s["bounds"][s["table"].long()].double().reshape(batch, width, kv, 2 * d)  # 64 bits: ranks near a border
    q = s["q"].double().reshape(batch, kv, -1, d)
    q = torch.cat([q.clamp_min(0.0), q.clamp_max(0.0)], -1).transpose(-1, -2).contiguous()
    score = torch.matmul(rows.transpose(1, 2).contiguous(), q).amax(-1).float()  # (batch, kv heads, blocks)
    blocks = (s["lengths"] + page - 1) // page
    at, n = torch.arange(width, device="cuda"), blocks[:, None, None]
    score = score.masked_fill((at < _FIRST) | (at >= n - _RECENT), float("inf")).masked_fill(at >= n, float("-inf"))
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :keep]  # ties: the lower block first
    best = best.masked_fill(torch.arange(keep, device="cuda") >= n, width).sort(dim=-1).values
    pages = torch.cat([s["table"], s["table"].new_full((batch, 1), -1)], 1)
    table = pages[:, None].expand(-1, kv, -1).gather(2, best)
    kept = blocks.clamp_max(keep)
    lengths = (kept - 1).clamp_min(0) * page + s["lengths"] - (blocks - 1).clamp_min(0) * page
    return [table, lengths]


def _sparse(s):
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import paged_attention

        table, lengths = _select(s)
        return [table, lengths, paged_attention(s["q"], s["pages"], table, lengths)]
    table, lengths = _select(s)
    batch, kv, d = case["batch"], case["kv_heads"], case["dim"]
    at = table.long().clamp_min(0), torch.arange(kv, device="cuda")[:, None]
    k, v = (_values(s[n][at], None if s[n + "_scale"] is None else s[n + "_scale"][at]).reshape(batch, kv, -1, d)
            for n in ("k", "v"))
    q = (s["q"].float() * d ** -0.5).reshape(batch, kv, -1, d).transpose(-1, -2).contiguous()
    x = torch.matmul(k, q)  # (batch, kv heads, slots, group)
    there = (torch.arange(k.shape[2], device="cuda") < lengths[:, None])[:, None, :, None]
    x = x.masked_fill(~there, float("-inf"))
    p = torch.exp(x - x.amax(2, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(2, keepdim=True).clamp_min(1e-38)  # (no key: all of it 0)
    out = torch.matmul(p.transpose(-1, -2).contiguous(), v.masked_fill(~there, 0.0))
    return [table, lengths, out.reshape(s["q"].shape).to(s["q"].dtype)]


# ------------------------------------------------------------------------------- what a pass needs


def work(case):
    """Each input once and each output once."""
    kind, kv, d = case["kind"], case["kv_heads"], case["dim"]
    if kind == "rope":
        values = case["tokens"] * (case["heads"] + kv) * d
        return {"bytes": values * 2 * _bytes_of(case["dtype"]) + case["tokens"] * case["axes"] * 8,
                "flops": values * (4.0 if case["norm"] else 0.0) + values * 3.0 * case["rotary"] / d}
    es, page = _bytes_of(case["pool"]), case["page"]
    row = d * es + (4 if case["pool"] == "int8" else 0)
    if kind == "copy":
        return {"bytes": 2 * case["pages"] * kv * page * (2 * row + (8 if case["tracked"] else 0)) + 8 * case["pages"],
                "flops": float(case["pages"])}
    bound = 2 * d * (4 if case["pool"] == "int8" else es)  # bytes of a block's bounds
    lengths = _even(case["batch"], case["lo"], case["hi"]).tolist()
    if kind == "bounds":
        if case["new"]:  # the block that the last token is in
            rows, blocks = sum((n - 1) % page + 1 for n in lengths if n), sum(1 for n in lengths if n)
        else:
            rows, blocks = sum(lengths), sum(-(-n // page) for n in lengths)
        return {"bytes": kv * (rows * row + blocks * bound) + 12 * case["batch"], "flops": 2.0 * kv * rows * d + 1}
    scored = kept = seen = 0
    for n in lengths:
        blocks = -(-n // page)
        scored += blocks if blocks > case["count"] else 0
        kept += min(blocks, case["count"])
        seen += n - (blocks - min(blocks, case["count"])) * page
    q = case["batch"] * case["heads"] * d * (2 if case["pool"] == "int8" else es)
    need = {"bytes": kv * (scored * bound + kept * 4) + q + 16 * case["batch"],
            "flops": 4.0 * scored * case["heads"] * d + 1}
    if kind == "sparse":
        need["bytes"] += kv * seen * 2 * row + q
        need["flops"] += 4.0 * seen * case["heads"] * d
    return need


# ------------------------------------------------------------------------------- results in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    if case["kind"] == "copy":
        out = []
        for name in ("k", "v", "weight", "position"):
            if name in s:
                for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                    s[name][b] = s[name][a]
                out.append(s[name] if name == "position" else s[name].double())
        return out
    page, kv, lengths = case["page"], case["kv_heads"], s["lengths"].tolist()
    if case["kind"] == "bounds":
        out = s["bounds"].double()
        for b, n in enumerate(lengths):
            begin = max(0, n - case["new"]) // page if case["new"] else 0
            for i in range(begin, -(-n // page)):
                p = int(s["table"][b, i])
                rows = s["k"][p, :, :min(page, n - i * page)].double()
                if s["k_scale"] is not None:
                    rows = rows * s["k_scale"][p, :, :rows.shape[1], None].double()
                out[p, :, 0], out[p, :, 1] = rows.max(1).values, rows.min(1).values
        return [out]
    group, d, width = case["heads"] // kv, case["dim"], s["table"].shape[1]
    table = torch.full((case["batch"], kv, min(case["count"], width)), -1, dtype=torch.int32, device="cuda")
    left, out = [], torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        blocks = -(-n // page)
        kept = min(blocks, case["count"])
        left.append(n - (blocks - kept) * page)
        if n == 0:
            continue
        pages = s["table"][b, :blocks].long()
        for h in range(kv):
            best = torch.full((blocks,), float("-inf"), dtype=torch.float64, device="cuda")
            for i in range(h * group, (h + 1) * group):
                q = s["q"][b, i].double()
                best = torch.maximum(best, (s["bounds"][pages, h].double() * q).amax(1).sum(-1))
            best = best.float().cpu()
            rank = sorted(range(blocks), key=lambda i: (i >= _FIRST and i < blocks - _RECENT, -float(best[i]), i))
            chosen = pages[torch.tensor(sorted(rank[:kept]), device="cuda")]
            table[b, h, :kept] = chosen.int()
            if case["kind"] == "select":
                continue
            k, v = (s[name][chosen, h].double() for name in ("k", "v"))
            if case["pool"] == "int8":
                k, v = (x * s[name][chosen, h].double()[..., None] for x, name in ((k, "k_scale"), (v, "v_scale")))
            k, v = (x.reshape(-1, d)[:left[-1]] for x in (k, v))
            x = s["q"][b, h * group:(h + 1) * group].double() @ k.t().contiguous() / math.sqrt(d)
            out[b, h * group:(h + 1) * group] = torch.softmax(x, -1) @ v
    first = [table, torch.tensor(left, device="cuda")]
    return first + [out] if case["kind"] == "sparse" else first


def _exact_rope(case, s):
    pairs, out = case["rotary"] // 2, []
    pos = s["positions"].double().reshape(case["tokens"], -1)
    axis = [0] * pairs if s["axes"] is None else s["axes"].tolist()
    for name in ("q", "k"):
        x = s[name].double()
        if case["norm"]:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s[name + "_gain"].double()
        y = x.clone()
        for p in range(pairs):
            i, j = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + pairs)
            turn = torch.polar(torch.ones_like(pos[:, 0]), pos[:, axis[p]] * s["inv_freq"][p].double())
            z = torch.complex(x[..., i], x[..., j]) * turn[:, None]
            y[..., i], y[..., j] = z.real, z.imag
        out.append(y)
    return out
