"""What the paged K/V cache operators are measured on, and what their results have to be.

  append      ``paged_kv_append``: the keys and values of new tokens into the pages of their sequences
  attention   ``paged_attention``: one new token a sequence against its cached keys, and with
              ``accumulate`` the softmax weight that each key received
  evict       ``kv_evict_plan`` + ``kv_evict_apply``: the slots worth keeping, moved to the front

``listed`` gives the fixed cases and ``draw`` further ones of the same ranges; ``prepare`` makes what a
program holds before the call, ``run`` is one pass, ``work`` what it cannot do without, ``exact`` its
results in 64 bits.  With ``own`` false ``run`` computes the operators from elementary torch operations.

Slot j of sequence b lives in page ``table[b, j // page]``, row ``j % page``; the pools are
(pages, kv heads, page, head dim).
"""

import os
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "cortex-engine_amd")
_TOKENS = 1 << 17  # cached tokens of the largest cases


def listed():
    return [
        # one token of one stream at the middle configuration's heads: the smallest call, all latency
        {"name": "append_token_b1", "kind": "append", "batch": 1, "lo": 600, "hi": 600, "new_lo": 1, "new_hi": 1,
         "kv_heads": 8, "dim": 64, "page": 16, "pool": "bfloat16", "tracked": False},
        # a decode step of 64 sequences into an int8 cache, its rows quantised on the way
        {"name": "append_tokens_int8_b64", "kind": "append", "batch": 64, "lo": 100, "hi": 1500, "new_lo": 1,
         "new_hi": 1, "kv_heads": 8, "dim": 128, "page": 32, "pool": "int8", "tracked": True},
        # ragged prompts of eight sequences at once, into pages that may be evicted from later
        {"name": "append_prompts_b8", "kind": "append", "batch": 8, "lo": 0, "hi": 37, "new_lo": 200, "new_hi": 4001,
         "kv_heads": 8, "dim": 128, "page": 16, "pool": "bfloat16", "tracked": True},
        # one query against one short stream, a key head for every query head: serving latency
        {"name": "decode_b1_short", "kind": "attention", "batch": 1, "lo": 600, "hi": 600, "heads": 8, "kv_heads": 8,
         "dim": 64, "page": 16, "pool": "bfloat16", "accumulate": False},
        # a serving batch of ragged lengths, four query heads to a key head
        {"name": "decode_b32_ragged", "kind": "attention", "batch": 32, "lo": 150, "hi": 8003, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "pool": "bfloat16", "accumulate": False},
        # one sequence with a very long cache: split over its length
        {"name": "decode_b1_long", "kind": "attention", "batch": 1, "lo": 131072, "hi": 131072, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "pool": "bfloat16", "accumulate": False},
        # int8 pages, eight query heads to a key head
        {"name": "decode_b16_int8", "kind": "attention", "batch": 16, "lo": 1000, "hi": 15001, "heads": 32,
         "kv_heads": 4, "dim": 128, "page": 32, "pool": "int8", "accumulate": False},
        # the fp32 mode at the largest configuration's twelve heads
        {"name": "decode_b8_fp32", "kind": "attention", "batch": 8, "lo": 101, "hi": 2049, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "pool": "float32", "accumulate": False},
        # the step of a cache under a budget: the weight that every key receives is kept
        {"name": "decode_b16_weights", "kind": "attention", "batch": 16, "lo": 2048, "hi": 4160, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "pool": "bfloat16", "accumulate": True},
        # one stream that outgrew its budget by a little
        {"name": "evict_b1", "kind": "evict", "batch": 1, "lo": 640, "hi": 640, "kv_heads": 8, "dim": 64, "page": 16,
         "pool": "bfloat16", "budget": 512, "recent": 128},
        # long prompts cut down to the budget: many rows move
        {"name": "evict_prompts_b32", "kind": "evict", "batch": 32, "lo": 2000, "hi": 9001, "kv_heads": 8, "dim": 128,
         "page": 16, "pool": "bfloat16", "budget": 2048, "recent": 256},
        # the steady state of a batch in fp32: a page's worth over the budget
        {"name": "evict_steady_fp32_b16", "kind": "evict", "batch": 16, "lo": 4112, "hi": 4160, "kv_heads": 12,
         "dim": 64, "page": 64, "pool": "float32", "budget": 4096, "recent": 1024},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "evict"))
    batch = _log_int(rng, 1, 64)
    pool = rng.choice(("bfloat16", "bfloat16", "float32") if kind == "evict" else
                      ("bfloat16", "bfloat16", "int8", "float32"))
    kv = rng.choice((1, 4, 8)) if pool == "float32" else rng.choice((1, 2, 4, 8, 12))
    case = {"kind": kind, "batch": batch, "kv_heads": kv, "dim": rng.choice((32, 64, 96, 128)),
            "page": rng.choice((8, 16, 32, 64, 128)), "pool": pool}
    most = _TOKENS // batch * 8 // (12 if pool != "float32" else 16)
    if kind == "append":
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 32768 // batch))
        lo = rng.randint(0, 500)
        return {**case, "lo": lo, "hi": lo + rng.randint(0, 500), "new_lo": 1 if new == 1 else rng.randint(0, new),
                "new_hi": new, "tracked": rng.random() < 0.5}
    hi = _log_int(rng, 1, min(most, 32768))
    lo = rng.randint(0, hi) if rng.random() < 0.7 else hi
    if kind == "attention":
        group = rng.choice((1, 2, 3, 4, 8, 16))
        return {**case, "lo": lo, "hi": hi, "heads": kv * group, "accumulate": rng.random() < 0.3}
    hi = max(hi, 24)
    budget = rng.randint(8, hi)
    return {**case, "lo": min(lo, hi), "hi": hi, "budget": budget, "recent": rng.randint(0, budget // 2)}


# ------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 7919 + 29)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _spread(g, batch, lo, hi):
    """Whole numbers spread evenly over [lo, hi], in an order of the seed's (their sum is the case's own)."""
    return _even(batch, lo, hi).cuda()[torch.randperm(batch, generator=g, device="cuda")]


def _even(batch, lo, hi):
    return torch.linspace(lo, hi, batch, dtype=torch.float64).round().long()


def _codes(x):
    """Rows as int8 codes and their scales, max|x| / 127."""
    scale = x.abs().amax(-1).clamp_min(1e-8) / x.new_full((), 127.0)
    return (x / scale[..., None]).round().clamp_(-127, 127).to(torch.int8), scale


def _pool(g, case, pages, std):
    """(pages, kv heads, page, dim) rows and, for int8, their scales: every row holds what some token left there."""
    x = _randn(g, pages, case["kv_heads"], case["page"], case["dim"], std=std)
    if case["pool"] == "int8":
        return _codes(x)
    return x.to(getattr(torch, case["pool"])), None


def prepare(case, seed):
    g = _gen(seed)
    batch, page = case["batch"], case["page"]
    lengths = _spread(g, batch, case["lo"], case["hi"])
    room = case["hi"] + case.get("new_hi", 0)
    width = max(1, -(-room // page))
    pages = batch * width + 3  # a few that belong to nobody
    s = {"case": case, "lengths": lengths}
    # the pages of a sequence lie anywhere in the pool
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[:batch * width].reshape(batch, width).int()
    s["k"], s["k_scale"] = _pool(g, case, pages, 1.0)
    s["v"], s["v_scale"] = _pool(g, case, pages, 1.0)
    x = torch.bfloat16 if case["pool"] == "int8" else s["k"].dtype
    slots = (pages, case["kv_heads"], page)
    if case.get("tracked") or case.get("accumulate") or case["kind"] == "evict":
        # heavy-tailed weights, as a few keys draw most of the attention
        s["weight"] = torch.exp(_randn(g, *slots, std=2.0))
        s["position"] = torch.zeros(slots, dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        new = _spread(g, batch, case["new_lo"], case["new_hi"])
        total = int(new.sum())
        s["new_k"] = _randn(g, total, case["kv_heads"], case["dim"]).to(x)
        s["new_v"] = _randn(g, total, case["kv_heads"], case["dim"]).to(x)
        if case["new_hi"] > 1:
            s["offsets"] = torch.cat([new.new_zeros(1), new.cumsum(0)])
    if case["kind"] == "attention":
        s["q"] = _randn(g, batch, case["heads"], case["dim"]).to(x)
    if case["kind"] == "evict":
        # after earlier evictions the slots are in no order: position of every slot of every head
        span = width * page
        j = torch.arange(span, device="cuda")
        key = torch.rand(batch, case["kv_heads"], span, generator=g, device="cuda")
        key = key + (j >= lengths[:, None, None]) * 2.0
        order = key.argsort(-1).int()
        s["position"][s["table"].long().reshape(-1)] = order.reshape(batch, case["kv_heads"], width, page).transpose(
            1, 2).reshape(batch * width, case["kv_heads"], page)
        s["ranked"] = s["weight"].clone(), s["position"].clone()  # what the plan reads: see run()
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from cortex.kernels.paged_kv import KVPages

        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        s["pages"] = KVPages(s["k"], s["v"], **scales, weight=s.get("weight"), position=s.get("position"))
        if "ranked" in s:
            s["ranked_pages"] = KVPages(s["k"], s["v"], **scales, weight=s["ranked"][0], position=s["ranked"][1])
    return s


# ------------------------------------------------------------------------------- one pass


def run(state):
    return {"append": _append, "attention": _attention, "evict": _evict}[state["case"]["kind"]](state)


def _slots(table, page, batch, slot):
    """Page and row of slot numbers of sequences."""
    return table[batch, slot // page].long(), slot % page


def _append(s):
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import paged_kv_append

        lengths = paged_kv_append(s["pages"], s["new_k"], s["new_v"], s["table"], s["lengths"],
                                  offsets=s.get("offsets"))
    else:
        off = s.get("offsets")
        t = torch.arange(s["new_k"].shape[0], device="cuda")
        b = t if off is None else torch.searchsorted(off[1:].contiguous(), t, right=True)
        slot = s["lengths"][b] + (0 if off is None else t - off[b])
        at, row = _slots(s["table"], case["page"], b, slot)
        for name in ("k", "v"):
            x = s["new_" + name]
            if case["pool"] == "int8":
                x, s[name + "_scale"][at, :, row] = _codes(x.float())
            s[name][at, :, row] = x
        if "weight" in s:
            s["weight"][at, :, row] = 0.0
            s["position"][at, :, row] = slot[:, None].int()
        lengths = s["lengths"] + (1 if off is None else off[1:] - off[:-1])
    out = [lengths]
    if case["pool"] == "int8":  # the rows just written, as the values that they stand for
        at, row = _slots(s["table"], case["page"], torch.arange(case["batch"], device="cuda"), s["lengths"]) \
            if case["new_hi"] == 1 else (slice(None), slice(None))
        for name in ("k", "v"):
            out.append(s[name][at, :, row].float() * s[name + "_scale"][at, :, row][..., None])
    else:
        out += [s["k"], s["v"]]
    return out + [s[n] for n in ("weight", "position") if n in s]


def _dense(pool, table):
    """The rows of every sequence in slot order: (batch, kv heads, slots, ...)."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _attention(s):
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import paged_attention

        out = paged_attention(s["q"], s["pages"], s["table"], s["lengths"], accumulate=case["accumulate"])
        return [out, s["weight"]] if case["accumulate"] else [out]
    kv, d = case["kv_heads"], case["dim"]
    k, v = _dense(s["k"], s["table"]).float(), _dense(s["v"], s["table"]).float()
    if case["pool"] == "int8":
        k, v = k * _dense(s["k_scale"], s["table"])[..., None], v * _dense(s["v_scale"], s["table"])[..., None]
    q = s["q"].float().reshape(case["batch"], kv, -1, d) * d ** -0.5
    x = torch.matmul(k, q.transpose(-1, -2).contiguous())  # (batch, kv heads, slots, group)
    there = (torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None])[:, None, :, None]
    x = x.masked_fill(~there, float("-inf"))
    p = torch.exp(x - x.amax(2, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(2, keepdim=True).clamp_min(1e-38)  # (no key: all of it 0)
    out = torch.matmul(p.transpose(-1, -2).contiguous(), v).reshape(s["q"].shape).to(s["q"].dtype)
    if not case["accumulate"]:
        return [out]
    table = s["table"].long()
    add = p.sum(-1).reshape(case["batch"], kv, -1, case["page"]).transpose(1, 2)
    s["weight"][table] += add
    return [out, s["weight"]]


def _evict(s):
    """The weights and positions that the plan ranks by are a copy of the pages' own: the plan of every pass is that
    of a program's one call (its source slots, at or past the budget, are not written, so neither are the rows)."""
    case = s["case"]
    if own:
        from cortex.kernels.paged_kv import kv_evict_apply, kv_evict_plan

        plan = kv_evict_plan(s["ranked_pages"], s["table"], s["lengths"], case["budget"], case["recent"])
        kv_evict_apply(s["pages"], s["table"], plan)
        dst, src, counts, lengths = plan.dst, plan.src, plan.counts, plan.lengths
    else:
        weight, pos = (_dense(x, s["table"]) for x in s["ranked"])
        batch, kv, span = weight.shape
        budget = case["budget"]
        j = torch.arange(span, device="cuda")
        n = s["lengths"][:, None, None]
        there = j < n
        newest = pos.masked_fill(~there, -1).amax(-1, keepdim=True)
        rank = weight.masked_fill(pos > newest - case["recent"], float("inf")).masked_fill(~there, float("-inf"))
        kept = torch.zeros_like(there.expand(batch, kv, span))
        first = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]  # ties: the lowest slot first
        kept.scatter_(-1, first, True)
        over = n > budget
        hole, mover = ~kept & (j < budget) & over, kept & (j >= budget) & over
        cap = max(0, min(budget, span - budget))
        counts = hole.sum(-1).int()
        dst, src = (torch.full((batch, kv, cap + 1), -1, dtype=torch.int32, device="cuda") for _ in range(2))
        for to, which in ((dst, hole), (src, mover)):
            place = torch.where(which, which.cumsum(-1) - 1, cap)  # (what does not move goes to a column that is cut off)
            to.scatter_(-1, place, torch.where(which, j, -1).int())
        dst, src = dst[..., :cap].contiguous(), src[..., :cap].contiguous()
        lengths = s["lengths"].clamp_max(budget)
        b, h, i = (torch.arange(cap, device="cuda") < counts[..., None]).nonzero(as_tuple=True)
        to, to_row = _slots(s["table"], case["page"], b, dst[b, h, i].long())
        at, row = _slots(s["table"], case["page"], b, src[b, h, i].long())
        for name in ("k", "v", "weight", "position"):
            s[name][to, h, to_row] = s[name][at, h, row]
    return [dst, src, counts, lengths, s["k"], s["v"], s["weight"], s["position"]]


# ------------------------------------------------------------------------------- what a pass needs


def _bytes_of(name):
    return {"int8": 1, "bfloat16": 2, "float32": 4}[name]


def work(case):
    """Each input once and each output once.  How many rows an eviction moves goes by chance: with the kept slots
    anywhere among n, budget * (n - budget) / n."""
    batch, kv, d = case["batch"], case["kv_heads"], case["dim"]
    es = _bytes_of(case["pool"])
    row = d * es + (4 if case["pool"] == "int8" else 0)
    x = 2 if case["pool"] == "int8" else es
    total = int(_even(batch, case["lo"], case["hi"]).sum())
    if case["kind"] == "append":
        new = int(_even(batch, case["new_lo"], case["new_hi"]).sum())
        return {"bytes": new * kv * (2 * d * x + 2 * row + (8 if case["tracked"] else 0)) + 20 * batch,
                "flops": 2.0 * new * kv * d}
    if case["kind"] == "attention":
        seen = total * kv * (2 * row + (8 if case["accumulate"] else 0)) + total // case["page"] * 4
        return {"bytes": seen + 2 * batch * case["heads"] * d * x + 8 * batch,
                "flops": 4.0 * total * case["heads"] * d + batch}
    moved, read = 0.0, 0
    for n in _even(batch, case["lo"], case["hi"]).tolist():
        if n > case["budget"]:
            moved += kv * case["budget"] * (n - case["budget"]) / n
            read += n * kv * 8
    return {"bytes": moved * (2 * (2 * row + 8) + 8) + read + 16 * batch, "flops": float(read + batch)}


# ------------------------------------------------------------------------------- results in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    lengths, table = s["lengths"].tolist(), s["table"].long()
    if case["kind"] == "append":
        if case["pool"] == "int8":  # (a code next to a border between two has no value in 64 bits)
            return None
        pools = [s["k"].double(), s["v"].double()]
        weight, position = s.get("weight"), s.get("position")
        ends = s["offsets"].tolist() if "offsets" in s else list(range(case["batch"] + 1))
        for b, n in enumerate(lengths):
            slot = torch.arange(n, n + ends[b + 1] - ends[b], device="cuda")
            at = table[b][slot // page], slice(None), slot % page
            for pool, x in zip(pools, (s["new_k"], s["new_v"])):
                pool[at] = x[ends[b]:ends[b + 1]].double()
            if weight is not None:
                weight[at] = 0.0
                position[at] = slot[:, None].int()
        out = [torch.tensor([n + ends[b + 1] - ends[b] for b, n in enumerate(lengths)]), *pools]
        return out + ([weight.double(), position] if weight is not None else [])
    if case["kind"] == "attention":
        group = case["heads"] // kv
        out = torch.zeros(case["batch"], kv, group, d, dtype=torch.float64, device="cuda")
        weight = s["weight"].double() if case["accumulate"] else None
        for b, n in enumerate(lengths):
            if n == 0:
                continue
            slot = torch.arange(n, device="cuda")
            at = table[b][slot // page], slice(None), slot % page
            k, v = s["k"][at].double(), s["v"][at].double()  # (slots, kv heads, dim)
            if case["pool"] == "int8":
                k, v = k * s["k_scale"][at].double()[..., None], v * s["v_scale"][at].double()[..., None]
            for h in range(kv):
                q = s["q"][b, h * group:(h + 1) * group].double()
                p = torch.softmax((q @ k[:, h].t().contiguous()) / d ** 0.5, -1)
                out[b, h] = p @ v[:, h].contiguous()
                if weight is not None:
                    weight[table[b][slot // page], h, slot % page] += p.sum(0)
        out = out.reshape(case["batch"], case["heads"], d)
        return [out, weight] if case["accumulate"] else [out]
    # eviction moves values and computes none: the places come from a sort on the host
    pools = [s["k"].double(), s["v"].double(), s["weight"].double()]
    for b, n in enumerate(lengths):
        if n <= case["budget"]:
            continue
        slot = torch.arange(n, device="cuda")
        at = table[b][slot // page]
        weight, position = (x[at, :, slot % page].cpu().numpy() for x in s["ranked"])
        for h in range(kv):
            keep = _kept(weight[:, h], position[:, h], case["budget"], case["recent"])
            dst = torch.tensor([i for i in range(case["budget"]) if not keep[i]], dtype=torch.long, device="cuda")
            src = torch.tensor([i for i in range(case["budget"], n) if keep[i]], dtype=torch.long, device="cuda")
            for pool in pools:
                pool[table[b][dst // page], h, dst % page] = pool[table[b][src // page], h, src % page]
    return [None, None, None, None, *pools, None]


def _kept(weight, position, budget, recent):
    import numpy as np

    n = weight.shape[0]
    young = position.astype(np.int64) > int(position.max()) - recent
    order = np.lexsort((np.arange(n), -weight.astype(np.float64), ~young))
    keep = np.zeros(n, dtype=bool)
    keep[order[:budget]] = True
    return keep.tolist()
