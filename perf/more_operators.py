"""Workloads of packed rows: their rotary positions, attention over whole prompts,
and trees of drafted tokens with the masks that attention over a cache reads.

Each case names an operator and its extents. `run` computes it in its plain
form, elementary torch operations in 32 bits (angles in 64), or, with `own`
set, by the library's operator. `exact` restates the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# Bounds of a drawn attention, at most those of the largest listed one:
# operations, scores that the plain form holds at a time, bytes of padded keys.
_MAX_FLOPS = 300e9
_MAX_SCORES = 500e6
_MAX_KEY_BYTES = 1 << 30


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


def listed():
    return [
        # The tokens of a decode step of 64 requests: one axis, halves.
        {"name": "rotary_tokens", "op": "rotary", "rows": 64, "heads": 32,
         "kv_heads": 8, "d": 128, "sections": "64", "interleaved": False,
         "far": 100000, "fused": True},
        # Frames of a video in one prompt: time, height and width.
        {"name": "rotary_video", "op": "rotary", "rows": 8191, "heads": 32,
         "kv_heads": 8, "d": 128, "sections": "16 24 24",
         "interleaved": False, "far": 4000, "fused": True},
        # The drafted trees of 32 requests, 8 to 64 nodes each.
        {"name": "masks_drafts", "op": "masks", "batch": 32, "new_lo": 8,
         "new_hi": 64, "chunk": 0, "words": 2, "pad": 0, "mix": 1},
        # Wide trees of 48 requests beside a prompt's 500 tokens, a chain.
        {"name": "masks_mixed", "op": "masks", "batch": 48, "new_lo": 1,
         "new_hi": 256, "chunk": 500, "words": 8, "pad": 9, "mix": 2},
        # One short prompt of a small model.
        {"name": "packed_small", "op": "packed", "batch": 1, "heads": 9,
         "kv_heads": 3, "d": 64, "dv": 64, "new_lo": 37, "new_hi": 37,
         "before": 0, "causal": True, "pad": 0, "fused": False, "mix": 3},
        # Texts to be encoded: many short sequences, every token sees all.
        {"name": "packed_texts", "op": "packed", "batch": 48, "heads": 12,
         "kv_heads": 12, "d": 64, "dv": 64, "new_lo": 1, "new_hi": 500,
         "before": 0, "causal": False, "pad": 5, "fused": True, "mix": 4},
        # The prompts of six requests of different lengths.
        {"name": "packed_prompts", "op": "packed", "batch": 6, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "new_lo": 17, "new_hi": 2000,
         "before": 0, "causal": True, "pad": 0, "fused": True, "mix": 5},
        # One long document.
        {"name": "packed_long", "op": "packed", "batch": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "new_lo": 8191, "new_hi": 8191,
         "before": 0, "causal": True, "pad": 0, "fused": False, "mix": 6},
        # A small tree of one request of a small model.
        {"name": "tree_small", "op": "tree", "batch": 1, "heads": 9,
         "kv_heads": 3, "d": 64, "dv": 64, "page": 16, "prefix": 0,
         "cached_lo": 100, "cached_hi": 100, "new_lo": 8, "new_hi": 8,
         "chunk": 0, "words": 1, "pad": 0, "spare": 2, "mix": 7},
        # Trees of up to 32 nodes of 16 requests, lengths far apart.
        {"name": "tree_drafts", "op": "tree", "batch": 16, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 16, "prefix": 0,
         "cached_lo": 100, "cached_hi": 4000, "new_lo": 4, "new_hi": 32,
         "chunk": 0, "words": 1, "pad": 3, "spare": 3, "mix": 8},
        # Trees of 24 requests behind a system prompt, beside a new prompt's
        # 300 tokens; more nodes than one word of a mask holds.
        {"name": "tree_prefix", "op": "tree", "batch": 24, "heads": 24,
         "kv_heads": 8, "d": 96, "dv": 96, "page": 32, "prefix": 2048,
         "cached_lo": 0, "cached_hi": 600, "new_lo": 1, "new_hi": 40,
         "chunk": 300, "words": 2, "pad": 0, "spare": 1, "mix": 9},
        # Trees of 64 nodes over four long conversations.
        {"name": "tree_long", "op": "tree", "batch": 4, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 64, "prefix": 0,
         "cached_lo": 20000, "cached_hi": 32000, "new_lo": 64, "new_hi": 64,
         "chunk": 0, "words": 2, "pad": 0, "spare": 0, "mix": 10},
    ]


# ------------------------------------------------------------------- draws --

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _page(rng):
    return rng.choice((8, 16, 16, 32, 64, 128, 256, rng.randint(5, 200)))


def _draw_rotary(rng):
    d = rng.choice((64, 64, 128, 128, 128, 80, 96, 40, 192, 256))
    half = d // 2 if rng.random() < 0.7 else d // 4
    axes = rng.choice((1, 1, 2, 3, 3, 4))
    cuts = sorted(rng.randint(0, half) for _ in range(axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
    hk = rng.choice((1, 2, 3, 4, 8, 32))
    heads = hk * rng.choice((1, 3, 4, 8)) if hk < 32 else hk
    rows = _log(rng, 1, max(1, 8191 * 40 * 128 // ((heads + hk) * d)))
    return {"op": "rotary", "rows": min(rows, 16384), "heads": heads,
            "kv_heads": hk, "d": d, "sections": " ".join(map(str, sections)),
            "interleaved": rng.random() < 0.4, "far": _log(rng, 10, 1 << 20),
            "fused": rng.random() < 0.5}


def _draw_masks(rng):
    batch = _log(rng, 1, 256)
    hi = _log(rng, 1, max(2, min(512, 12000 // batch)))
    chunk = _log(rng, 64, 1000) if rng.random() < 0.3 else 0
    return {"op": "masks", "batch": batch, "new_lo": rng.choice((0, 1, hi)),
            "new_hi": hi, "chunk": chunk, "words": _up(hi, 32)
            + rng.choice((0, 0, 1)), "pad": rng.choice((0, rng.randint(1, 64))),
            "mix": rng.randrange(1 << 20)}


def _draw_packed(rng):
    while True:
        kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
        d = rng.choice((64, 64, 128, 128, 128, 80, 96, 40, 192, 256))
        hi = _log(rng, 1, 8000)
        behind = rng.random() < 0.25
        case = {
            "op": "packed", "batch": _log(rng, 1, 64),
            "heads": kv_heads * rng.choice((1, 1, 3, 4, 8)),
            "kv_heads": kv_heads, "d": d, "dv": 128 if d == 192 else d,
            "new_lo": rng.choice((0, 1, max(1, hi // 3), hi)), "new_hi": hi,
            "before": _log(rng, 1, 8000) if behind else 0,
            "causal": rng.random() < 0.7,
            "pad": rng.choice((0, rng.randint(1, 16))),
            "fused": rng.random() < 0.5, "mix": rng.randrange(1 << 20)}
        keys, added = _packed_lengths(case)
        if (sum(added) and sum(added) <= 32768 and sum(keys) <= 65536
                and work(case)["flops"] <= _MAX_FLOPS
                and max(a * n for a, n in zip(added, keys)) * case["heads"]
                // kv_heads <= _MAX_SCORES):
            return case


def _draw_tree(rng):
    while True:
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        d = rng.choice((64, 64, 128, 128, 128, 80, 96, 40, 192))
        hi = _log(rng, 1, 128)
        case = {
            "op": "tree", "batch": _log(rng, 1, 64),
            "heads": kv_heads * rng.choice((1, 3, 4, 8)),
            "kv_heads": kv_heads, "d": d, "dv": 128 if d == 192 else d,
            "page": _page(rng),
            "prefix": rng.choice((0, 0, _log(rng, 1, 8192))),
            "cached_lo": rng.choice((0, 1)),
            "cached_hi": _log(rng, 1, 16000),
            "new_lo": rng.choice((0, 1, hi)), "new_hi": hi,
            "chunk": _log(rng, 64, 600) if rng.random() < 0.2 else 0,
            "words": _up(hi, 32), "pad": rng.choice((0, rng.randint(1, 16))),
            "spare": rng.randint(0, 5), "mix": rng.randrange(1 << 20)}
        cached, added = _lengths(case)
        rows, batch = sum(added), case["batch"]
        most = max(c + a for c, a in zip(cached, added))
        if (rows and work(case)["flops"] <= _MAX_FLOPS
                and rows * case["heads"] * case["prefix"] <= _MAX_SCORES
                and batch * max(added) * case["heads"] * most <= _MAX_SCORES
                and batch * most * kv_heads * d * 4 <= _MAX_KEY_BYTES):
            return case


def draw(rng):
    return rng.choice((_draw_rotary, _draw_masks, _draw_packed, _draw_packed,
                       _draw_tree, _draw_tree))(rng)


# ------------------------------------------------------------------ inputs --

def _up(n, size):
    return -(-n // size)


def _lengths(case):
    """Tokens that each request has in its pages and those it adds."""
    rng = random.Random(case["mix"])
    cached = [rng.randint(case.get("cached_lo", 0),
                          max(case.get("cached_lo", 0),
                              case.get("cached_hi", 0)))
              for _ in range(case["batch"])]
    added = [rng.randint(case["new_lo"], case["new_hi"])
             for _ in range(case["batch"])]
    if case["chunk"]:
        added[case["batch"] // 2] = case["chunk"]
    return cached, added


def _packed_lengths(case):
    """Keys and new rows of each sequence."""
    rng = random.Random(case["mix"])
    added = [rng.randint(case["new_lo"], case["new_hi"])
             for _ in range(case["batch"])]
    return [a + rng.randint(0, case["before"]) if case["before"] else a
            for a in added], added


class _Values:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.rng = random.Random(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda",
                           dtype=torch.float32).to(torch.float16)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda",
                              dtype=torch.int32)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, generator=self.g, device="cuda",
                             dtype=torch.int32)

    def parents(self, added, chain):
        """A random tree's parents for each request; request `chain` has a
        prompt, each token behind the one before."""
        out = []
        for b, n in enumerate(added):
            for i in range(n):
                if b == chain:
                    out.append(i - 1)
                else:  # near nodes more often: some depth, some width
                    out.append(i - 1 - self.rng.randrange(min(i + 1, 6)))
        return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(added):
    out = [0]
    for a in added:
        out.append(out[-1] + a)
    return _ints(out)


def _heads_of(v, rows, parts, fused):
    """Rows of several (heads, d) each, beside each other in one projection's
    result or apart."""
    if not fused:
        return [v.normal(rows, h, d) for h, d in parts]
    whole = v.normal(rows, sum(h * d for h, d in parts))
    return [p.unflatten(1, hd) for p, hd in zip(
        whole.split([h * d for h, d in parts], 1), parts)]


def _inputs(case, seed):
    v, op = _Values(seed), case["op"]
    if op == "rotary":
        h, hk, d = (case[n] for n in ("heads", "kv_heads", "d"))
        sections = [int(n) for n in case["sections"].split()]
        half, axes = sum(sections), len(sections)
        q, k = _heads_of(v, case["rows"], ((h, d), (hk, d)), case["fused"])
        f = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        return {"q": q, "k": k, "sections": sections,
                "frequencies": f.float().cuda(),
                "positions": v.below(case["far"], axes, case["rows"])}
    if op == "masks":
        _, added = _lengths(case)
        rows = sum(added) + case["pad"]
        chain = case["batch"] // 2 if case["chunk"] else -1
        return {"rows": rows, "row_starts": _starts(added),
                "parents": _ints(v.parents(added, chain)
                                 + [-1] * case["pad"])}
    h, hk, d, dv = (case[n] for n in ("heads", "kv_heads", "d", "dv"))
    if op == "packed":
        keys, added = _packed_lengths(case)
        rows = sum(added) + case["pad"]
        t = {"rows": rows, "row_starts": _starts(added), "key_starts": None}
        if case["before"]:
            t["key_starts"] = _starts(keys)
            t["q"] = v.normal(rows, h, d)
            t["k"], t["v"] = _heads_of(v, max(1, sum(keys)),
                                       ((hk, d), (hk, dv)), case["fused"])
        else:
            t["q"], t["k"], t["v"] = _heads_of(
                v, rows, ((h, d), (hk, d), (hk, dv)), case["fused"])
        return t
    page = case["page"]
    cached, added = _lengths(case)
    most = max(_up(c + a, page) for c, a in zip(cached, added))
    rows = sum(added) + case["pad"]
    t = {"rows": rows, "width": max(1, most + case["spare"])}
    lead = _up(case["prefix"], page)
    pages = lead + sum(_up(c + a, page) for c, a in zip(cached, added)) + 3
    order = v.order(pages)
    t["prefix_pages"] = order[:lead].clone()
    held = _ints([_up(c + a, page) for c, a in zip(cached, added)])
    columns = torch.arange(t["width"], device="cuda")
    ours = lead + (held.cumsum(0) - held)[:, None] + columns
    t["table"] = torch.where(columns < held[:, None],
                             order[ours.clamp(max=pages - 1)], -1).int()
    t["lengths"] = _ints([c + a for c, a in zip(cached, added)])
    t["row_starts"] = _starts(added)
    t["q"] = v.normal(rows, h, d)
    t["k_cache"] = v.normal(pages, hk, page, d)
    t["v_cache"] = v.normal(pages, hk, page, dv)
    chain = case["batch"] // 2 if case["chunk"] else -1
    # which new tokens each sees, as masks of 32 bits a word
    parents, masks, row = v.parents(added, chain), [], 0
    for a in added:
        seen = []
        for i in range(a):
            up = parents[row + i]
            seen.append((1 << i) | (seen[up] if up >= 0 else 0))
        row += a
        masks += seen
    words = [[_signed(m >> (32 * w)) for w in range(case["words"])]
             for m in masks + [0] * case["pad"]]
    t["masks"] = _ints(words).reshape(rows, case["words"])
    return t


def _signed(word):
    word &= 0xffffffff
    return word - (1 << 32) if word >> 31 else word


def prepare(case, seed):
    t = _inputs(case, seed)
    t["case"] = case
    if case["op"] in ("packed", "tree"):
        t["o"] = torch.zeros(t["rows"], case["heads"], case["dv"],
                             dtype=torch.float16, device="cuda")
    # what a program that packs its batches knows of their extents
    if case["op"] == "packed":
        t["keys"], t["added"] = _packed_lengths(case)
    if case["op"] in ("masks", "tree"):
        cached, added = _lengths(case)
        t["most_new"] = max(added)
        t["most_keys"] = max(c + a for c, a in zip(cached, added))
    return t


# -------------------------------------------------------------- plain form --

def _plain_rotary(t, case):
    half = sum(t["sections"])
    at = torch.repeat_interleave(
        torch.arange(len(t["sections"]), device="cuda"),
        torch.tensor(t["sections"], device="cuda"), output_size=half)
    angle = (t["positions"].double()[at] * t["frequencies"].double()[:, None])
    cos = angle.cos().float().t()[:, None]
    sin = angle.sin().float().t()[:, None]

    def rotated(x):
        out, x = x.float(), x.float()
        if case["interleaved"]:
            x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
            pairs = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
            out = torch.cat([pairs.flatten(-2), x[..., 2 * half:]], -1)
        else:
            x1, x2 = x[..., :half], x[..., half:2 * half]
            out = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin,
                             x[..., 2 * half:]], -1)
        return out.half()

    return {"q": rotated(t["q"]), "k": rotated(t["k"])}


def _plain_masks(t, case):
    rows, bits = t["rows"], 32 * case["words"]
    starts = t["row_starts"].long()
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(starts[1:], r, right=True)
    real = b < case["batch"]
    first = starts[b.clamp(max=case["batch"] - 1)]
    node = r - first
    up = t["parents"].long()
    # the row of each node's parent; `rows`: none
    up = torch.where(real & (up >= 0) & (up < node), first + up, rows)
    up = torch.cat([up, up.new_tensor([rows])])
    seen = torch.zeros(rows + 1, bits, dtype=torch.bool, device="cuda")
    seen[:rows] = (torch.arange(bits, device="cuda") == node[:, None])
    seen[:rows] &= real[:, None]
    depth = (up < rows).long()
    for _ in range(max(1, case["batch"] and t["most_new"]).bit_length()):
        seen |= seen[up]
        depth = depth + depth[up]
        up = up[up]
    weight = 2 ** torch.arange(32, device="cuda")
    words = (seen[:rows].unflatten(1, (-1, 32)) * weight).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words)
    return {"masks": words.int(), "depths": depth[:rows].int()}


def _plain_packed(t, case):
    hk, dv = case["kv_heads"], case["dv"]
    group, row, key = case["heads"] // hk, 0, 0
    for a, n in zip(t["added"], t["keys"]):
        q = t["q"][row:row + a].float().unflatten(1, (hk, group))
        k = t["k"][key:key + n].float()
        v = t["v"][key:key + n].float()
        if a and n:
            i = torch.arange(a, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            hidden = (j > n - a + i) if case["causal"] else None
            # a KV head at a time, or all where they are few scores
            step = hk if a * n * case["heads"] <= _MAX_SCORES else 1
            for g in range(0, hk, step):
                qs = q[:, g:g + step].permute(1, 2, 0, 3).flatten(1, 2)
                ks = k[:, g:g + step].permute(1, 2, 0)
                s = torch.matmul(qs.contiguous() * case["d"] ** -0.5,
                                 ks.contiguous())
                if hidden is not None:
                    s = s.unflatten(1, (group, a))
                    s = s.masked_fill_(hidden, -math.inf).flatten(1, 2)
                s -= s.amax(-1, keepdim=True)
                s.exp_()
                o = torch.matmul(
                    s, v[:, g:g + step].permute(1, 0, 2).contiguous())
                o /= s.sum(-1, keepdim=True)
                o = o.unflatten(1, (group, a)).permute(2, 0, 1, 3)
                t["o"][row:row + a, g * group:(g + step) * group] = (
                    o.reshape(a, -1, dv))
        row, key = row + a, key + n
    return t["o"]


def _part(scores, values):
    """(maximum, sum, weighted values) of the keys of one part."""
    top = scores.amax(-1, keepdim=True)
    weights = (scores - top.clamp(min=-3e38)).exp_()
    return top, weights.sum(-1, keepdim=True), weights @ values


def _plain_tree(t, case):
    page, hk, dv = case["page"], case["kv_heads"], case["dv"]
    group, rows, batch = case["heads"] // hk, t["rows"], case["batch"]
    q = t["q"].float().unflatten(1, (hk, group)) * case["d"] ** -0.5
    # each request's own keys, padded to the longest
    n, keys = t["most_new"], t["most_keys"]
    starts = t["row_starts"].long()
    new = starts[1:] - starts[:-1]
    lengths = t["lengths"].long()
    key = torch.arange(keys, device="cuda")
    at = t["table"][:, key // page].long().clamp(min=0)
    k = t["k_cache"][at, :, key % page].float().permute(0, 2, 3, 1)
    v = t["v_cache"][at, :, key % page].float().permute(0, 2, 1, 3)
    i = torch.arange(n, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=rows - 1)
    qs = q[row].permute(0, 2, 1, 3, 4).flatten(2, 3)  # b, kv head, i * group
    s = torch.matmul(qs, k.contiguous()).unflatten(2, (n, group))
    # request, new token, key: the new token that a key is, and its bit
    node = key - (lengths - new)[:, None]
    word = t["masks"][row]
    bit = (node // 32).clamp(0, case["words"] - 1)
    bit = word.gather(2, bit[:, None].expand(-1, n, -1))
    bit = (bit >> (node % 32)[:, None]) & 1
    sees = (node[:, None] < 0) | ((node[:, None] <= i[:, None]) & (
        (bit == 1) | (node[:, None] >= 32 * case["words"])))
    s.masked_fill_(~sees[:, None, :, None], -math.inf)
    hidden = key >= lengths[:, None]
    v = v.masked_fill(hidden[:, None, :, None], 0.0)
    own_part = _part(s.flatten(2, 3), v)
    # to the packed rows
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(starts[1:], r, right=True).clamp(max=batch - 1)
    at = (r - starts[b]).clamp(0, n - 1)
    top, total, acc = (
        x.unflatten(2, (n, group))[b, :, at] for x in own_part)
    if case["prefix"]:
        key = torch.arange(case["prefix"], device="cuda")
        at = t["prefix_pages"][key // page].long()
        k = t["k_cache"][at, :, key % page].float().permute(1, 2, 0)
        v = t["v_cache"][at, :, key % page].float().permute(1, 0, 2)
        qs = q.permute(1, 0, 2, 3).flatten(1, 2)  # kv head, row * group
        s = torch.matmul(qs, k.contiguous())
        shared = (x.unflatten(1, (rows, group)).transpose(0, 1)
                  for x in _part(s, v.contiguous()))
        top2, total2, acc2 = shared
        both = torch.maximum(top, top2)
        f, f2 = (top - both).exp(), (top2 - both).exp()
        total, acc = total * f + total2 * f2, acc * f + acc2 * f2
    out = torch.where(total > 0, acc / total, 0.0).reshape(rows, -1, dv)
    real = r < starts[-1]
    t["o"].copy_(torch.where(real[:, None, None], out, t["o"]))
    return t["o"]


def run(state):
    t, case, op = state, state["case"], state["case"]["op"]
    if op == "rotary":
        if own:
            q, k = _pkg().rotary(t["q"], t["k"], t["positions"],
                                 t["frequencies"], t["sections"],
                                 interleaved=case["interleaved"])
            return {"q": q, "k": k}
        return _plain_rotary(t, case)
    if op == "masks":
        if own:
            masks, depths = _pkg().tree_masks(t["parents"], t["row_starts"],
                                              case["words"])
            return {"masks": masks, "depths": depths}
        return _plain_masks(t, case)
    if op == "packed":
        if own:
            return _pkg().packed_attention(
                t["q"], t["k"], t["v"], t["row_starts"], t["key_starts"],
                t["o"], causal=case["causal"])
        return _plain_packed(t, case)
    if own:
        return _pkg().tree_attention(
            t["q"], t["k_cache"], t["v_cache"], t["row_starts"],
            t["lengths"], t["table"], t["masks"], t["prefix_pages"],
            case["prefix"], t["o"])
    return _plain_tree(t, case)


def work(case):
    op = case["op"]
    if op == "rotary":
        one = case["rows"] * (case["heads"] + case["kv_heads"]) * case["d"]
        sections = [int(n) for n in case["sections"].split()]
        return {"bytes": 4 * one + 4 * len(sections) * case["rows"]
                + 4 * sum(sections),
                "flops": 6 * one // case["d"] * sum(sections)}
    if op == "masks":
        rows = sum(_lengths(case)[1])
        return {"bytes": 4 * (rows + case["batch"] + 1)
                + 4 * (rows + case["pad"]) * (case["words"] + 1), "flops": 0}
    wide = case["d"] + case["dv"]
    if op == "packed":
        keys, added = _packed_lengths(case)
        seen = sum(a * n - (a * (a - 1) // 2 if case["causal"] else 0)
                   for a, n in zip(added, keys))
        held = sum(n for a, n in zip(added, keys) if a)
        tables = 1 + (1 if case["before"] else 0)
        return {"bytes": 2 * wide * (case["heads"] * sum(added)
                                     + case["kv_heads"] * held)
                + 4 * tables * (case["batch"] + 1),
                "flops": 2 * wide * case["heads"] * seen}
    cached, added = _lengths(case)
    page, batch, rows = case["page"], case["batch"], sum(added)
    held = sum(_up(c + a, page) for c, a in zip(cached, added))
    keys = case["prefix"] + sum(c + a for c, a in zip(cached, added) if a)
    # a row of a tree sees fewer new tokens than those before it: cached ones
    # and itself are counted
    seen = sum(a * (case["prefix"] + c + 1) for c, a in zip(cached, added))
    return {"bytes": 2 * wide * (case["heads"] * rows
                                 + case["kv_heads"] * keys)
            + 4 * (2 * batch + 1 + held + _up(case["prefix"], page)
                   + rows * case["words"]),
            "flops": 2 * wide * case["heads"] * seen}


# ---------------------------------------------------------------- 64 bits --

def _exact_rotary(t, case):
    axis = [a for a, n in enumerate(t["sections"]) for _ in range(n)]
    half, out = len(axis), {}
    for name in ("q", "k"):
        x = t[name].double()
        y = x.clone()
        for i, a in enumerate(axis):
            angle = t["positions"][a].double() * t["frequencies"][i].double()
            turn = torch.polar(torch.ones_like(angle), angle)[:, None]
            at = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
            z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
        out[name] = y
    return out


def _exact_masks(t, case):
    _, added = _lengths(case)
    parents, masks, depths, row = t["parents"].tolist(), [], [], 0
    for a in added:
        for i in range(a):
            bits, depth, at = 1 << i, 0, parents[row + i]
            while at >= 0:
                bits, depth, at = bits | 1 << at, depth + 1, parents[row + at]
            masks.append([_signed(bits >> (32 * w))
                          for w in range(case["words"])])
            depths.append(depth)
        row += a
    masks += [[0] * case["words"]] * case["pad"]
    return {"masks": _ints(masks).reshape(t["rows"], case["words"]),
            "depths": _ints(depths + [0] * case["pad"])}


def _exact_packed(t, case):
    hk, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    keys, added = _packed_lengths(case)
    out = torch.zeros(t["rows"], case["heads"], case["dv"],
                      dtype=torch.float64, device="cuda")
    row = key = 0
    for a, n in zip(added, keys):
        sees = torch.ones(a, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            sees = sees.tril(n - a)
        for h in range(case["heads"] if a and n else 0):
            k = t["k"][key:key + n, h // group].double()
            v = t["v"][key:key + n, h // group].double()
            s = t["q"][row:row + a, h].double() @ k.t() * case["d"] ** -0.5
            s = torch.where(sees, s, -math.inf)
            out[row:row + a, h] = torch.softmax(s, -1) @ v
        row, key = row + a, key + n
    return out


def _exact_tree(t, case):
    page, hk, lead = case["page"], case["kv_heads"], case["prefix"]
    group = case["heads"] // hk
    starts, lengths = t["row_starts"].tolist(), t["lengths"].tolist()

    def rows_of(cache, pages, n, head):
        """The first n tokens' rows of one head, in order."""
        return cache[pages.long(), head].flatten(0, 1)[:n].double()

    out = torch.zeros(t["rows"], case["heads"], case["dv"],
                      dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        first, last, n = starts[b], starts[b + 1], lengths[b]
        a = last - first
        if not a:
            continue
        pages = t["table"][b, :_up(n, page)]
        sees = torch.ones(a, lead + n, dtype=torch.bool, device="cuda")
        tail = torch.ones(a, a, dtype=torch.bool, device="cuda")
        for j in range(min(a, 32 * case["words"])):
            tail[:, j] = (t["masks"][first:last, j // 32] >> (j % 32) & 1) == 1
        sees[:, lead + n - a:] = tail.tril()
        for g in range(hk):
            k = torch.cat([rows_of(t["k_cache"], t["prefix_pages"], lead, g),
                           rows_of(t["k_cache"], pages, n, g)])
            v = torch.cat([rows_of(t["v_cache"], t["prefix_pages"], lead, g),
                           rows_of(t["v_cache"], pages, n, g)])
            for h in range(g * group, (g + 1) * group):
                s = t["q"][first:last, h].double() @ k.t()
                s = (s * case["d"] ** -0.5).masked_fill_(~sees, -math.inf)
                out[first:last, h] = torch.softmax(s, -1) @ v
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    return {"rotary": _exact_rotary, "masks": _exact_masks,
            "packed": _exact_packed, "tree": _exact_tree}[case["op"]](t, case)
