"""Workloads of the paged KV cache: its tables, the rows appended to it and the
attention that reads it, over the sizes that a server's steps call them with.

Each case names an operator and its extents. `run` computes it in its plain
form, elementary torch operations in 32 bits, or, with `own` set, by the
library's operator. `exact` restates the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# Bounds of a drawn attention, those of the largest listed one: operations,
# scores that the plain form holds at a time, bytes of its padded keys.
_MAX_FLOPS = 150e9
_MAX_SCORES = 250e6
_MAX_KEY_BYTES = 512 << 20


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


def listed():
    return [
        # One new token of a single request: the smallest step.
        {"name": "tables_one", "op": "tables", "batch": 1, "cached_lo": 1000,
         "cached_hi": 1000, "new_lo": 1, "new_hi": 1, "page": 16, "pad": 0,
         "spare": 100, "mix": 1},
        # A decode step of 256 requests, rows padded to the step's capacity.
        {"name": "tables_tokens", "op": "tables", "batch": 256,
         "cached_lo": 1, "cached_hi": 4000, "new_lo": 1, "new_hi": 1,
         "page": 16, "pad": 44, "spare": 6, "mix": 2},
        # Prompts of 48 new requests, some of them continued.
        {"name": "tables_prompts", "op": "tables", "batch": 48,
         "cached_lo": 0, "cached_hi": 1000, "new_lo": 17, "new_hi": 2000,
         "page": 64, "pad": 0, "spare": 0, "mix": 3},
        # A decode step's rows into pages of [head, token] order.
        {"name": "append_tokens", "op": "append", "rows": 64, "kv_heads": 8,
         "d": 128, "dv": 128, "page": 16, "pages": 2000, "pad": 3,
         "apart": True, "token_major": False},
        # A prompt's rows into pages of [token, head] order.
        {"name": "append_prompt", "op": "append", "rows": 8191,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 16, "pages": 1000,
         "pad": 0, "apart": False, "token_major": True},
        # Four requests of a small model behind a short instruction.
        {"name": "attend_small", "op": "attend", "batch": 4, "heads": 9,
         "kv_heads": 3, "d": 64, "dv": 64, "page": 16, "prefix": 64,
         "cached_lo": 0, "cached_hi": 100, "new_lo": 1, "new_hi": 1,
         "chunk": 0, "pad": 0, "spare": 2, "token_major": False, "mix": 4},
        # One token of 64 requests behind a system prompt, 1 to 1000 tokens
        # into their own text.
        {"name": "attend_tokens", "op": "attend", "batch": 64, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 16, "prefix": 8192,
         "cached_lo": 0, "cached_hi": 1000, "new_lo": 1, "new_hi": 1,
         "chunk": 0, "pad": 0, "spare": 2, "token_major": False, "mix": 5},
        # Questions about one long document: nearly all keys are shared.
        {"name": "attend_document", "op": "attend", "batch": 24, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 64, "prefix": 32749,
         "cached_lo": 3, "cached_hi": 300, "new_lo": 1, "new_hi": 1,
         "chunk": 0, "pad": 8, "spare": 0, "token_major": True, "mix": 6},
        # No shared prefix: a decode step over pages, lengths far apart.
        {"name": "attend_pages", "op": "attend", "batch": 32, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 32, "prefix": 0,
         "cached_lo": 1, "cached_hi": 4000, "new_lo": 1, "new_hi": 1,
         "chunk": 0, "pad": 0, "spare": 3, "token_major": False, "mix": 7},
        # Up to five drafted tokens a request to check at once, one KV head
        # per query head, pages of a size that no tile divides.
        {"name": "attend_drafts", "op": "attend", "batch": 12, "heads": 32,
         "kv_heads": 32, "d": 64, "dv": 64, "page": 24, "prefix": 1001,
         "cached_lo": 10, "cached_hi": 700, "new_lo": 1, "new_hi": 5,
         "chunk": 0, "pad": 5, "spare": 1, "token_major": False, "mix": 8},
        # One request's prompt of 500 tokens beside the tokens of 40 others.
        {"name": "attend_mixed", "op": "attend", "batch": 41, "heads": 24,
         "kv_heads": 3, "d": 96, "dv": 96, "page": 16, "prefix": 777,
         "cached_lo": 0, "cached_hi": 900, "new_lo": 1, "new_hi": 1,
         "chunk": 500, "pad": 0, "spare": 2, "token_major": False, "mix": 9},
        # The prompts of four requests behind the same instruction.
        {"name": "attend_prompts", "op": "attend", "batch": 4, "heads": 32,
         "kv_heads": 8, "d": 128, "dv": 128, "page": 64, "prefix": 4096,
         "cached_lo": 0, "cached_hi": 1500, "new_lo": 400, "new_hi": 700,
         "chunk": 0, "pad": 0, "spare": 1, "token_major": False, "mix": 10},
    ]


# ------------------------------------------------------------------- draws --

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _page(rng):
    return rng.choice((8, 16, 16, 32, 64, 128, 256, rng.randint(5, 200)))


def draw(rng):
    op = rng.choice(("tables", "append", "attend", "attend", "attend"))
    mix = rng.randrange(1 << 20)
    if op == "tables":
        batch = _log(rng, 1, 1024)
        tokens = rng.random() < 0.5
        hi = 1 if tokens else _log(rng, 2, max(2, 48000 // batch))
        cached_hi = _log(rng, 1, 4000)
        return {"op": op, "batch": batch, "cached_lo": rng.choice((0, 1)),
                "cached_hi": cached_hi, "new_lo": rng.choice((0, 1)),
                "new_hi": hi, "page": _page(rng), "spare": rng.randint(0, 50),
                "pad": rng.choice((0, rng.randint(1, 64))), "mix": mix}
    if op == "append":
        d = rng.choice((64, 64, 128, 128, 80, 96, 40, 192, 256))
        heads, rows, page = rng.choice((1, 2, 3, 8, 32)), 0, _page(rng)
        while rows * heads * d not in range(1, 8191 * 8 * 128 + 1):
            rows = _log(rng, 1, 16384)
        return {"op": op, "rows": rows, "kv_heads": heads, "d": d,
                "dv": 128 if d == 192 else d, "page": page,
                "pages": rows // page + rng.randint(1, 1000) // page + 2,
                "pad": rng.choice((0, rng.randint(1, 64))),
                "apart": rows <= 256 and rng.random() < 0.7,
                "token_major": rng.random() < 0.5}
    while True:
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        d = rng.choice((64, 64, 128, 128, 128, 80, 96, 40, 192))
        kind = rng.choice(("tokens", "tokens", "drafts", "mixed", "prompts"))
        case = {
            "op": op,
            "batch": _log(rng, 1, 8 if kind == "prompts" else 128),
            "heads": kv_heads * rng.choice((1, 3, 4, 8)),
            "kv_heads": kv_heads, "d": d, "dv": 128 if d == 192 else d,
            "page": _page(rng),
            "prefix": rng.choice((0, _log(rng, 1, 32768),
                                  _log(rng, 64, 8192))),
            "cached_lo": rng.choice((0, 1)),
            "cached_hi": _log(rng, 1, 4000),
            "new_lo": 1, "new_hi": 1,
            "chunk": _log(rng, 64, 1000) if kind == "mixed" else 0,
            "pad": rng.choice((0, rng.randint(1, 16))),
            "spare": rng.randint(0, 5), "token_major": rng.random() < 0.3,
            "mix": mix}
        if kind == "drafts":
            case["new_lo"], case["new_hi"] = 0, rng.randint(2, 8)
        if kind == "prompts":
            case["new_hi"] = _log(rng, 32, 1500)
            case["new_lo"] = max(1, case["new_hi"] // 3)
        cached, added = _lengths(case)
        rows, batch = sum(added), case["batch"]
        most = max(c + a for c, a in zip(cached, added))
        if (rows and work(case)["flops"] <= _MAX_FLOPS
                and rows * case["heads"] * case["prefix"] <= _MAX_SCORES
                and batch * max(added) * case["heads"] * most <= _MAX_SCORES
                and batch * most * kv_heads * d * 4 <= _MAX_KEY_BYTES):
            return case


# ------------------------------------------------------------------ inputs --

def _lengths(case):
    """Tokens that each request has in its pages and those it adds."""
    rng = random.Random(case["mix"])
    cached = [rng.randint(case["cached_lo"],
                          max(case["cached_lo"], case["cached_hi"]))
              for _ in range(case["batch"])]
    added = [rng.randint(case["new_lo"], case["new_hi"])
             for _ in range(case["batch"])]
    if case.get("chunk"):
        added[case["batch"] // 2] = case["chunk"]
    return cached, added


def _up(n, page):
    return -(-n // page)


class _Values:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda",
                           dtype=torch.float32).to(torch.float16)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda",
                              dtype=torch.int32)

    def cache(self, pages, heads, page, d, token_major):
        """[pages, heads, page, d], in memory [pages, page, heads, d] for
        token_major."""
        if token_major:
            return self.normal(pages, page, heads, d).permute(0, 2, 1, 3)
        return self.normal(pages, heads, page, d)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    v, op, page = _Values(seed), case["op"], case["page"]
    if op == "append":
        rows, h, d, dv = (case[n] for n in ("rows", "kv_heads", "d", "dv"))
        # K and V beside each other in the rows of one projection's result
        kv = v.normal(rows + case["pad"], h * (d + dv))
        if case["apart"]:  # a token of each of many requests
            slots = v.order(case["pages"] * page)[:rows]
        else:              # prompts: page after page
            slots = v.order(case["pages"])[:, None] * page
            slots = slots + torch.arange(page, device="cuda")
            slots = slots.flatten()[page // 2:][:rows].int()
        slots = torch.cat([slots, _ints([-1] * case["pad"])])
        return {"k": kv[:, :h * d].unflatten(1, (h, d)),
                "v": kv[:, h * d:].unflatten(1, (h, dv)),
                "k_cache": v.cache(case["pages"], h, page, d,
                                   case["token_major"]),
                "v_cache": v.cache(case["pages"], h, page, dv,
                                   case["token_major"]),
                "slots": slots}
    cached, added = _lengths(case)
    most = max(_up(c + a, page) for c, a in zip(cached, added))
    rows = sum(added) + case["pad"]
    t = {"rows": rows, "width": max(1, most + case["spare"])}
    if op == "tables":
        held = [_up(c, page) for c in cached]
        need = sum(_up(c + a, page) for c, a in zip(cached, added))
        order = v.order(need + 64)
        columns = torch.arange(t["width"], device="cuda")
        first = _ints([0] + held[:-1]).cumsum(0)
        ours = first[:, None] + columns
        t["table"] = torch.where(columns < _ints(held)[:, None],
                                 order[ours.clamp(max=need)], -1).int()
        t["free"] = order[sum(held):].clone()
        t["cached"], t["added"] = _ints(cached), _ints(added)
        return t
    h, hk, d, dv = (case[n] for n in ("heads", "kv_heads", "d", "dv"))
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
    t["row_starts"] = _ints([0] + added).cumsum(0).int()
    t["q"] = v.normal(rows, h, d)
    t["k_cache"] = v.cache(pages, hk, page, d, case["token_major"])
    t["v_cache"] = v.cache(pages, hk, page, dv, case["token_major"])
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    t["case"] = case
    if case["op"] == "attend":
        t["o"] = torch.zeros(t["rows"], case["heads"], case["dv"],
                             dtype=torch.float16, device="cuda")
        # what a program that pads its batches knows of their extents
        cached, added = _lengths(case)
        t["most_new"] = max(added)
        t["most_keys"] = max(c + a for c, a in zip(cached, added))
    return t


# -------------------------------------------------------------- plain form --

def _plain_tables(t, case):
    page, table, free = case["page"], t["table"], t["free"]
    cached, added = t["cached"].long(), t["added"].long()
    lengths = cached + added
    held = (cached + page - 1) // page
    take = (lengths + page - 1) // page - held
    first = take.cumsum(0) - take
    ends = added.cumsum(0)
    starts = ends - added
    column = torch.arange(table.shape[1], device="cuda")
    nth = column - held[:, None]
    at = first[:, None] + nth
    page_at = torch.where(at < free.numel(),
                          free[at.clamp(0, free.numel() - 1)], -1)
    fresh = (nth >= 0) & (nth < take[:, None])
    table.copy_(torch.where(fresh, page_at, table))
    row = torch.arange(t["rows"], device="cuda")
    b = torch.searchsorted(ends, row, right=True).clamp(max=len(added) - 1)
    at = cached[b] + row - starts[b]
    column = at // page
    named = table[b, column.clamp(0, table.shape[1] - 1)]
    real = (row < ends[-1]) & (column < table.shape[1]) & (named >= 0)
    slots = torch.where(real, named * page + at % page, -1)
    return {"table": table, "lengths": lengths.int(), "slots": slots.int(),
            "row_starts": torch.cat([starts, ends[-1:]]).int(),
            "needed": take.sum().int().reshape(1)}


def _plain_append(t, case):
    real = t["slots"] >= 0
    slots = t["slots"][real].long()
    at, inside = slots // case["page"], slots % case["page"]
    t["k_cache"][at, :, inside] = t["k"][real]
    t["v_cache"][at, :, inside] = t["v"][real]
    return {"k_cache": t["k_cache"], "v_cache": t["v_cache"]}


def _part(scores, values):
    """(maximum, sum, weighted values) of the keys of one part."""
    top = scores.amax(-1, keepdim=True)
    weights = (scores - top.clamp(min=-3e38)).exp_()
    return top, weights.sum(-1, keepdim=True), weights @ values


def _plain_attend(t, case):
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
    sees = (lengths - new)[:, None] + i + 1
    hidden = key >= sees[..., None]
    s.masked_fill_(hidden[:, None, :, None], -math.inf)
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
    t, case = state, state["case"]
    if case["op"] == "tables":
        if own:
            starts, lengths, slots, needed = _pkg().page_tables(
                t["cached"], t["added"], t["free"], t["table"], case["page"],
                t["rows"])
            return {"table": t["table"], "lengths": lengths, "slots": slots,
                    "row_starts": starts, "needed": needed}
        return _plain_tables(t, case)
    if case["op"] == "append":
        if own:
            _pkg().append_kv(t["k"], t["v"], t["k_cache"], t["v_cache"],
                             t["slots"])
            return {"k_cache": t["k_cache"], "v_cache": t["v_cache"]}
        return _plain_append(t, case)
    if own:
        return _pkg().shared_prefix_attention(
            t["q"], t["k_cache"], t["v_cache"], t["row_starts"],
            t["lengths"], t["table"], t["prefix_pages"], case["prefix"],
            t["o"])
    return _plain_attend(t, case)


def work(case):
    if case["op"] == "append":
        one = case["kv_heads"] * (case["d"] + case["dv"]) * 2
        rows = case["rows"]
        return {"bytes": 2 * rows * one + 4 * (rows + case["pad"]),
                "flops": 0}
    cached, added = _lengths(case)
    page, batch, rows = case["page"], case["batch"], sum(added)
    if case["op"] == "tables":
        fresh = sum(_up(c + a, page) - _up(c, page)
                    for c, a in zip(cached, added))
        return {"bytes": 4 * (4 * batch + 2 + 2 * fresh + rows + case["pad"]),
                "flops": 0}
    wide = case["d"] + case["dv"]
    held = sum(_up(c + a, page) for c, a in zip(cached, added))
    keys = case["prefix"] + sum(c + a for c, a in zip(cached, added) if a)
    seen = sum(a * (case["prefix"] + c) + a * (a + 1) // 2
               for c, a in zip(cached, added))
    return {"bytes": 2 * wide * (case["heads"] * rows
                                 + case["kv_heads"] * keys)
            + 4 * (2 * batch + 1 + held + _up(case["prefix"], page)),
            "flops": 2 * wide * case["heads"] * seen}


# ---------------------------------------------------------------- 64 bits --

def _exact_tables(t, case):
    page, table = case["page"], t["table"].tolist()
    cached, added, free = (t[n].tolist() for n in ("cached", "added", "free"))
    starts, slots, taken = [0], [-1] * t["rows"], 0
    for b, row in enumerate(table):
        n = cached[b] + added[b]
        for column in range(_up(cached[b], page), _up(n, page)):
            row[column] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(cached[b], n):
            slots[starts[b] + p - cached[b]] = (row[p // page] * page
                                                + p % page)
        starts.append(starts[b] + added[b])
    return {"table": _ints(table), "slots": _ints(slots),
            "lengths": _ints([c + a for c, a in zip(cached, added)]),
            "row_starts": _ints(starts), "needed": _ints([taken])}


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "tables":
        return _exact_tables(t, case)
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            flat = t[name + "_cache"].transpose(1, 2).double()
            flat = flat.reshape(-1, *flat.shape[2:])
            for row, slot in enumerate(t["slots"].tolist()):
                if slot >= 0:
                    flat[slot] = t[name][row].double()
            out[name + "_cache"] = flat.unflatten(
                0, (case["pages"], case["page"])).transpose(1, 2)
        return out
    page, hk, lead = case["page"], case["kv_heads"], case["prefix"]
    group = case["heads"] // hk
    starts, lengths = t["row_starts"].tolist(), t["lengths"].tolist()

    def rows_of(cache, pages, n, head):
        """The first n tokens' rows of one head, in order."""
        flat = cache[pages.long(), head].flatten(0, 1)
        return flat[:n].double()

    out = torch.zeros(t["rows"], case["heads"], case["dv"],
                      dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        first, last, n = starts[b], starts[b + 1], lengths[b]
        if first == last:
            continue
        pages = t["table"][b, :_up(n, page)]
        i = torch.arange(last - first, device="cuda")[:, None]
        j = torch.arange(lead + n, device="cuda")
        hidden = j > lead + n - (last - first) + i
        for g in range(hk):
            k = torch.cat([rows_of(t["k_cache"], t["prefix_pages"], lead, g),
                           rows_of(t["k_cache"], pages, n, g)])
            v = torch.cat([rows_of(t["v_cache"], t["prefix_pages"], lead, g),
                           rows_of(t["v_cache"], pages, n, g)])
            for h in range(g * group, (g + 1) * group):
                s = t["q"][first:last, h].double() @ k.t()
                s = s * case["d"] ** -0.5
                s.masked_fill_(hidden, -math.inf)
                out[first:last, h] = torch.softmax(s, -1) @ v
    return out
