"""The operators of the paged key-value cache, as cases to be timed and compared.

A decoder that serves many sequences keeps their keys and values in a pool of pages:
``k_pages`` and ``v_pages`` [P, KV, page, hd], entry i of sequence b in page
``table[b, i // page]`` at row ``i % page``. Beside them go, per entry and key head, the
accumulated attention weight ``mass`` [P, KV, page] (32-bit float) and the token's position
``pos`` [P, KV, page] (32-bit integer). Five operators work on it:

    append   the new tokens' keys and values into the pages; their mass 0, their positions
    attend   one new token per sequence over its whole cache (or its window and sinks),
             optionally adding every entry's attention weight to its mass
    observe  the attention weights of a prompt's last queries, summed into the mass
    select   which entries leave when a sequence is over its budget: the lightest, outside
             the first tokens and the most recent ones; as moves of the kept entries past
             the budget into the places that become free
    move     those moves

``run`` computes them in plain torch operations when ``own`` is false and calls
``pseudobrain_b200.paged_cache`` when it is true; ``exact`` computes them from their
definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a chat turn just begun: one sequence, a few hundred tokens; latency is all that counts
        {"name": "attend one short", "op": "attend", "batch": 1, "length": 517, "ragged": 0, "heads": 32, "kv": 8,
         "hd": 128, "page": 16, "dtype": "bf16", "window": 0, "sinks": 0, "weights": False},
        # a server's batch in full swing: ragged lengths, weights kept for the eviction
        {"name": "attend ragged batch", "op": "attend", "batch": 64, "length": 8191, "ragged": 1, "heads": 32,
         "kv": 8, "hd": 128, "page": 16, "dtype": "bf16", "window": 0, "sinks": 0, "weights": True},
        # one document of a million tokens, the cache of the benchmark's retrieval workload attended whole
        {"name": "attend one long", "op": "attend", "batch": 1, "length": 1048576, "ragged": 0, "heads": 32, "kv": 8,
         "hd": 128, "page": 16, "dtype": "bf16", "window": 0, "sinks": 0, "weights": False},
        # the hybrid model's 24 query and 4 key heads of 256 with its window of 4096 and 4 sinks
        {"name": "attend window", "op": "attend", "batch": 24, "length": 20011, "ragged": 1, "heads": 24, "kv": 4,
         "hd": 256, "page": 64, "dtype": "fp16", "window": 4096, "sinks": 4, "weights": False},
        # a bounded cache of 4096 entries in steady state, every weight kept
        {"name": "attend bounded", "op": "attend", "batch": 8, "length": 4107, "ragged": 0, "heads": 24, "kv": 4,
         "hd": 256, "page": 16, "dtype": "bf16", "window": 0, "sinks": 0, "weights": True},
        # the end of a short prompt: its last 16 queries, heads of 64 without sharing
        {"name": "observe short", "op": "observe", "batch": 2, "length": 1003, "ragged": 0, "heads": 12, "kv": 12,
         "hd": 64, "page": 16, "dtype": "fp16", "queries": 16},
        # the end of a long prompt: its last 32 queries over 131072 entries
        {"name": "observe long", "op": "observe", "batch": 1, "length": 131072, "ragged": 0, "heads": 32, "kv": 8,
         "hd": 128, "page": 16, "dtype": "bf16", "queries": 32},
        # one token for each of 64 sequences
        {"name": "append tokens", "op": "append", "batch": 64, "length": 4096, "ragged": 1, "tokens": 1, "kv": 8,
         "hd": 128, "page": 16, "dtype": "bf16"},
        # prompts of up to 16384 tokens put into the cache
        {"name": "append prompts", "op": "append", "batch": 6, "length": 77, "ragged": 1, "tokens": 16384, "kv": 8,
         "hd": 128, "page": 16, "dtype": "bf16"},
        # a prompt of 131072 entries cut down to 4096
        {"name": "select after prompt", "op": "select", "batch": 1, "length": 131072, "ragged": 0, "kv": 8,
         "page": 16, "budget": 4096, "recent": 512, "sinks": 4},
        # a batch in steady state: every 16 tokens, 16 entries go
        {"name": "select steady", "op": "select", "batch": 64, "length": 4112, "ragged": 0, "kv": 8, "page": 16,
         "budget": 4096, "recent": 256, "sinks": 4},
        # the moves of a batch of prompts cut down to 4096 entries each
        {"name": "move after prompts", "op": "move", "batch": 8, "length": 16384, "ragged": 1, "kv": 8, "hd": 128,
         "page": 16, "dtype": "bf16", "budget": 4096},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "observe", "append", "select", "move"])
    top = max(work(c)["bytes"] for c in listed())
    while True:
        case = {"op": op, "batch": _spread(rng, 1, 128), "length": _spread(rng, 1, 200000), "ragged": rng.choice([0, 1]),
                "page": rng.choice([8, 16, 32, 64, 128])}
        kv, groups = rng.choice([(1, 8), (1, 24), (2, 5), (4, 6), (4, 8), (8, 4), (8, 1), (3, 2), (12, 1), (16, 2)])
        case["kv"] = kv
        if op != "select":
            case["hd"] = rng.choice([64, 128, 256])
            case["dtype"] = rng.choice(["bf16", "fp16"])
        if op == "attend":
            case.update(heads=kv * groups, window=rng.choice([0, 0, _spread(rng, 1, 8192)]),
                        weights=rng.choice([False, True]))
            case["sinks"] = rng.choice([0, 1, 4, 64]) if case["window"] else 0
        elif op == "observe":
            case.update(heads=kv * groups, queries=_spread(rng, 1, 64))
        elif op == "append":
            case["tokens"] = _spread(rng, 1, 16384)
            case["length"] = _spread(rng, 1, 4096)
        else:
            case["budget"] = _spread(rng, 16, 16384)
            if op == "select":
                case["sinks"] = rng.choice([0, 1, 4])
                case["recent"] = _spread(rng, 1, max(1, case["budget"] // 2))
        pool = case["batch"] * (case["length"] + case.get("tokens", 0)) * kv * case.get("hd", 4)
        scores = case["batch"] * case["length"] * case.get("heads", 0) * case.get("queries", 1)
        if op in ("select", "move") and case["length"] < case["budget"] + 2:
            continue  # nothing leaves
        if work(case)["bytes"] <= top / 4 and pool <= 2 ** 29 and scores <= 2 ** 29:
            return case


# ---------------------------------------------------------------- sizes that follow from a case
def _lengths(case):
    """Entries per sequence: all alike, or spread from 0 to ``length`` with the longest first."""
    n, b = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    r = random.Random(n * 131 + b)
    out = [n] + [r.randint(1, n) for _ in range(b - 1)]
    if b > 4:
        out[2], out[3] = 1, 0
    return out


def _counts(case):
    """New tokens per sequence of an append."""
    n, b = case["tokens"], case["batch"]
    if n == 1 or not case["ragged"]:
        return [n] * b
    r = random.Random(n * 137 + b)
    return [n] + [r.randint(0, n) for _ in range(b - 1)]


def _pages(case):
    """Pages per sequence in the table."""
    most = max(_lengths(case)) + (max(_counts(case)) if case["op"] == "append" else 0)
    return max(1, -(-most // case["page"]))


def _moves(case):
    """Moves per sequence and key head of a move: half the entries that stay were past the budget."""
    return [max(0, min(case["budget"], n - case["budget"]) // 2) for n in _lengths(case)]


def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    lens, kv, op = _lengths(case), case["kv"], case["op"]
    b, hd = case["batch"], case.get("hd", 0)
    row = hd * 2
    if op == "attend":
        if case["window"]:
            seen = sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) for n in lens)
        else:
            seen = sum(lens)
        bytes_ = seen * kv * 2 * row + 2 * b * case["heads"] * row + 4 * b * case["heads"]
        if case["weights"]:
            bytes_ += 8 * seen * kv
        return {"bytes": bytes_, "flops": 4 * seen * case["heads"] * hd}
    if op == "observe":
        w = case["queries"]
        return {"bytes": sum(lens) * kv * (row + 8) + b * w * case["heads"] * row,
                "flops": sum(2 * n * case["heads"] * min(w, n) * hd for n in lens)}
    if op == "append":
        n = sum(_counts(case))
        return {"bytes": n * kv * (4 * row + 8), "flops": 0}
    if op == "select":
        cap = _pages(case) * case["page"]
        m = max(0, min(case["budget"], cap - case["budget"]))
        over = sum(n for n in lens if n > case["budget"])
        return {"bytes": over * kv * 8 + b * kv * (8 * m + 4), "flops": over * kv}
    n = sum(_moves(case)) * kv
    return {"bytes": n * (4 * row + 16 + 8), "flops": 0}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, b, kv, page, m = case["op"], case["batch"], case["kv"], case["page"], _pages(case)
    lens = _lengths(case)
    pool = b * m
    s = {"case": case}
    # pages are handed out as they come free: the table is a permutation of the pool
    s["table"] = torch.randperm(pool, generator=g, device=dev).to(torch.int32).view(b, m)
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["seen"] = s["lengths"].clone()  # tokens seen so far
    if op != "select":
        dt, hd = DTYPES[case["dtype"]], case["hd"]
        s["k_pages"] = torch.randn(pool, kv, page, hd, generator=g, device=dev, dtype=dt)
        s["v_pages"] = torch.randn(pool, kv, page, hd, generator=g, device=dev, dtype=dt)
    # a cache's accumulated weights are few large ones among many small ones
    if op in ("select", "move", "append") or case.get("weights") or op == "observe":
        u = torch.rand(pool, kv, page, generator=g, device=dev)
        s["mass"] = u.pow(8) * 0.01 if op in ("attend", "observe") else u.pow(8) * 50
    if op in ("append", "select", "move"):
        s["pos"] = torch.zeros(pool, kv, page, dtype=torch.int32, device=dev)
        # the entries of a cache that has evicted before lie in any order
        x = torch.rand(b, kv, m * page, generator=g, device=dev)
        x = torch.where(torch.arange(m * page, device=dev) < s["lengths"][:, None, None], x, 2.0)
        rank = x.argsort(dim=-1, stable=True).argsort(dim=-1).to(torch.int32)
        s["pos"][s["table"].long()] = rank.view(b, kv, m, page).transpose(1, 2)
    if op == "attend":
        s["q"] = torch.randn(b, case["heads"], hd, generator=g, device=dev, dtype=dt) * 2
    elif op == "observe":
        s["q"] = torch.randn(b, case["queries"], case["heads"], hd, generator=g, device=dev, dtype=dt) * 2
    elif op == "append":
        counts = _counts(case)
        n = sum(counts)
        s["k"] = torch.randn(n, kv, hd, generator=g, device=dev, dtype=dt)
        s["v"] = torch.randn(n, kv, hd, generator=g, device=dev, dtype=dt)
        s["cu_seqlens"] = torch.tensor([sum(counts[:i]) for i in range(b + 1)], dtype=torch.int32, device=dev)
    elif op == "move":
        counts = torch.tensor(_moves(case), dtype=torch.int32, device=dev)
        width = max(_moves(case))
        n = case["budget"]
        s["count"] = counts[:, None].expand(b, kv).contiguous()
        keep = torch.arange(width, device=dev)[None, None, :] < s["count"][..., None]

        def some(low, high):  # `count` ascending places of [low, high) for every row
            room = (high - low).clamp(min=1)
            x = torch.rand(b, kv, width, generator=g, device=dev)
            x = torch.where(keep, x, 2.0).sort(-1).values
            step = torch.arange(width, device=dev)
            free = (room[:, None, None] - s["count"][..., None]).clamp(min=0)
            return torch.where(keep, low[:, None, None] + step + (x * free).long().clamp(max=free), -1).to(torch.int32)

        zero = torch.zeros(b, dtype=torch.long, device=dev)
        s["dst"] = some(zero, zero + n)
        s["src"] = some(zero + n, torch.maximum(s["lengths"].long(), zero + n))
    if own:
        from pseudobrain_b200 import paged_cache as P
        s["cache"] = P.PagedCache(s.get("k_pages"), s.get("v_pages"), s.get("mass"), s.get("pos"))
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend, "observe": _observe, "append": _append, "select": _select,
            "move": _move}[state["case"]["op"]](state)


def _run_own(s):
    from pseudobrain_b200 import paged_cache as P
    c, cache = s["case"], s["cache"]
    if c["op"] == "attend":
        out, lse = P.paged_attend(cache, s["q"], s["table"], s["lengths"], window=c["window"] or None,
                                  sinks=c["sinks"], accumulate=c["weights"])
        return (out, lse, s["mass"]) if c["weights"] else (out, lse)
    if c["op"] == "observe":
        P.paged_observe_(cache, s["q"], s["table"], s["lengths"])
        return s["mass"]
    if c["op"] == "append":
        P.paged_append_(cache, s["k"], s["v"], s["table"], s["lengths"], s["seen"],
                        cu_seqlens=s["cu_seqlens"] if c["tokens"] != 1 else None)
        return s["k_pages"], s["v_pages"], s["mass"], s["pos"]
    if c["op"] == "select":
        return P.select_evictions(cache, s["table"], s["lengths"], s["seen"], c["budget"], recent=c["recent"],
                                  sinks=c["sinks"])
    P.move_entries_(cache, s["table"], s["src"], s["dst"], s["count"])
    return s["k_pages"], s["v_pages"], s["mass"], s["pos"]


def _entries(pages, table):
    """[P, KV, page, ...] through a table [B, M] -> [B, KV, M * page, ...]."""
    x = pages[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], x.shape[2] * x.shape[3], *x.shape[4:])


def _add_entries(pages, table, add):
    """pages [P, KV, page] with add [B, KV, M * page] added through the table."""
    b, m = table.shape
    t = table.long()
    pages[t] = pages[t] + add.view(b, add.shape[1], m, -1).transpose(1, 2)


def _attend(s):
    c, q = s["case"], s["q"]
    b, h, hd = q.shape
    kv = c["kv"]
    k = _entries(s["k_pages"], s["table"]).float()
    at = torch.arange(k.shape[2], device=q.device)[None, :]
    n = s["lengths"].long()[:, None]
    visible = at < n
    if c["window"]:
        visible = visible & ((at >= n - c["window"]) | (at < c["sinks"]))
    visible = visible[:, None, None, :]
    x = (q.float().view(b, kv, h // kv, hd) @ k.transpose(-1, -2)) * hd ** -0.5
    del k
    x = torch.where(visible, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = torch.where(visible[:, :, 0, :, None], _entries(s["v_pages"], s["table"]).float(), 0.0)
    out = (p @ v).view(b, h, hd).to(q.dtype)
    lse = (torch.log(total) + top).view(b, h)
    if not c["weights"]:
        return out, lse
    _add_entries(s["mass"], s["table"], p.sum(2))
    return out, lse, s["mass"]


def _observe(s):
    c, q = s["case"], s["q"]
    b, w, h, hd = q.shape
    kv = c["kv"]
    k = _entries(s["k_pages"], s["table"]).float()
    at = torch.arange(k.shape[2], device=q.device)
    x = q.float().view(b, w, kv, h // kv, hd).permute(0, 2, 3, 1, 4) @ k[:, :, None].transpose(-1, -2)
    x = x * hd ** -0.5
    place = s["lengths"].long()[:, None] - w + torch.arange(w, device=q.device)  # of each query's own entry
    visible = (at[None, None, :] <= place[:, :, None])[:, None, None]
    x = torch.where(visible, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    _add_entries(s["mass"], s["table"], p.sum((2, 3)))
    return s["mass"]


def _append(s):
    starts = s["cu_seqlens"].long()
    n, page = s["k"].shape[0], s["case"]["page"]
    token = torch.arange(n, device=starts.device)
    seq = torch.bucketize(token, starts[1:], right=True)
    i = token - starts[seq]
    e = s["lengths"].long()[seq] + i
    p, r = s["table"].long()[seq, e // page], e % page
    s["k_pages"][p, :, r] = s["k"]
    s["v_pages"][p, :, r] = s["v"]
    s["mass"][p, :, r] = 0.0
    s["pos"][p, :, r] = (s["seen"][seq] + i.to(torch.int32))[:, None]
    return s["k_pages"], s["v_pages"], s["mass"], s["pos"]


def _select(s):
    c = s["case"]
    budget = c["budget"]
    mass, pos = _entries(s["mass"], s["table"]), _entries(s["pos"], s["table"])
    b, kv, cap = mass.shape
    most = max(0, min(budget, cap - budget))
    at = torch.arange(cap, device=mass.device)
    n = s["lengths"].long()[:, None, None]
    safe = ((pos >= 0) & (pos < c["sinks"])) | (pos >= (s["seen"] - c["recent"])[:, None, None])
    weight = torch.where(safe, math.inf, mass)
    weight = torch.where(at < n, weight, -math.inf)
    order = weight.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(b, kv, cap, dtype=torch.bool, device=mass.device)
    kept.scatter_(-1, order[..., :budget], True)
    over = n > budget
    hole = over & (at < budget) & ~kept
    mover = over & (at >= budget) & kept

    def places(mask):
        out = torch.full((b, kv, most + 1), -1, dtype=torch.int32, device=mass.device)
        rank = torch.where(mask, mask.cumsum(-1) - 1, most)
        out.scatter_(-1, rank, torch.where(mask, at, -1).to(torch.int32))
        return out[..., :most].contiguous()

    return places(mover), places(hole), hole.sum(-1).to(torch.int32)


def _move(s):
    c, table = s["case"], s["table"].long()
    b, kv, width = s["src"].shape
    valid = torch.arange(width, device=table.device) < s["count"][..., None]
    seq, head, j = valid.nonzero(as_tuple=True)
    src, dst = s["src"].long()[seq, head, j], s["dst"].long()[seq, head, j]
    page = c["page"]
    a = (table[seq, src // page], head, src % page)
    z = (table[seq, dst // page], head, dst % page)
    s["k_pages"][z] = s["k_pages"][a]
    s["v_pages"][z] = s["v_pages"][a]
    s["mass"][z] = s["mass"][a]
    s["pos"][z] = s["pos"][a]
    return s["k_pages"], s["v_pages"], s["mass"], s["pos"]


# ---------------------------------------------------------------- the definitions, in 64 bits
def _rows(s, pages, i, head, n):
    """Entries 0 .. n - 1 of key head ``head`` of sequence i, in 64 bits."""
    page = pages.shape[2]
    used = s["table"][i, : -(-n // page)].long()
    return pages[used, head].flatten(0, 1)[:n].double()


def exact(case, seed):
    s = prepare(case, seed)
    op, page, kv = case["op"], case["page"], case["kv"]
    lens = _lengths(case)
    if op == "select":
        return None  # whole numbers only
    if op == "append":
        out = [s[k].double() for k in ("k_pages", "v_pages", "mass")]
        for i, n in enumerate(_counts(case)):
            lo = int(s["cu_seqlens"][i])
            e = torch.arange(n, device=out[0].device) + lens[i]
            p, r = s["table"].long()[i, e // page], e % page
            out[0][p, :, r] = s["k"][lo:lo + n].double()
            out[1][p, :, r] = s["v"][lo:lo + n].double()
            out[2][p, :, r] = 0
        return out[0], out[1], out[2], None
    if op == "move":
        out = [s[k].double() for k in ("k_pages", "v_pages", "mass")]
        for i in range(case["batch"]):
            for head in range(kv):
                n = int(s["count"][i, head])
                a, z = s["src"][i, head, :n].long(), s["dst"][i, head, :n].long()
                for x, y in zip(out, ("k_pages", "v_pages", "mass")):
                    x[s["table"].long()[i, z // page], head, z % page] = s[y][
                        s["table"].long()[i, a // page], head, a % page].double()
        return out[0], out[1], out[2], None
    h, hd = case["heads"], case["hd"]
    per = h // kv
    mass = s["mass"].double() if "mass" in s else None
    if op == "attend":
        out = torch.zeros(case["batch"], h, hd, dtype=torch.float64, device="cuda")
        lse = torch.full((case["batch"], h), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        first = case["queries"] if op == "observe" else 1
        first = n - min(first, n)  # the entry of the first query that has one
        for head in range(kv):
            k = _rows(s, s["k_pages"], i, head, n)
            if op == "attend":
                q = s["q"][i, head * per:(head + 1) * per].double()
                see = torch.arange(n, device="cuda")
                see = (see >= n - case["window"]) | (see < case["sinks"]) if case["window"] else see >= 0
                see = see.expand(per, n)
            else:
                q = s["q"][i, first - n:, head * per:(head + 1) * per].double().flatten(0, 1)
                own_place = torch.arange(first, n, device="cuda").repeat_interleave(per)
                see = torch.arange(n, device="cuda")[None, :] <= own_place[:, None]
            x = (q @ k.T / math.sqrt(hd)).masked_fill(~see, -math.inf)
            z = torch.logsumexp(x, -1, keepdim=True)
            p = torch.exp(x - z)
            if op == "attend":
                out[i, head * per:(head + 1) * per] = p @ _rows(s, s["v_pages"], i, head, n)
                lse[i, head * per:(head + 1) * per] = z[:, 0]
            if mass is not None:
                used = s["table"][i, : -(-n // page)].long()
                add = torch.zeros(len(used) * page, dtype=torch.float64, device="cuda")
                add[:n] = p.sum(0)
                mass[used, head] += add.view(-1, page)
    if op == "observe":
        return mass
    return (out, lse, mass) if mass is not None else (out, lse)
