"""Cases, plain forms and 64-bit definitions of the serving operators.

Four operators that a decode step needs beside the quantized projections:

  plan       page tables, slots, positions and tree masks of one step, from request lengths
  append     rows of new keys and values written into a paged cache
  attention  attention of a tree of drafted tokens over a paged cache (one token: plain decoding)
  lora       low-rank adapters of many requests added to a shared projection's output

``run`` computes an operator in elementary torch operations in 32 bits (``own`` false) or through
the library's public calls (``own`` true).  ``exact`` computes the same outputs in 64 bits, request
by request, from the definition.
"""

import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _hqb():
    """The library's Python module (imported where its own kernels run)."""
    pkg = str(Path(__file__).resolve().parents[1] / "harp-q_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import harpq_b200

    return harpq_b200


# ---- cases ------------------------------------------------------------------------------


def listed():
    return [
        # 64 requests decode one token each: the call whose latency every step pays
        {"name": "plan 64x1", "op": "plan", "requests": 64, "new": 1, "context": 2048, "page": 16, "tree": False},
        # 512 requests verify drafted trees of up to 64 nodes: slots, tree positions and masks at once
        {"name": "plan 512 trees", "op": "plan", "requests": 512, "new": 64, "context": 4096, "page": 32,
         "tree": True},
        # one decode step of 16 requests, a layer of 32 heads of 128
        {"name": "append 16", "op": "append", "rows": 16, "heads": 32, "dim": 128, "page": 16, "type": "f16",
         "picked": False},
        # a prompt's keys and values, or a step's accepted nodes picked out of its drafts; 8 heads of 128
        {"name": "append 8192 picked", "op": "append", "rows": 8192, "heads": 8, "dim": 128, "page": 64,
         "type": "bf16", "picked": True},
        # one user, one token, 32 heads with a key head each: the smallest call
        {"name": "attention 1x1", "op": "attention", "requests": 1, "new": 1, "context": 301, "q_heads": 32,
         "kv_heads": 32, "dim": 128, "page": 16, "type": "f16"},
        # a batch of single tokens over long contexts, 64 query heads over 8 key heads
        {"name": "attention 16x1", "op": "attention", "requests": 16, "new": 1, "context": 8192, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "page": 32, "type": "bf16"},
        # ragged trees of odd sizes, heads of 64
        {"name": "attention 7x33", "op": "attention", "requests": 7, "new": 33, "context": 3001, "q_heads": 12,
         "kv_heads": 4, "dim": 64, "page": 16, "type": "f16"},
        # the largest: 32 requests verify trees of up to 64 nodes over contexts of up to 8192 tokens
        {"name": "attention 32x64", "op": "attention", "requests": 32, "new": 64, "context": 8192, "q_heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16"},
        # one token, one adapter beside a 4096x4096 projection
        {"name": "lora 1", "op": "lora", "tokens": 1, "cols": 4096, "rows": 4096, "adapters": 4, "rank": 16,
         "type": "f16", "out": "f16", "run": 1},
        # a decode batch in which every request has its own adapter, beside stacked query, key and value rows
        {"name": "lora 48 mixed", "op": "lora", "tokens": 48, "cols": 4096, "rows": 12288, "adapters": 16, "rank": 32,
         "type": "f16", "out": "f32", "run": 1},
        # ragged request lengths, an odd rank, a narrow output
        {"name": "lora 777 ragged", "op": "lora", "tokens": 777, "cols": 8192, "rows": 1024, "adapters": 6,
         "rank": 24, "type": "bf16", "out": "bf16", "run": 37},
        # the prompts of a batch at once beside an 11008x4096 projection
        {"name": "lora 8192", "op": "lora", "tokens": 8192, "cols": 4096, "rows": 11008, "adapters": 8, "rank": 64,
         "type": "bf16", "out": "bf16", "run": 512},
    ]


def _log(rng, low, high):
    """A whole number, spread over the logarithm of low..high; odd where it is large."""
    n = min(high, max(low, round(low * (high / low) ** rng.random())))
    return n if n < 1000 else n - 1 + n % 2


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "lora", "lora"])
    if op == "plan":
        tree = rng.random() < 0.5
        new = _log(rng, 1, 64)
        most = 512 * 64 * 2 // (3 * new)  # never more tokens than the largest listed case
        return {"op": op, "requests": _log(rng, 1, min(most, 512 if tree else 4096)), "new": new,
                "context": _log(rng, 1, 8192), "page": rng.choice([16, 32, 64, 24]), "tree": tree}
    if op == "append":
        heads, dim = rng.choice([1, 4, 8, 8, 32]), rng.choice([64, 128, 128, 96])
        most = 8192 * 8 * 128 // (heads * dim)
        return {"op": op, "rows": _log(rng, 1, min(most, 16384)), "heads": heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 24]), "type": rng.choice(["f16", "bf16"]),
                "picked": rng.random() < 0.5}
    if op == "attention":
        q_heads, kv_heads = rng.choice([(32, 32), (64, 8), (64, 8), (12, 4), (8, 1), (5, 5)])
        requests, new = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        # never more key-query pairs or cached keys than the largest listed case
        context = min(8192, 32 * 64 * 8192 * 64 // (requests * new * q_heads), 32 * 8192 * 8 // (requests * kv_heads))
        return {"op": op, "requests": requests, "new": new, "context": _log(rng, 1, max(1, context)),
                "q_heads": q_heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128, 96]),
                "page": rng.choice([16, 32, 64, 24]), "type": rng.choice(["f16", "bf16"])}
    kind = rng.choice(["f16", "bf16"])
    out = rng.choice([kind, kind, "f32"])
    cols = rng.choice([4096, 4096, 8192, 2040 + 8 * rng.randrange(128)])
    rows = rng.choice([4096, 11008, 1024, 2040 + 8 * rng.randrange(128)])
    rank = rng.choice([8, 16, 16, 32, 64, rng.randrange(1, 65)])
    # never more bytes or products than the largest listed case
    most = min(8192 * (4096 + 2 * 11008) // (cols + (4 if out == "f32" else 2) * rows),
               8192 * (4096 + 11008) // (cols + rows))
    tokens = _log(rng, 1, min(8192, most))
    return {"op": op, "tokens": tokens, "cols": cols, "rows": rows, "adapters": rng.randrange(1, 9), "rank": rank,
            "type": kind, "out": out, "run": rng.choice([1, _log(rng, 1, 512)])}


# ---- inputs -----------------------------------------------------------------------------


def _lengths(case):
    """The case's context lengths and new tokens of each request: ragged, the same for every seed
    (they set the outputs' shapes)."""
    r = random.Random(case["requests"] * 1000003 + case["context"] * 101 + case["new"])
    ctx = [case["context"]] + [r.randint(case["context"] // 4, case["context"]) for _ in range(case["requests"] - 1)]
    new = [case["new"]] + [r.randint(-(-case["new"] // 3), case["new"]) for _ in range(case["requests"] - 1)]
    return ctx, new


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _trees(case, new, seed):
    """Parents of each request's drafted nodes (-1: a root), earlier nodes only."""
    g = torch.Generator("cuda").manual_seed(seed * 7 + 3)
    n = torch.tensor(new, device="cuda")
    node = torch.arange(case["new"], device="cuda").expand(len(new), -1)
    # one in four nodes continues the node before it; the others hang anywhere earlier
    u = torch.rand(len(new), case["new"], generator=g, device="cuda")
    chain = torch.rand(len(new), case["new"], generator=g, device="cuda") < 0.25
    parent = torch.where(chain, node - 1, (u * (node + 1)).long() - 1)
    return parent[node < n[:, None]].to(torch.int32)


def prepare(case, seed):
    seed = int(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    if case["op"] == "plan":
        return _prepare_plan(case, seed, g)
    if case["op"] == "append":
        return _prepare_append(case, seed, g)
    if case["op"] == "attention":
        return _prepare_attention(case, seed, g)
    return _prepare_lora(case, seed, g)


def _prepare_plan(case, seed, g):
    ctx, new = _lengths(case)
    page = case["page"]
    held = [-(-c // page) for c in ctx]
    width = -(-(case["context"] + case["new"]) // page)
    pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + 64
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
    heldt = _ints(held)
    inside = torch.arange(width, device="cuda")[None, :] < heldt[:, None]
    used = sum(held)
    tables[inside] = perm[:used]
    s = {"op": "plan", "page": page, "pages": pages, "tokens": sum(new), "max_new": case["new"], "ctx": _ints(ctx),
         "new": _ints(new), "held": heldt, "tables": tables, "free": perm[used:].contiguous(),
         "head": torch.zeros(1, dtype=torch.int32, device="cuda"),
         "parents": _trees(case, new, seed) if case["tree"] else None}
    if own:
        hqb = _hqb()
        s["plan"] = hqb.PagePlan(len(ctx), sum(new), page, pages, max_new=case["new"] if case["tree"] else 0)
    return s


def _prepare_append(case, seed, g):
    rows, heads, dim, page = case["rows"], case["heads"], case["dim"], case["page"]
    kind = DTYPES[case["type"]]
    source = 2 * rows if case["picked"] else rows
    pages = -(-rows // page) + 4
    k, v = (torch.randn(source, heads, dim, generator=g, device="cuda").to(kind) for _ in range(2))
    kc, vc = (torch.zeros(pages, page, heads, dim, dtype=kind, device="cuda") for _ in range(2))
    slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
    slots = slots.reshape(-1)[:rows].to(torch.int32).contiguous()
    # a step that runs at a fixed size ends in rows without a slot
    if rows > 8:
        slots[-2:] = -1
    picked = torch.randperm(source, generator=g, device="cuda")[:rows].sort()[0].to(torch.int32) if case["picked"] else None
    s = {"op": "append", "k": k, "v": v, "kc": kc, "vc": vc, "slots": slots, "rows": picked}
    if own:
        s["cache"] = _hqb().PagedCache(kc, vc)
    return s


def _prepare_attention(case, seed, g):
    ctx, new = _lengths(case)
    page, kind, dim = case["page"], DTYPES[case["type"]], case["dim"]
    tokens, width = sum(new), -(-max(ctx) // page)
    held = [-(-c // page) for c in ctx]
    pages = sum(held) + 8
    q = torch.randn(tokens, case["q_heads"], dim, generator=g, device="cuda").to(kind)
    k, v = (torch.randn(tokens, case["kv_heads"], dim, generator=g, device="cuda").to(kind) for _ in range(2))
    kc, vc = (torch.randn(pages, page, case["kv_heads"], dim, generator=g, device="cuda", dtype=kind) for _ in range(2))
    tables = torch.zeros(len(ctx), width, dtype=torch.int32, device="cuda")
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables[torch.arange(width, device="cuda")[None, :] < _ints(held)[:, None]] = perm[:sum(held)]
    starts = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    parents = _trees(case, new, seed)
    s = {"op": "attention", "q": q, "k": k, "v": v, "kc": kc, "vc": vc, "tables": tables, "ctx": _ints(ctx),
         "starts": starts, "max_new": case["new"], "max_context": max(ctx), "scale": dim ** -0.5,
         "mask": _pack(_reach(parents, starts, case["new"]), starts, tokens)}
    if own:
        hqb = _hqb()
        s["attention"] = hqb.TreeAttention(hqb.PagedCache(kc, vc), case["q_heads"], len(ctx), tokens, case["new"],
                                           max(ctx))
        s["out"] = torch.empty_like(q)
        s["lse"] = torch.empty(tokens, case["q_heads"], dtype=torch.float32, device="cuda")
    return s


def _prepare_lora(case, seed, g):
    kind, tokens, adapters, rank = DTYPES[case["type"]], case["tokens"], case["adapters"], case["rank"]
    r = random.Random(seed)
    x = torch.randn(tokens, case["cols"], generator=g, device="cuda").to(kind)
    a = (torch.randn(adapters, rank, case["cols"], generator=g, device="cuda") * case["cols"] ** -0.5).to(kind)
    b = (torch.randn(adapters, case["rows"], rank, generator=g, device="cuda") * 0.2).to(kind)
    base = torch.randn(tokens, case["rows"], generator=g, device="cuda").to(DTYPES[case["out"]])
    # adapters of different ranks share the set; the first has the whole rank
    ranks = _ints([rank] + [r.choice([rank, -(-rank // 2), rank]) for _ in range(adapters - 1)])
    scales = torch.rand(adapters, generator=g, device="cuda") + 0.5
    # each request's tokens lie together and have one adapter; one request in eight has none
    pick = torch.randint(0, 8 * adapters, (-(-tokens // case["run"]),), generator=g, device="cuda")
    ids = torch.where(pick % 8 == 7, -1, pick // 8).repeat_interleave(case["run"])[:tokens].to(torch.int32).contiguous()
    s = {"op": "lora", "x": x, "a": a, "b": b, "ranks": ranks, "scales": scales, "ids": ids, "base": base}
    if own:
        s["set"] = _hqb().LoraSet(a, b, ranks, scales)
        s["out"] = torch.empty_like(base)
    return s


# ---- one pass ---------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "lora": _plain_lora}[s["op"]](s)


def _run_own(s):
    if s["op"] == "plan":
        p = s["plan"].build(s["ctx"], s["new"], held=s["held"], tables=s["tables"], free_pages=s["free"],
                            free_head=s["head"], parents=s["parents"])
        out = {"starts": p.starts, "slots": p.slots, "positions": p.positions, "requests": p.requests,
               "held": p.held, "head": p.free_head, "tables": s["tables"]}
        if s["parents"] is not None:
            out["mask"] = p.mask
        return out
    if s["op"] == "append":
        s["cache"].append(s["k"], s["v"], s["slots"], rows=s["rows"])
        return s["kc"], s["vc"]
    if s["op"] == "attention":
        s["attention"](s["q"], s["k"], s["v"], s["tables"], s["ctx"], s["starts"], s["mask"], scale=s["scale"],
                       out=s["out"], lse=s["lse"])
        return s["out"], s["lse"]
    return s["set"].apply(s["x"], s["ids"], base=s["base"], out=s["out"])


def _reach(parents, starts, most):
    """[requests, most, most] truth values: node j is node i or an ancestor of it."""
    n = starts[1:] - starts[:-1]
    inside = torch.arange(most, device=starts.device)[None, :] < n[:, None]
    parent = torch.full(inside.shape, -1, dtype=torch.long, device=starts.device)
    parent[inside] = parents.long()
    step = torch.zeros(len(n), most, most + 1, device=starts.device)
    step.scatter_(2, torch.where(parent >= 0, parent, most)[:, :, None], 1.0)
    step = step[:, :, :most] + torch.eye(most, device=starts.device)
    # (I + parent)^64 counts the ways up the tree: not zero for every ancestor of up to 64 levels
    return (torch.linalg.matrix_power(step, 64) > 0) & inside[:, :, None]


def _pack(reach, starts, tokens):
    """[tokens, words] bits of each token's row of `reach`."""
    most = reach.shape[1]
    words = -(-most // 32)
    bits = torch.nn.functional.pad(reach, (0, 32 * words - most)).reshape(len(reach), most, words, 32).long()
    packed = (bits << torch.arange(32, device=reach.device)).sum(-1)
    packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
    n = starts[1:] - starts[:-1]
    return packed[torch.arange(most, device=reach.device)[None, :] < n[:, None]].contiguous()


def _plain_plan(s):
    page, tokens = s["page"], s["tokens"]
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.cat([zero, s["new"].cumsum(0, dtype=torch.int32)])
    token = torch.arange(tokens, dtype=torch.int32, device="cuda")
    request = torch.searchsorted(starts, token, right=True) - 1
    node = token - starts[request]
    need = (s["ctx"] + s["new"] + page - 1) // page
    fresh = torch.where(s["new"] > 0, (need - s["held"]).clamp(min=0), 0)
    first = s["head"] + torch.cat([zero, fresh.cumsum(0, dtype=torch.int32)])
    column = torch.arange(s["tables"].shape[1], dtype=torch.int32, device="cuda")[None, :]
    taken = (column >= s["held"][:, None]) & (column < (s["held"] + fresh)[:, None])
    at = (first[:-1, None] + column - s["held"][:, None]).clamp(0, len(s["free"]) - 1)
    tables = torch.where(taken, s["free"][at], s["tables"])
    place = s["ctx"][request] + node
    slots = tables[request, place // page] * page + place % page
    depth = node
    out = {}
    if s["parents"] is not None:
        reach = _reach(s["parents"], starts, s["max_new"])
        depth = reach.sum(-1)[request, node] - 1
        out["mask"] = _pack(reach, starts, tokens)
    out.update(starts=starts, slots=slots, positions=(s["ctx"][request] + depth).to(torch.int32),
               requests=request.to(torch.int32), held=s["held"] + fresh, head=first[-1:], tables=tables)
    return out


def _plain_append(s):
    keep = s["slots"] >= 0
    rows = torch.arange(len(s["slots"]), device="cuda") if s["rows"] is None else s["rows"].long()
    at = torch.where(keep, s["slots"], 0).long()
    for cache, new in ((s["kc"], s["k"]), (s["vc"], s["v"])):
        flat = cache.view(-1, *cache.shape[2:])
        flat[at[keep]] = new[rows[keep]]
    return s["kc"], s["vc"]


def _plain_attention(s):
    q, k, v, starts, most = s["q"], s["k"], s["v"], s["starts"], s["max_new"]
    requests, heads, dim = len(starts) - 1, k.shape[1], k.shape[2]
    n, page, width = starts[1:] - starts[:-1], s["kc"].shape[1], s["max_context"]
    node = torch.arange(most, device="cuda")
    inside = node[None, :] < n[:, None]
    token = torch.where(inside, starts[:-1, None] + node[None, :], 0).long()
    place = torch.arange(width, device="cuda")
    slot = (s["tables"].long()[:, place // page] * page + place % page)
    # keys and values of a request: its context through the page table, then its drafted nodes
    keys = torch.cat([s["kc"].view(-1, heads, dim)[slot], k[token]], 1).float()
    values = torch.cat([s["vc"].view(-1, heads, dim)[slot], v[token]], 1).float()
    words = s["mask"][token]
    drafted = (words[:, :, node // 32] >> (node % 32)) & 1 > 0
    cached = (place[None, :] < s["ctx"][:, None])[:, None, :].expand(-1, most, -1)
    visible = torch.cat([cached, drafted & inside[:, None, :]], 2)[:, None, None]
    rows = q[token].float().view(requests, most, heads, -1, dim).permute(0, 2, 3, 1, 4)
    group = rows.shape[2]
    scores = (rows.reshape(requests, heads, group * most, dim) @ keys.permute(0, 2, 3, 1)) * s["scale"]
    scores = scores.view(requests, heads, group, most, -1).masked_fill_(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0, top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = weights.view(requests, heads, group * most, -1) @ values.permute(0, 2, 1, 3)
    out = out.view(requests, heads, group, most, dim) / torch.where(total == 0, 1, total)
    lse = (total.log() + top)[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(requests, most, -1, dim)[inside]
    return out.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(requests, most, -1)[inside]


def _plain_lora(s):
    adapters, rank, cols = s["a"].shape
    column = torch.arange(adapters * rank, device="cuda")
    mine = column[None, :] // rank == s["ids"][:, None]
    real = column % rank < s["ranks"][column // rank]
    weight = torch.where(mine & real, s["scales"][column // rank], 0)
    inner = s["x"].float() @ s["a"].float().view(adapters * rank, cols).T
    outer = s["b"].float().permute(0, 2, 1).reshape(adapters * rank, -1)
    return (s["base"].float() + (inner * weight) @ outer).to(s["base"].dtype)


# ---- work and the 64-bit definition -----------------------------------------------------


def work(case):
    if case["op"] == "plan":
        ctx, new = _lengths(case)
        words = -(-case["new"] // 32) if case["tree"] else 0
        pages = sum(max(0, -(-(c + n) // case["page"]) + (-c // case["page"])) for c, n in zip(ctx, new))
        tokens = sum(new)
        return {"bytes": 4 * (5 * len(ctx) + 2 + 2 * pages + tokens * (3 + words + (1 if case["tree"] else 0))), "flops": 0}
    if case["op"] == "append":
        live = case["rows"] - (2 if case["rows"] > 8 else 0)
        return {"bytes": 2 * 2 * 2 * live * case["heads"] * case["dim"] + 4 * case["rows"], "flops": 0}
    if case["op"] == "attention":
        ctx, new = _lengths(case)
        keys = sum(ctx) + sum(new)
        pairs = sum(n * (c + 1) for c, n in zip(ctx, new))
        return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + sum(new) * case["q_heads"] * (4 * case["dim"] + 4),
                "flops": 4 * pairs * case["q_heads"] * case["dim"]}
    tokens, cols, rows = case["tokens"], case["cols"], case["rows"]
    used = min(case["adapters"], -(-tokens // case["run"]))
    wide = 4 if case["out"] == "f32" else 2
    # seven in eight requests have an adapter; half of the other adapters have half the rank
    return {"bytes": 2 * tokens * cols + 2 * wide * tokens * rows + 2 * used * case["rank"] * (cols + rows),
            "flops": 2 * tokens * case["rank"] * (cols + rows) * 7 / 8}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        where = s["slots"].tolist()
        rows = list(range(len(where))) if s["rows"] is None else s["rows"].tolist()
        for cache, new in ((kc, s["k"]), (vc, s["v"])):
            new = new.double()
            live = [(a, r) for a, r in zip(where, rows) if a >= 0]
            at, row = torch.tensor(live, device="cuda").T
            cache[at // case["page"], at % case["page"]] = new[row]
        return kc, vc
    if case["op"] == "lora":
        x, y = s["x"].double(), s["base"].double()
        ids, ranks, scales = s["ids"].long(), s["ranks"].tolist(), s["scales"].double()
        for adapter, rank in enumerate(ranks):
            mine = (ids == adapter).nonzero()[:, 0]
            a, b = s["a"][adapter, :rank].double(), s["b"][adapter, :, :rank].double()
            y[mine] += scales[adapter] * (x[mine] @ a.T @ b.T)
        return y
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    starts, ctx, page = s["starts"].tolist(), s["ctx"].tolist(), case["page"]
    group = case["q_heads"] // case["kv_heads"]
    bit = torch.arange(case["new"], device="cuda")
    for r, length in enumerate(ctx):
        a, b = starts[r], starts[r + 1]
        pages = s["tables"][r, :-(-length // page)].long()
        seen = (s["mask"][a:b][:, bit[:b - a] // 32] >> (bit[:b - a] % 32)) & 1
        seen = torch.cat([torch.ones(b - a, length, device="cuda", dtype=torch.int32), seen], 1) > 0
        for h in range(case["kv_heads"]):
            key, value = (torch.cat([c[pages, :, h].reshape(-1, case["dim"])[:length], n[a:b, h]]).double()
                          for c, n in ((s["kc"], s["k"]), (s["vc"], s["v"])))
            heads = slice(h * group, (h + 1) * group)
            score = torch.einsum("nhd,kd->hnk", s["q"][a:b, heads].double(), key) * s["scale"]
            score = score.masked_fill(~seen, float("-inf"))
            total = torch.logsumexp(score, -1, keepdim=True)
            out[a:b, heads] = torch.einsum("hnk,kd->nhd", (score - total).exp(), value)
            lse[a:b, heads] = total[..., 0].T
    return out, lse
