"""GPU: the serving operators (page plan, cache append, tree attention, adapters) against plain
implementations in 64 bits, over the sizes, masks, strides and bad values where they can go wrong.

Tolerances, fixed before the first run.  u is the unit roundoff of the 16-bit type (2^-11 FP16,
2^-8 BF16).
* attention: the weights are rounded to the type for the product with v (relative u; FP16 weights
  below its normal range absolutely, 2^-25), the output once more (u); scores are FP32 sums of
  exact products, so with S = scale * sum |q||k| their absolute error is below dim * 2^-24 * S, which
  moves weights by that much relatively; 2^-20 covers the exponential and the FP32 sums.
* adapters: t = A x within cols * 2^-24 * sum |a||x|; its rounding to the type is u * |t| (16-bit outputs)
  or 2^-21 * max |t| (FP32 outputs); the second product adds (rank + 2) * 2^-24 * sum |b||t|, the output u or 2^-24.
* plan and append are exact.
"""

from __future__ import annotations

import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import harpq_b200 as hqb  # noqa: E402

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- page plan ----------------------------------------------------------------------------


def plan_reference(ctx, new, page, pages, held=None, tables=None, free=None, head=0, parents=None, words=0, cap=0):
    """The plan by loops: (outputs, whether any bit of each kind is due)."""
    starts, req, pos, slots, mask, held_out = [0], [], [], [], [], []
    tables = None if tables is None else [list(row) for row in tables]
    bad = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        if c < 0 or n < 0:
            bad |= hqb.DEVERR_INDEX
        c, n = max(c, 0), max(n, 0)
        first = starts[-1]
        if first + n > cap:
            bad |= hqb.DEVERR_INDEX
            n = cap - first
        starts.append(first + n)
        row = None if tables is None else tables[r]
        have = -(-c // page) if held is None else held[r]
        if row is not None:
            if have < 0 or have > len(row) or have < -(-c // page):
                bad |= hqb.DEVERR_INDEX
            have = min(max(have, 0), len(row))
            if n > 0:
                need = -(-(c + n) // page)
                if need > len(row):
                    bad |= hqb.DEVERR_PAGES
                for col in range(have, min(need, len(row))):
                    if head >= len(free):
                        bad |= hqb.DEVERR_PAGES
                        break
                    row[col] = free[head]
                    head += 1
                    have += 1
            held_out.append(have)
        for i in range(n):
            req.append(r)
            depth, bits = i, 0
            if parents is not None:
                at, depth = i, 0
                while True:
                    if at < 32 * words:
                        bits |= 1 << at
                    else:
                        bad |= hqb.DEVERR_INDEX
                    up = parents[first + at]
                    if up < -1 or up >= at:
                        bad |= hqb.DEVERR_INDEX
                    if not 0 <= up < at:
                        break
                    at, depth = up, depth + 1
            mask.append([(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)])
            pos.append(c + depth)
            if row is not None:
                col = (c + i) // page
                got = row[col] if col < have else -1
                if not 0 <= got < pages:
                    bad |= hqb.DEVERR_PAGES
                    slots.append(-1)
                else:
                    slots.append(got * page + (c + i) % page)
    fill = cap - len(req)
    return {"starts": starts, "requests": req + [-1] * fill, "positions": pos + [-1] * fill, "slots": slots + [-1] * fill,
            "mask": mask + [[0] * words] * fill, "held": held_out, "head": head, "tables": tables, "bad": bad}


def run_plan(ctx, new, page, pages, cap, held=None, tables=None, free=None, head=0, parents=None, max_new=0, requests=None):
    plan = hqb.PagePlan(len(ctx), cap, page, pages, max_new=max_new)
    dev = None if tables is None else ints(tables)
    plan.build(ints(ctx), ints(new), held=None if held is None else ints(held), tables=dev,
               free_pages=None if free is None else ints(free), free_head=None if tables is None else ints([head]),
               parents=None if parents is None else ints(parents))
    want = plan_reference(ctx, new, page, pages, held, tables, free, head, parents, plan.words if parents is not None else 0, cap)
    assert plan.starts.tolist() == want["starts"]
    assert plan.requests.tolist() == want["requests"]
    assert plan.positions.tolist() == want["positions"]
    if tables is not None:
        assert plan.slots.tolist() == want["slots"]
        assert plan.held.tolist() == want["held"]
        assert plan.free_head.item() == want["head"]
        assert dev.tolist() == want["tables"]
    if parents is not None:
        assert (plan.mask.to(torch.int64) & 0xFFFFFFFF).tolist() == want["mask"]
    assert plan.flags.item() == want["bad"]
    return plan


def random_plan(rng, requests, page, most_ctx, most_new, slack=4, tree=False, spare=0):
    ctx = [rng.randint(0, most_ctx) for _ in range(requests)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(requests)]
    # some requests hold more pages than their context fills (rejected drafts left them)
    held = [-(-c // page) + rng.choice([0, 0, 1]) for c in ctx]
    width = -(-(most_ctx + most_new) // page) + 1
    pages = requests * width + slack
    pool = list(range(pages))
    rng.shuffle(pool)
    tables = []
    for h in held:
        tables.append([pool.pop() for _ in range(h)] + [-7] * (width - h))
    parents = []
    for n in new:
        parents += [rng.randint(-1, i - 1) if rng.random() < 0.7 else i - 1 for i in range(n)]
    return dict(ctx=ctx, new=new, page=page, pages=pages, held=held, tables=tables, free=pool, head=rng.randint(0, 3),
                cap=sum(new) + spare or 1, parents=parents + [-1] if tree else None, max_new=max(max(new), 1) if tree else 0)


@pytest.mark.parametrize("requests,page,most_ctx,most_new,tree,spare", [
    (1, 16, 40, 1, False, 0), (3, 1, 5, 4, True, 5), (64, 16, 500, 1, False, 0), (255, 24, 100, 9, True, 1),
    (257, 32, 300, 64, True, 700), (1000, 16, 50, 3, False, 0), (5, 64, 1000, 256, True, 3), (600, 7, 9, 90, False, 10)])
def test_plan(requests, page, most_ctx, most_new, tree, spare):
    rng = random.Random(requests * page)
    run_plan(**random_plan(rng, requests, page, most_ctx, most_new, tree=tree, spare=spare))


def test_plan_without_pages_and_without_held():
    run_plan([5, 0, 9], [2, 3, 1], 4, 10, 8)
    run_plan([5, 0, 9], [2, 3, 1], 4, 10, 8, parents=[-1, 0, -1, -1, 1, -1], max_new=3)
    run_plan([5, 0, 9], [2, 3, 1], 4, 20, 8, tables=[[0, 1, -1, -1], [-1] * 4, [2, 3, 4, -1]], free=[9, 8, 7])


def test_plan_runs_out():
    # the pool ends inside the second request; the third gets nothing; the counts stop
    run_plan([4, 4, 4], [4, 9, 5], 4, 20, 18, held=[1, 1, 1], tables=[[0, -1, -1, -1], [1, -1, -1, -1], [2, -1, -1, -1]],
             free=[9, 8, 7])
    # a table row that is too short
    run_plan([4, 4], [9, 1], 4, 20, 10, held=[1, 1], tables=[[0, -1], [1, -1]], free=[9, 8, 7, 6])
    # no free page at all
    run_plan([4, 3], [1, 1], 4, 20, 2, held=[1, 1], tables=[[0, -1], [1, -1]], free=[5], head=1)


def test_plan_bad_values():
    run_plan([-3, 4], [2, -5], 4, 20, 6, held=[0, 1], tables=[[-1, -1], [1, -1]], free=[9, 8])
    run_plan([2, 2, 2], [3, 3, 3], 4, 20, 5, held=[1, 1, 1], tables=[[0, -1], [1, -1], [2, -1]], free=[9, 8, 7])
    run_plan([2, 2], [3, 3], 4, 20, 6, held=[1, 9], tables=[[0, -1], [1, 4]], free=[9, 8, 7])  # more held than the row
    run_plan([2, 9], [1, 2], 4, 20, 3, held=[1, 1], tables=[[0, -1, -1], [1, -1, -1]], free=[9, 8, 7])  # fewer held
    run_plan([2, 2], [1, 1], 4, 20, 2, held=[1, 1], tables=[[25, -1], [-4, -1]], free=[9])  # pages out of range
    run_plan([2], [4], 4, 20, 4, held=[1], tables=[[0, -1]], free=[99])
    run_plan([0], [4], 4, 20, 4, parents=[0, -5, 3, 1], max_new=4)  # parents that are not earlier
    run_plan([0], [40], 4, 20, 40, parents=[i - 1 for i in range(40)], max_new=32)  # nodes past the mask
    run_plan([1, 2], [2 ** 31 - 1, 2 ** 31 - 1], 4, 20, 3)  # sums that pass 32 bits


def test_plan_is_repeatable_and_captured():
    rng = random.Random(5)
    a = random_plan(rng, 40, 16, 200, 20, tree=True)
    plan = hqb.PagePlan(40, a["cap"], 16, a["pages"], max_new=a["max_new"])
    dev = {k: ints(a[k]) for k in ("ctx", "new", "held", "tables", "free", "parents")}
    head = ints([a["head"]])

    def step():
        plan.build(dev["ctx"], dev["new"], held=dev["held"], tables=dev["tables"], free_pages=dev["free"], free_head=head,
                   parents=dev["parents"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    first = [t.clone() for t in (plan.starts, plan.slots, plan.positions, plan.mask, plan.held, plan.free_head, dev["tables"])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    plan.slots.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(first, (plan.starts, plan.slots, plan.positions, plan.mask, plan.held, plan.free_head, dev["tables"])):
        assert torch.equal(x, y)


# ---- cache append --------------------------------------------------------------------------


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("source", [F16, BF16, F32])
@pytest.mark.parametrize("rows,heads,dim,page,heads_first,picked", [
    (1, 1, 8, 1, False, False), (16, 32, 128, 16, False, False), (37, 3, 100, 7, True, True), (5, 2, 1, 4, False, True),
    (300, 8, 64, 24, True, False), (9, 4, 96, 64, False, True)])
def test_append(kind, source, rows, heads, dim, page, heads_first, picked):
    g = torch.Generator("cuda").manual_seed(rows * dim)
    pages = -(-rows // page) + 2
    shape = (pages, heads, page, dim) if heads_first else (pages, page, heads, dim)
    store = [torch.randn(shape, generator=g, device="cuda").to(kind) for _ in range(2)]
    kc, vc = [t.transpose(1, 2) if heads_first else t for t in store]
    cache = hqb.PagedCache(kc, vc)
    # rows inside a wider buffer, as a stacked projection's output leaves them
    total = 2 * rows
    wide = torch.randn(total, 2 * heads * dim + 8, generator=g, device="cuda").to(source)
    k = wide[:, :heads * dim].view(total, heads, dim)
    v = wide[:, heads * dim:2 * heads * dim].view(total, heads, dim)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    if rows > 4:
        slots[2] = -1
    pick = torch.randint(0, total, (rows,), generator=g, device="cuda").to(torch.int32) if picked else None
    if picked and rows > 4:
        pick[3] = -1
    want = [t.clone() for t in (kc, vc)]
    for i in range(rows):
        s, r = int(slots[i]), i if pick is None else int(pick[i])
        if s >= 0 and r >= 0:
            for t, x in zip(want, (k, v)):
                t[s // page, s % page] = x[r].to(kind)
    cache.append(k, v, slots, rows=pick)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    assert cache.flags.item() == 0


def test_append_bad_values_are_skipped():
    kc, vc = torch.zeros(2, 4, 2, 16, dtype=F16, device="cuda"), torch.zeros(2, 4, 2, 16, dtype=F16, device="cuda")
    cache = hqb.PagedCache(kc, vc)
    k = torch.ones(3, 2, 16, dtype=F16, device="cuda")
    cache.append(k, k, ints([8, 1, 2 ** 31 - 1]))
    assert cache.flags.item() == hqb.DEVERR_PAGES
    cache.flags.zero_()
    cache.append(k, k, ints([2, 5]), rows=ints([3, 2]))
    assert cache.flags.item() == hqb.DEVERR_INDEX
    assert kc.view(8, -1).sum(1).tolist() == [0, 32, 0, 0, 0, 32, 0, 0]
    cache.append(k[:0], k[:0], ints([]))


def test_append_past_32_bits():
    # the last page lies beyond 2^32 elements: k and v share one buffer's pages
    page, heads, dim = 64, 8, 128
    pages = 2 ** 32 // (page * heads * dim) + 3
    store = torch.empty(pages, page, heads, dim, dtype=BF16, device="cuda")
    store[-1].zero_(), store[0].zero_(), store[1].zero_(), store[2].zero_()
    cache = hqb.PagedCache(store, store)
    k = torch.randn(2, heads, dim, device="cuda").to(BF16)
    cache.append(k, k, ints([(pages - 1) * page + 5, 7]))
    assert torch.equal(store[-1, 5], k[0]) and torch.equal(store[0, 7], k[1])
    assert store[-1].count_nonzero() <= heads * dim and store[1].count_nonzero() == 0
    # and the attention reads it there
    q = torch.randn(1, heads, dim, device="cuda").to(BF16)
    table = ints([[pages - 1]])
    store[-1].copy_(torch.randn(page, heads, dim, device="cuda"))
    attend = hqb.TreeAttention(cache, heads, 1, 1, 1, page)
    out = attend(q, k[:1], k[:1], table, ints([page]), ints([0, 1]))
    near = hqb.PagedCache(store[-1:].clone(), store[-1:].clone())
    want = hqb.TreeAttention(near, heads, 1, 1, 1, page)(q, k[:1], k[:1], ints([[0]]), ints([page]), ints([0, 1]))
    assert torch.equal(out, want)


# ---- tree attention --------------------------------------------------------------------------


def bits_of(mask, n):
    """[tokens, n] truth values of packed mask rows."""
    j = torch.arange(n, device=mask.device)
    return (mask[:, j // 32] >> (j % 32)) & 1 > 0


def pack(rows, words):
    """Packed int32 mask of [tokens, n] truth values."""
    n = rows.shape[1]
    bits = torch.nn.functional.pad(rows.long(), (0, 32 * words - n)).view(len(rows), words, 32)
    packed = (bits << torch.arange(32, device=rows.device)).sum(-1)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


def attention_reference(q, k, v, cache, tables, ctx, starts, mask, scale):
    """(out, lse, tolerances of both) in 64 bits.  Hidden keys are left out, not weighted by zero."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    group, u, dim = q.shape[1] // k.shape[1], U[q.dtype], q.shape[2]
    place = torch.arange(max([1, *ctx]), device=q.device)
    for r, c in enumerate(ctx):
        a, b = starts[r], starts[r + 1]
        page = tables[r].long()[(place[:c] // cache.page_size)] if c else place[:0]
        kk, vv = (torch.cat([t[page, place[:c] % cache.page_size], x[a:b]]).double() for t, x in ((cache.k, k), (cache.v, v)))
        for i in range(a, b):
            seen = torch.ones(c + b - a, dtype=torch.bool, device=q.device)
            seen[c:] = bits_of(mask[i:i + 1], b - a)[0] if mask is not None else torch.arange(b - a, device=q.device) <= i - a
            if not seen.any():
                continue
            ks, vs = (t[seen].repeat_interleave(group, 1) for t in (kk, vv))  # [keys, q_heads, dim]
            qi = q[i].double()
            s = scale * torch.einsum("hd,khd->kh", qi, ks)
            top = s.amax(0)
            w = (s - top).exp()
            total = w.sum(0)
            out[i] = torch.einsum("kh,khd->hd", w, vs) / total[:, None]
            lse[i] = top + total.log()
            # bounds
            size = abs(scale) * torch.einsum("hd,khd->kh", qi.abs(), ks.abs()).amax(0)
            moved = dim * 2.0 ** -24 * size + 2.0 ** -20
            spread = torch.einsum("kh,khd->hd", w, vs.abs()) / total[:, None]
            tol[i] = (u + 2 * moved[:, None]) * spread + u * out[i].abs()
            if q.dtype == F16:
                tol[i] += 2.0 ** -25 * (vs.abs().sum(0) / total[:, None] + 1)
            ltol[i] = 2 * moved + 2.0 ** -20 * lse[i].abs()
    return out, lse, tol, ltol


def make_attention(seed, ctx, new, q_heads, kv_heads, dim, page, kind, heads_first=False, mask="tree", stacked=False, pad=3):
    g = torch.Generator("cuda").manual_seed(seed)
    rng = random.Random(seed)
    tokens, held = sum(new), [-(-c // page) for c in ctx]
    pages = sum(held) + pad
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    kc, vc = (torch.randn(shape, generator=g, device="cuda").to(kind) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    if stacked:  # q | k | v of one projection's output
        y = torch.randn(tokens, (q_heads + 2 * kv_heads) * dim, generator=g, device="cuda").to(kind)
        q = y[:, :q_heads * dim].view(tokens, q_heads, dim)
        k = y[:, q_heads * dim:(q_heads + kv_heads) * dim].view(tokens, kv_heads, dim)
        v = y[:, (q_heads + kv_heads) * dim:].view(tokens, kv_heads, dim)
    else:
        q = torch.randn(tokens, q_heads, dim, generator=g, device="cuda").to(kind)
        k, v = (torch.randn(tokens, kv_heads, dim, generator=g, device="cuda").to(kind) for _ in range(2))
    order = list(range(pages))
    rng.shuffle(order)
    width = max(1, max(held))
    tables = [[order.pop() for _ in range(h)] + [0] * (width - h) for h in held]
    starts = np.cumsum([0, *new]).tolist()
    most = max(new)
    rows = torch.zeros(tokens, most, dtype=torch.bool)
    for r, n in enumerate(new):
        for i in range(n):
            if mask == "tree":
                rows[starts[r] + i, i] = True
                up = rng.randint(-1, i - 1)
                if up >= 0:
                    rows[starts[r] + i] |= rows[starts[r] + up]
            else:  # any pattern, empty rows among them
                if rng.random() < 0.7:
                    rows[starts[r] + i] = torch.rand(most, generator=torch.Generator().manual_seed(rng.randrange(1 << 30))) < 0.4
    packed = None if mask is None else pack(rows.cuda(), -(-most // 32))
    return dict(q=q, k=k, v=v, kc=kc, vc=vc, tables=ints(tables), ctx=ctx, starts=starts, mask=packed, most=most)


def check_attention(s, scale=None, max_context=None, twice=True):
    cache = hqb.PagedCache(s["kc"], s["vc"])
    q = s["q"]
    scale = cache.dim ** -0.5 if scale is None else scale
    attend = hqb.TreeAttention(cache, q.shape[1], len(s["ctx"]), q.shape[0], s["most"],
                               max(s["ctx"]) if max_context is None else max_context)
    lse = torch.full(q.shape[:2], math.nan, device="cuda")
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    attend(q, s["k"], s["v"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"], scale=scale, out=out, lse=lse)
    want, wlse, tol, ltol = attention_reference(q, s["k"], s["v"], cache, s["tables"], s["ctx"], s["starts"], s["mask"], scale)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {(err - tol).max():.3e} over, err {err.max():.3e}"
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and bool((out[empty] == 0).all())
    lerr = (lse.double() - wlse).abs()[~empty]
    assert bool((lerr <= ltol[~empty]).all()), f"lse err {lerr.max():.3e}"
    assert attend.ws.error_flags() == 0
    if twice:
        again = attend(q, s["k"], s["v"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"], scale=scale)
        assert torch.equal(out, again)
    return out, lse


SHAPES = [
    # ctx, new, q_heads, kv_heads, dim, page
    ([0], [1], 1, 1, 64, 16), ([1], [1], 4, 4, 128, 16), ([63, 64, 65], [1, 1, 1], 8, 8, 128, 16),
    ([300], [1], 32, 32, 128, 16), ([2000, 17, 700], [1, 1, 1], 16, 2, 128, 64), ([5000], [1], 8, 1, 128, 32),
    ([700, 0, 130], [5, 33, 1], 12, 4, 64, 16), ([129, 1000], [64, 17], 8, 1, 128, 24), ([400], [256], 2, 1, 128, 16),
    ([3000, 50], [31, 64], 64, 8, 128, 64), ([100, 200], [7, 9], 6, 2, 96, 16), ([777], [20], 5, 5, 40, 7),
    ([90, 300], [3, 2], 4, 2, 256, 16), ([1500], [30], 16, 1, 160, 300), ([33], [2], 3, 1, 8, 1), ([513], [100], 40, 1, 64, 16),
    ([64 * k for k in range(20)], [1 + k % 5 for k in range(20)], 16, 4, 128, 16),
    # many short pieces of items a CTA, with and without an item's end in them
    ([4096 - 131 * k for k in range(16)], [8 - k % 6 for k in range(16)], 64, 8, 128, 32),
    ([1024 + 128 * k for k in range(24)], [3] * 24, 32, 4, 64, 64), ([640] * 30, [40] * 30, 8, 2, 128, 128),
]


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0][0]}x{len(s[0])}-{s[1][0]}-{s[2]}:{s[3]}x{s[4]}-p{s[5]}")
def test_attention(kind, shape):
    ctx, new, hq, hk, dim, page = shape
    check_attention(make_attention(len(ctx) * 1000 + dim + new[0], ctx, new, hq, hk, dim, page, kind))


@pytest.mark.parametrize("mask", ["tree", "any", None])
@pytest.mark.parametrize("heads_first,stacked", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("hq,hk,dim", [(4, 4, 128), (16, 2, 64), (32, 2, 128)])
def test_attention_layouts_and_masks(mask, heads_first, stacked, hq, hk, dim):
    s = make_attention(77, [90, 0, 700, 65], [9, 40, 1, 12], hq, hk, dim, 16, BF16, heads_first, mask, stacked)
    check_attention(s)


@pytest.mark.parametrize("dim", [1, 3, 100, 130, 254])
def test_attention_unaligned(dim):
    """Head sizes and strides that no 16-byte copy fits."""
    check_attention(make_attention(dim, [70, 3], [6, 2], 6, 3, dim, 5, F16, stacked=True))
    check_attention(make_attention(dim, [130], [40], 8, 1, dim, 16, BF16, heads_first=True, mask="any"))


def test_attention_base_off_16_bytes():
    s = make_attention(9, [200], [12], 8, 1, 128, 16, F16)
    big = torch.randn(s["q"].numel() + 1, device="cuda").half()
    s["q"] = big[1:].view(s["q"].shape)
    check_attention(s)


def test_attention_requests_without_tokens():
    s = make_attention(3, [50, 900, 30, 0, 10], [2, 0, 0, 6, 0], 8, 2, 128, 16, F16)
    check_attention(s)


@pytest.mark.parametrize("hq", [2, 16])
def test_attention_empty_rows(hq):
    """No context and no visible node: zeros and lse -inf, beside rows that see something."""
    s = make_attention(4, [0, 0], [5, 70], hq, 1, 128, 16, BF16)
    s["mask"].zero_()
    s["mask"][2, 0] = 1 << 3
    s["mask"][9, 1] = 1
    out, lse = check_attention(s)
    assert int((lse > -math.inf).sum()) == 2 * hq


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("hq,new", [(1, 6), (8, 40)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_hidden_values_change_nothing(kind, hq, new, bad):
    """NaN and infinities in unused slots of the last page, in pages of others, and in drafted
    keys and values that a node does not see."""
    s = make_attention(6, [45, 300], [new, 3], hq, 1, 128, 16, kind)
    page = 16
    used = torch.zeros(s["kc"].shape[0] * page, dtype=torch.bool, device="cuda")
    for r, c in enumerate(s["ctx"]):
        at = torch.arange(c, device="cuda")
        used[s["tables"][r].long()[at // page] * page + at % page] = True
    for t in (s["kc"], s["vc"]):
        t.view(-1, *t.shape[2:])[~used] = bad
    # nobody sees node 1 of the first request any more; only node 4 sees node 2
    s["mask"][:, 0] &= ~0b110
    s["mask"][4, 0] |= 0b100
    for t in (s["k"], s["v"]):
        t[1] = bad
    check_attention(s)
    # a visible infinity reaches the nodes that see it, and no other
    s["v"][2, 0, 5] = math.inf
    cache = hqb.PagedCache(s["kc"], s["vc"])
    attend = hqb.TreeAttention(cache, hq, 2, new + 3, s["most"], 300)
    out = attend(s["q"], s["k"], s["v"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"])
    lost = ~out.isfinite()
    assert lost[4, :, 5].all() and int(lost.sum()) == hq
    assert (out[4, :, 5] == math.inf).all()


def test_attention_nan_scores_stay_in_their_row():
    s = make_attention(8, [100], [20], 8, 1, 128, 16, F16)
    s["q"][7, 3] = math.nan
    cache = hqb.PagedCache(s["kc"], s["vc"])
    out = hqb.TreeAttention(cache, 8, 1, 20, 20, 100)(s["q"], s["k"], s["v"], s["tables"], ints([100]), ints([0, 20]), s["mask"])
    bad = out.isnan()
    assert bad[7, 3].all() and int(bad.sum()) == 128


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_attention_scales(scale):
    check_attention(make_attention(10, [210], [20], 8, 1, 64, 16, BF16), scale=scale)


@pytest.mark.parametrize("max_context", [0, 40, 100000])
def test_attention_context_bound_is_only_a_bound(max_context):
    check_attention(make_attention(11, [2000, 3], [3, 20], 8, 1, 128, 16, F16), max_context=max_context)


def test_attention_bad_device_values():
    """Clamped or skipped, reported, and nothing else disturbed."""
    s = make_attention(12, [40, 40], [2, 2], 4, 1, 64, 16, F16)
    cache = hqb.PagedCache(s["kc"], s["vc"])
    attend = hqb.TreeAttention(cache, 4, 2, 4, 2, 40)
    args = (s["q"], s["k"], s["v"])
    good = attend(*args, s["tables"], ints([40, 40]), ints([0, 2, 4]), s["mask"])
    tables = s["tables"].clone()
    tables[0, 1] = 10 ** 6
    out = attend(*args, tables, ints([40, 40]), ints([0, 2, 4]), s["mask"])
    assert attend.ws.error_flags() == hqb.DEVERR_PAGES and torch.equal(out[2:], good[2:])
    attend.ws.reset()
    out = attend(*args, s["tables"], ints([1000, 40]), ints([0, 2, 4]), s["mask"])  # past its table row
    assert attend.ws.error_flags() == hqb.DEVERR_PAGES and torch.equal(out[2:], good[2:])
    attend.ws.reset()
    attend(*args, s["tables"], ints([-5, 40]), ints([0, 2, 4]), s["mask"])
    assert attend.ws.error_flags() == hqb.DEVERR_INDEX
    attend.ws.reset()
    for starts in ([0, 3, 4], [-1, 2, 4], [0, 2, 9], [2, 0, 4]):
        attend(*args, s["tables"], ints([40, 40]), ints(starts), s["mask"])
        assert attend.ws.error_flags() == hqb.DEVERR_INDEX, starts
        attend.ws.reset()


@pytest.mark.parametrize("hq,new", [(8, 1), (16, 30)])
def test_attention_streams_and_graphs(hq, new):
    """On another stream, and replayed with lengths that changed on the device."""
    s = make_attention(13, [1200, 30], [new, new], hq, 1, 128, 16, BF16)
    cache = hqb.PagedCache(s["kc"], s["vc"])
    attend = hqb.TreeAttention(cache, hq, 2, 2 * new, new, 1200)
    ctx, starts = ints(s["ctx"]), ints(s["starts"])
    out = torch.empty_like(s["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(s["q"], s["k"], s["v"], s["tables"], ctx, starts, s["mask"], out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(s["q"], s["k"], s["v"], s["tables"], ctx, starts, s["mask"], out=out)
    for lengths in ([1200, 30], [7, 16], [1111, 0]):
        ctx.copy_(ints(lengths))
        out.fill_(math.nan)
        graph.replay()
        want, _, tol, _ = attention_reference(s["q"], s["k"], s["v"], cache, s["tables"], lengths, s["starts"], s["mask"], 128 ** -0.5)
        assert bool(((out.double() - want).abs() <= tol).all()), lengths


# ---- adapters ----------------------------------------------------------------------------------


def lora_reference(x, a, b, ranks, scales, ids, base, kind):
    y = torch.zeros(len(x), b.shape[1], dtype=torch.float64, device="cuda") if base is None else base.double()
    tol = torch.zeros_like(y)
    u, cols = U[x.dtype], x.shape[1]
    for i in range(a.shape[0]):
        mine = (ids == i).nonzero()[:, 0]
        r = a.shape[1] if ranks is None else int(ranks[i])
        if r == 0 or len(mine) == 0:
            continue
        f = 1.0 if scales is None else float(scales[i])
        ai, bi, xi = a[i, :r].double(), b[i, :, :r].double(), x[mine].double()
        t = xi @ ai.T
        y[mine] += f * (t @ bi.T)
        dt = cols * 2.0 ** -24 * (xi.abs() @ ai.abs().T)
        dt += 2.0 ** -21 * t.abs().amax(1, keepdim=True) if kind == F32 else u * t.abs() + 2.0 ** -38 * t.abs().amax(1, keepdim=True)
        tol[mine] += abs(f) * ((dt + (r + 2) * 2.0 ** -24 * t.abs()) @ bi.abs().T)
    return y, tol + U[kind] * y.abs() + (2.0 ** -25 if kind == F16 else 0.0)


def make_lora(seed, tokens, cols, rows, adapters, rank, kind, y_kind, ids=None, full=False):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(tokens, cols, generator=g, device="cuda").to(kind)
    a = (torch.randn(adapters, rank, cols, generator=g, device="cuda") * cols ** -0.5).to(kind)
    b = (torch.randn(adapters, rows, rank, generator=g, device="cuda") * 0.2).to(kind)
    base = torch.randn(tokens, rows, generator=g, device="cuda").to(y_kind)
    ranks = torch.randint(0, rank + 1, (adapters,), generator=g, device="cuda").to(torch.int32)
    ranks[0] = rank
    if full:
        ranks.fill_(rank)
    for i in range(adapters):  # what lies past an adapter's rank is never used
        a[i, int(ranks[i]):] = math.nan
        b[i, :, int(ranks[i]):] = math.inf
    scales = torch.rand(adapters, generator=g, device="cuda") + 0.5
    if ids is None:
        ids = torch.randint(-1, adapters, (tokens,), generator=g, device="cuda").to(torch.int32)
    return x, a, b, ranks, scales, ids, base


def check_lora(x, a, b, ranks, scales, ids, base, y_kind):
    s = hqb.LoraSet(a, b, ranks, scales)
    want, tol = lora_reference(x, a, b, ranks, scales, ids, base, y_kind)
    y = s.apply(x, ids, base=base, y_dtype=y_kind)
    err = (y.double() - want).abs()
    assert y.dtype == y_kind and bool((err <= tol).all()), f"worst {(err - tol).max():.3e} over"
    assert torch.equal(y, s.apply(x, ids, base=base, y_dtype=y_kind))
    if base is not None:
        place = base.clone()
        s.apply(x, ids, base=place, out=place)
        assert torch.equal(place, y)
    assert all(w.error_flags() == 0 for w in s._ws.values())
    return y


@pytest.mark.parametrize("kind,y_kind", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("tokens,cols,rows,adapters,rank", [
    (1, 4096, 4096, 3, 16), (1, 64, 8, 1, 8), (17, 512, 264, 4, 16), (48, 4096, 1024, 16, 32), (5, 1000, 1000, 2, 24),
    (256, 256, 96, 3, 64), (257, 256, 96, 3, 64), (700, 1096, 520, 7, 32), (1500, 512, 768, 2, 128), (33, 768, 320, 5, 128),
    (2000, 128, 64, 300, 8), (640, 2048, 40, 1, 48)])
def test_lora(kind, y_kind, tokens, cols, rows, adapters, rank):
    check_lora(*make_lora(tokens + rank, tokens, cols, rows, adapters, rank, kind, y_kind), y_kind)


@pytest.mark.parametrize("tokens,cols,rows,adapters,rank", [
    (1, 1, 1, 1, 1), (3, 37, 11, 2, 5), (20, 130, 67, 3, 12), (300, 99, 33, 4, 7), (9, 100, 70, 2, 127)])
@pytest.mark.parametrize("kind,y_kind", [(F16, F32), (BF16, BF16), (F16, F16)])
def test_lora_unaligned(kind, y_kind, tokens, cols, rows, adapters, rank):
    check_lora(*make_lora(rank, tokens, cols, rows, adapters, rank, kind, y_kind), y_kind)


@pytest.mark.parametrize("run", [1, 37, 2000])
@pytest.mark.parametrize("tokens,adapters", [(255, 40), (1023, 3), (1024, 1), (1024, 95), (1000, 96), (1025, 5), (513, 700)])
def test_lora_groups_tokens(tokens, adapters, run):
    """Runs of one adapter and mixed ids, on both sides of the sizes at which tokens are grouped in another way."""
    x, a, b, ranks, scales, _, base = make_lora(tokens, tokens, 64, 40, adapters, 16, BF16, BF16)
    g = torch.Generator("cuda").manual_seed(run)
    ids = torch.randint(-1, adapters, (-(-tokens // run),), generator=g, device="cuda").to(torch.int32)
    check_lora(x, a, b, ranks, scales, ids.repeat_interleave(run)[:tokens].contiguous(), base, BF16)


@pytest.mark.parametrize("tokens,rows,adapters,rank", [
    (257, 264, 3, 27), (1000, 520, 8, 61), (1100, 512, 100, 5), (3000, 1024, 7, 33), (2500, 256, 2, 121), (300, 64, 158, 1),
    (300, 64, 159, 1), (1, 512, 3, 27), (20, 264, 18, 13), (20, 264, 19, 13), (256, 520, 8, 63)])
@pytest.mark.parametrize("kind,y_kind", [(F16, F32), (BF16, BF16)])
def test_lora_odd_ranks(kind, y_kind, tokens, rows, adapters, rank):
    """Rows of b that no 16-byte access fits, on both sides of the tokens at which they are laid out."""
    check_lora(*make_lora(rank, tokens, 256, rows, adapters, rank, kind, y_kind), y_kind)


@pytest.mark.parametrize("tokens", [7, 500])
def test_lora_defaults_and_no_base(tokens):
    x, a, b, _, _, ids, _ = make_lora(1, tokens, 256, 128, 3, 16, F16, F16, full=True)
    for kind in (F16, F32):
        check_lora(x, a, b, None, None, ids, None, kind)


@pytest.mark.parametrize("tokens", [40, 400])
def test_lora_one_adapter_and_none(tokens):
    same = torch.full((tokens,), 1, dtype=torch.int32, device="cuda")
    check_lora(*make_lora(2, tokens, 512, 256, 2, 16, BF16, BF16, ids=same, full=True), BF16)
    args = make_lora(3, tokens, 512, 256, 2, 16, BF16, BF16, ids=-same)
    assert torch.equal(check_lora(*args, BF16), args[-1])


@pytest.mark.parametrize("tokens", [30, 333])
def test_lora_strides(tokens):
    """x, base and the result inside wider buffers; an offset that no 16-byte access fits."""
    x, a, b, ranks, scales, ids, base = make_lora(4, tokens, 256, 128, 4, 16, F16, F16)
    want, tol = lora_reference(x, a, b, ranks, scales, ids, base, F16)
    for off in (8, 3):
        xs, bs, ys = (torch.zeros(tokens, n + 16, dtype=F16, device="cuda") for n in (256, 128, 128))
        xs[:, off:off + 256], bs[:, off:off + 128] = x, base
        y = hqb.LoraSet(a, b, ranks, scales).apply(xs[:, off:off + 256], ids, base=bs[:, off:off + 128], out=ys[:, off:off + 128])
        assert bool(((y.double() - want).abs() <= tol).all())
        ys[:, off:off + 128] = 0
        assert ys.count_nonzero() == 0


@pytest.mark.parametrize("size", [2.0 ** -20, 6e4])
def test_lora_activation_range(size):
    """FP16 activations near both ends of the type: the inner vector leaves FP16's range."""
    x, a, b, ranks, scales, ids, _ = make_lora(5, 20, 512, 64, 2, 16, F16, F32, full=True)
    x = (x.float().clamp(-1, 1) * size).half()
    check_lora(x, (a.float() * 20).half(), b, ranks, scales, ids, None, F32)


@pytest.mark.parametrize("tokens", [20, 300])
def test_lora_infinities_stay_in_their_token(tokens):
    x, a, b, ranks, scales, ids, base = make_lora(6, tokens, 256, 64, 2, 16, BF16, BF16, full=True)
    ids.fill_(0)
    x[3, 7], x[5, 9] = math.inf, math.nan
    y = hqb.LoraSet(a, b, ranks, scales).apply(x, ids, base=base)
    t = a[0].float() @ x[3].float()
    want = base[3].float() + float(scales[0]) * (b[0].float() @ t)
    assert torch.equal(y[3].isnan(), want.isnan()) and torch.equal(y[3].isinf(), want.isinf())
    assert y[5].isnan().all()
    rest = torch.ones(tokens, dtype=torch.bool, device="cuda")
    rest[3] = rest[5] = False
    assert y[rest].isfinite().all()


@pytest.mark.parametrize("tokens", [10, 400])
def test_lora_bad_device_values(tokens):
    x, a, b, ranks, scales, ids, base = make_lora(7, tokens, 256, 64, 2, 16, F16, F16, full=True)
    s = hqb.LoraSet(a, b, ranks, scales)
    ids.fill_(0)
    good = s.apply(x, ids, base=base)
    ids[4] = 9
    y = s.apply(x, ids, base=base)
    ws = next(iter(s._ws.values()))
    assert ws.error_flags() == hqb.DEVERR_INDEX
    keep = torch.arange(tokens, device="cuda") != 4
    assert torch.equal(y[4], base[4]) and torch.equal(y[keep], good[keep])
    ws.reset()
    ranks[0] = 99
    ids[4] = 0
    assert torch.equal(s.apply(x, ids, base=base), good) and ws.error_flags() == hqb.DEVERR_INDEX


@pytest.mark.parametrize("tokens", [20, 500])
def test_lora_streams_and_graphs(tokens):
    x, a, b, ranks, scales, ids, base = make_lora(8, tokens, 512, 256, 4, 32, BF16, BF16)
    s = hqb.LoraSet(a, b, ranks, scales)
    out = torch.empty_like(base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.apply(x, ids, base=base, out=out)
    torch.cuda.current_stream().wait_stream(side)
    want = out.clone()
    ws = s.workspace(tokens, torch.cuda.current_stream().cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.apply(x, ids, base=base, out=out, workspace=ws)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    ids.fill_(-1)
    graph.replay()
    assert torch.equal(out, base)


def test_lora_graph_outlives_a_larger_call():
    """A captured call keeps its workspace when a later call needs a larger one."""
    import harpq_b200_ops  # noqa: F401

    x, a, b, ranks, scales, ids, base = make_lora(9, 3000, 512, 256, 4, 32, BF16, BF16)
    s = hqb.LoraSet(a, b, ranks, scales, max_tokens=300)
    out, few = torch.empty_like(base[:300]), (x[:300], ids[:300])
    want = s.apply(*few, base=base[:300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # as a capture wants it: warmed up on its stream
        s.apply(*few, base=base[:300], out=out)
        torch.ops.harpq_b200.lora(x[:300], a, b, ids[:300], ranks, scales, base[:300])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.apply(*few, base=base[:300], out=out)
            other = torch.ops.harpq_b200.lora(x[:300], a, b, ids[:300], ranks, scales, base[:300])
        s.apply(x, ids, base=base)
        torch.ops.harpq_b200.lora(x, a, b, ids, ranks, scales, base)
        filler = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]  # takes what was freed
        out.zero_()
        graph.replay()
        filler.append(filler[0].clone())
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want)
    assert all(bool((f == -1).all()) for f in filler)


def test_lora_beside_a_plane_matrix():
    """In place on a quantized projection's output, as a decoder layer runs it."""
    from conftest import plane_matrix, random_matrix

    pm = plane_matrix(random_matrix(np.random.default_rng(3), 384, 512))
    x, a, b, ranks, scales, ids, _ = make_lora(9, 12, 512, 384, 3, 16, F16, F32)
    y = pm.gemv(x, prefix=2, y_dtype=F32)
    want, tol = lora_reference(x, a, b, ranks, scales, ids, y.clone(), F32)
    hqb.LoraSet(a, b, ranks, scales).apply(x, ids, base=y, out=y)
    assert bool(((y.double() - want).abs() <= tol).all())


# ---- refusals of the binding, the PyTorch operators, the example ---------------------------------


def test_binding_refusals():
    k = torch.zeros(4, 16, 2, 64, dtype=F16, device="cuda")
    cache = hqb.PagedCache(k, k.clone())
    for bad in ((k, k.bfloat16()), (k, k[:2]), (k, k.transpose(1, 2)), (k[..., ::2], k[..., ::2]), (k[0], k[0])):
        with pytest.raises(ValueError):
            hqb.PagedCache(*bad)
    with pytest.raises(TypeError):
        hqb.PagedCache(k.float(), k.float())
    rows, slots = torch.zeros(3, 2, 64, dtype=F16, device="cuda"), ints([0, 1, 2])
    for bad in ((rows[:2], rows[:2], slots), (rows, rows[:2], slots), (rows[:, :1], rows[:, :1], slots), (rows, rows, slots.long()),
                (rows, rows, slots.cpu()), (rows, rows.transpose(0, 1).contiguous().transpose(0, 1), slots)):
        with pytest.raises(ValueError):
            cache.append(*bad)
    with pytest.raises(TypeError):
        cache.append(rows.double(), rows.double(), slots)
    for bad in (dict(q_heads=3), dict(max_new=0), dict(max_new=257), dict(requests=0), dict(tokens=0)):
        with pytest.raises(ValueError):
            hqb.TreeAttention(cache, **{**dict(q_heads=4, requests=1, tokens=3, max_new=3, max_context=10), **bad})
    attend = hqb.TreeAttention(cache, 4, 1, 3, 3, 10)
    q, tables, one, starts = torch.zeros(3, 4, 64, dtype=F16, device="cuda"), ints([[0]]), ints([3]), ints([0, 3])
    good = dict(q=q, k=rows, v=rows, tables=tables, context_lens=one, starts=starts)
    attend(**good)
    for bad in (dict(q=q[:, :2]), dict(k=rows[:2]), dict(tables=ints([0])), dict(starts=ints([0])), dict(mask=ints([[1]])),
                dict(context_lens=one.long()), dict(lse=torch.zeros(3, 4, device="cuda").half()), dict(out=q[:2])):
        with pytest.raises((ValueError, TypeError)):
            attend(**{**good, **bad})
    with pytest.raises(TypeError):
        attend(**{**good, "q": q.bfloat16()})
    with pytest.raises(ValueError):
        attend(torch.zeros(4, 4, 64, dtype=F16, device="cuda"), *[torch.zeros(4, 2, 64, dtype=F16, device="cuda")] * 2, tables, one, starts)
    a, b = torch.zeros(2, 8, 64, dtype=F16, device="cuda"), torch.zeros(2, 32, 8, dtype=F16, device="cuda")
    for bad in ((a, b[:1]), (a, b.transpose(1, 2)), (a[:, :, ::2], b), (torch.zeros(2, 129, 4, device="cuda").half(), torch.zeros(2, 4, 129, device="cuda").half())):
        with pytest.raises(ValueError):
            hqb.LoraSet(*bad)
    with pytest.raises(TypeError):
        hqb.LoraSet(a, b.bfloat16())
    with pytest.raises(ValueError):
        hqb.LoraSet(a, b, ranks=ints([1]))
    s, x, ids = hqb.LoraSet(a, b), torch.zeros(3, 64, dtype=F16, device="cuda"), ints([0, 1, -1])
    for bad in (dict(x=x[:, :32]), dict(x=x.float()), dict(ids=ids[:2]), dict(base=x), dict(out=torch.zeros(3, 32, device="cuda").bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            s.apply(**{**dict(x=x, ids=ids), **bad})
    plan = hqb.PagePlan(2, 4, 16, 8)
    for bad in (dict(context_lens=ints([1])), dict(new_lens=ints([1, 2]).long()), dict(tables=ints([[0], [1]])), dict(parents=ints([-1, 0, -1, 0]))):
        with pytest.raises(ValueError):
            plan.build(**{**dict(context_lens=ints([1, 2]), new_lens=ints([2, 2])), **bad})


def test_torch_operators_match_the_binding():
    import harpq_b200_ops  # noqa: F401

    ops = torch.ops.harpq_b200
    s = make_attention(21, [40, 300], [5, 9], 8, 2, 64, 16, F16)
    out, _ = check_attention(s)
    again = ops.tree_attention(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"],
                               s["most"], 300, None)
    assert torch.equal(out, again)
    slots = torch.arange(14, dtype=torch.int32, device="cuda").flip(0).contiguous()
    kc, vc = s["kc"].clone(), s["vc"].clone()
    hqb.PagedCache(kc, vc).append(s["k"], s["v"], slots)
    ops.cache_append(s["kc"], s["vc"], s["k"], s["v"], slots)
    assert torch.equal(kc, s["kc"]) and torch.equal(vc, s["vc"])
    for tokens in (9, 600):
        x, a, b, ranks, scales, ids, base = make_lora(22, tokens, 128, 64, 3, 16, BF16, BF16)
        y = hqb.LoraSet(a, b, ranks, scales).apply(x, ids, base=base)
        assert torch.equal(y, ops.lora(x, a, b, ids, ranks, scales, base))


@pytest.mark.parametrize("requests", [1, 3])
def test_drafted_trees_decode_as_plain_decoding(requests):
    """The example: page plan, adapters, tree attention and cache append around quantized projections."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import draft_tree_decode

    same, rate = draft_tree_decode.main(requests, 20)
    assert same and rate >= 1.0
