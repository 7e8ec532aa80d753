"""GPU: cases at the edges of the serving operators' contracts, each against the plain forms of
test_gpu_serving.py (whose tolerances hold here too)."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import harpq_b200 as hqb  # noqa: E402
from test_gpu_serving import BF16, F16, F32, U, check_attention, ints, lora_reference, make_attention, make_lora, plan_reference  # noqa: E402


# ---- page plan ----------------------------------------------------------------------------


@pytest.mark.parametrize("requests,nodes,given", [(1, 4, 1), (3, 5, 7), (3, 5, 5), (300, 7, 900), (2, 200, 201), (4, 3, 0)])
def test_plan_with_fewer_parents_than_tokens(requests, nodes, given):
    """Tokens past the parents count as roots, with HQB_DEVERR_INDEX; nothing past them is read."""
    tokens = requests * nodes
    parents = [i % nodes - 1 for i in range(tokens)]
    plan = hqb.PagePlan(requests, tokens + 3, 16, 8, max_new=nodes)
    # the entries stand before others that would be valid parents
    store = ints(parents + [0] * 16)
    plan.build(ints([9] * requests), ints([nodes] * requests), parents=store[:given])
    roots = parents[:given] + [-1] * (tokens - given)
    want = plan_reference([9] * requests, [nodes] * requests, 16, 8, parents=roots, words=plan.words, cap=tokens + 3)
    assert plan.positions.tolist() == want["positions"]
    assert (plan.mask.to(torch.int64) & 0xFFFFFFFF).tolist() == want["mask"]
    assert plan.flags.item() == hqb.DEVERR_INDEX


def test_plan_of_no_tokens_takes_no_parents():
    plan = hqb.PagePlan(2, 3, 16, 8, max_new=4)
    plan.build(ints([9, 4]), ints([0, 0]), parents=ints([]))
    assert plan.starts.tolist() == [0, 0, 0] and plan.positions.tolist() == [-1] * 3 and plan.flags.item() == 0


def test_plan_gives_no_outputs_of_an_earlier_build():
    """A tree's mask would hide a later chain's nodes; slots of an earlier step would be written again."""
    plan = hqb.PagePlan(1, 4, 16, 8, max_new=4)
    assert plan.slots is not None and plan.mask is not None
    paged = dict(held=ints([1]), tables=ints([[3, -1]]), free_pages=ints([5, 6]), free_head=ints([0]))
    plan.build(ints([14]), ints([4]), parents=ints([-1, 0, 0, 1]), **paged)
    assert plan.slots.tolist() == [62, 63, 80, 81] and plan.held.tolist() == [2] and plan.free_head.tolist() == [1]
    assert plan.mask.flatten().tolist() == [1, 3, 5, 11]
    plan.build(ints([14]), ints([4]), parents=ints([-1, 0, 0, 1]))
    assert plan.slots is None and plan.held is None and plan.free_head is None and plan.mask is not None
    plan.build(ints([14]), ints([4]), **paged)
    assert plan.slots is not None and plan.mask is None


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("hq", [1, 24])
@pytest.mark.parametrize("above", [1.3, 2.0, 2.009, 2.02, 5.5, 5.6, 40.0])
def test_attention_maximum_grows(kind, hq, above):
    """A later key above all earlier ones by less and by more than what the kernels' reference may lag behind
    (2.9 and 8 in the exponent to base 2): no weight leaves its type."""
    s = make_attention(31, [1500, 700], [1, 1], hq, 1, 64, 16, kind)
    s["q"].zero_(), s["kc"].zero_()
    s["q"][..., 0] = 1
    for r, key in ((0, 1200), (1, 600)):
        s["kc"][s["tables"][r, key // 16], key % 16, 0, 0] = above
    check_attention(s, scale=1.0)


# ---- memory that callers bring --------------------------------------------------------------


def test_workspaces_in_host_memory_are_refused():
    k = torch.zeros(4, 16, 2, 64, dtype=F16, device="cuda")
    with pytest.raises(ValueError):
        hqb.TreeAttention(hqb.PagedCache(k, k), 4, 1, 3, 3, 10, workspace=lambda need: hqb.Workspace(need, "cpu"))
    x, a, b, ranks, scales, ids, base = make_lora(1, 5, 64, 32, 2, 8, BF16, BF16)
    with pytest.raises(ValueError):
        hqb.LoraSet(a, b, ranks, scales).apply(x, ids, base=base, workspace=hqb.Workspace(1 << 20, "cpu"))


def test_captures_have_workspaces_of_their_own():
    """Two graphs captured on one stream, and eager calls on it, may run at once."""
    import harpq_b200_ops  # noqa: F401

    many = make_lora(2, 3000, 256, 128, 5, 32, BF16, BF16)
    a, b, ranks, scales = many[1:5]
    s = hqb.LoraSet(a, b, ranks, scales, max_tokens=0)
    sizes = (3000, 1700, 2300)
    inputs = [(many[0][:n].clone(), many[5][:n].clone(), many[6][:n].clone()) for n in sizes]
    want = [s.apply(x, ids, base=base).clone() for x, ids, base in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs, places = [], [], []
    for x, ids, base in inputs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append((s.apply(x, ids, base=base), torch.ops.harpq_b200.lora(x, a, b, ids, ranks, scales, base)))
            places.append(s.workspace(len(x), side.cuda_stream).ptr())
        graphs.append(graph)
    with torch.cuda.stream(side):
        places.append(s.workspace(3000, side.cuda_stream).ptr())
        assert s.workspace(3000, side.cuda_stream).error_flags() == 0  # though no graph has run yet
    assert len(set(places)) == 3
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(side):
            eager = s.apply(*inputs[2][:2], base=inputs[2][2])
    torch.cuda.synchronize()
    assert torch.equal(eager, want[2])
    for (own, op), w in zip(outs, want):
        assert torch.equal(own, w) and torch.equal(op, w)


def test_captured_operators_of_attention_have_workspaces_of_their_own():
    import harpq_b200_ops

    graphs, outs, want, keep, places = [], [], [], [], []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        s = make_attention(seed, [3000, 2000], [9, 7], 16, 2, 64, 16, F16)
        keep.append((s["q"], s["k"], s["v"], s["kc"], s["vc"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"], s["most"], 3000))
        want.append(torch.ops.harpq_b200.tree_attention(*keep[-1]))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(torch.ops.harpq_b200.tree_attention(*keep[-1]))
            place = harpq_b200_ops._serving_workspace("attention", keep[-1][0].device, side.cuda_stream, 1).ptr()
        assert place not in places
        places.append(place)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_workspace_given_to_a_capture_is_kept():
    """Also where it is the stream's own, and a later call replaces that one."""
    x, a, b, ranks, scales, ids, base = make_lora(2, 3000, 256, 128, 5, 32, BF16, BF16)
    s, stream = hqb.LoraSet(a, b, ranks, scales, max_tokens=0), torch.cuda.current_stream().cuda_stream
    few = (x[:1100], ids[:1100])
    want = s.apply(*few, base=base[:1100])
    graph, place = torch.cuda.CUDAGraph(), s.workspace(1100, stream).ptr()
    with torch.cuda.graph(graph):
        out = s.apply(*few, base=base[:1100], workspace=s._ws[stream])
    size = s.workspace(1100, stream).nbytes
    s.apply(x, ids, base=base)
    filler = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]  # takes what was freed
    assert s.workspace(1, stream).ptr() != place and all(f.data_ptr() != place for f in filler)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want) and all(bool((f == 255).all()) for f in filler)


def test_a_grown_workspace_keeps_its_error_word():
    x, a, b, ranks, scales, ids, base = make_lora(3, 3000, 256, 64, 2, 16, F16, F16, full=True)
    s = hqb.LoraSet(a, b, ranks, scales, max_tokens=0)
    bad = ids[:300].clone()
    bad[7] = 9
    s.apply(x[:300], bad, base=base[:300])
    s.apply(x, ids, base=base)
    assert s.workspace(1, torch.cuda.current_stream().cuda_stream).error_flags() == hqb.DEVERR_INDEX


# ---- tree attention -------------------------------------------------------------------------


@pytest.mark.parametrize("hq", [1, 16])
@pytest.mark.parametrize("max_context", [40, 4000])
@pytest.mark.parametrize("ctx,starts", [([40], [2, 0]), ([40], [-1, -1]), ([-5], [0, 0]), ([3, 40], [4, 1, 0]), ([40], [9, 9])])
def test_attention_reports_bad_lengths_where_nothing_is_left_to_do(hq, max_context, ctx, starts):
    s = make_attention(12, [40, 40], [2, 2], hq, 1, 64, 16, F16)
    attend = hqb.TreeAttention(hqb.PagedCache(s["kc"], s["vc"]), hq, 2, 4, 2, max_context)
    attend(s["q"], s["k"], s["v"], s["tables"][:len(ctx)].contiguous(), ints(ctx), ints(starts), s["mask"])
    assert attend.ws.error_flags() == hqb.DEVERR_INDEX


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("group,heads,keys,gap", [
    (1, 1, 60000, 18.25), (32, 1, 60000, 18.25), (1, 1, 400, 14.0), (24, 1, 400, 14.0), (32, 1, 3000, 12.5),
    # more heads than CTAs: one of them sees nearly all keys of a head
    (1, 296, 8000, 18.25), (24, 148, 8000, 18.25)])
def test_attention_many_small_weights(kind, group, heads, keys, gap):
    """One key far above very many others, whose values make up the result: weights w of 2^-18 to 2^-26.3
    of the largest.  A weight is rounded by at most u w, or by 2^-25 of FP16's weights up to 2^13 for the
    largest key (2^-38 of that one); scores here are exact, the exponential within 2^-20."""
    hq = group * heads
    q = torch.zeros(1, hq, 64, dtype=kind, device="cuda")
    q[..., 0] = 1
    k, v = (torch.zeros(-(-keys // 16), 16, heads, 64, dtype=kind, device="cuda") for _ in range(2))
    k[keys // 16 // 2, 3, :, 0] = gap
    v[:] = 1000
    v[keys // 16 // 2, 3] = 0
    own = torch.zeros(1, heads, 64, dtype=kind, device="cuda")
    own[..., 0] = -60000.0  # the step's own key counts for nothing
    attend = hqb.TreeAttention(hqb.PagedCache(k, v), hq, 1, 1, 1, keys)
    lse = torch.empty(1, hq, device="cuda")
    out = attend(q, own, own, ints([list(range(len(k)))]), ints([keys]), ints([0, 1]), scale=1.0, lse=lse)
    small = (keys - 1) * math.exp(-gap)
    want = 1000 * small / (1 + small)
    tol = (2 * U[kind] + 2.0 ** -19) * want + 2.0 ** -38 * (keys - 1) * 1000 / (1 + small)
    err = (out.double() - want).abs().max().item()
    assert err <= tol, f"{err:.3e} over {tol:.3e} at {want:.3e}"
    assert (lse.double() - gap - math.log1p(small)).abs().max().item() <= 2.0 ** -20 * gap + 2.0 ** -20
    assert attend.ws.error_flags() == 0


@pytest.mark.parametrize("requests", [33, 64, 100])
@pytest.mark.parametrize("hq,hk,dim", [(2, 2, 64), (8, 2, 128), (40, 2, 64)])
@pytest.mark.parametrize("most", [60, 700])
def test_attention_of_many_requests(requests, hq, hk, dim, most):
    """More requests than one round of 32 lengths, some without tokens where two rounds meet."""
    ctx = [(r * 97 + 13) % most for r in range(requests)]
    new = [1 + r % 3 for r in range(requests)]
    for r in (0, 31, 32, 63, 64, 65, requests - 1):
        if r < requests:
            new[r] = 0
    ctx[5], ctx[31] = most, most * 2
    check_attention(make_attention(requests, ctx, new, hq, hk, dim, 16, F16))


def test_attention_of_many_requests_without_tokens():
    """Whole rounds of requests without tokens before and behind the one that has some."""
    new = [0] * 70 + [5] + [0] * 60
    for hq in (2, 16):
        check_attention(make_attention(1, [3 * r for r in range(131)], new, hq, 1, 64, 16, BF16))


@pytest.mark.parametrize("page", [64, 4])
@pytest.mark.parametrize("group", [1, 32])
def test_attention_past_32_bits(group, page):
    """Pages beyond 2^32 elements, and rows of q, k, v and out beyond 2^31, by each kernel and kind of copy."""
    heads, dim = 4, 128
    pages = 2 ** 32 // (page * heads * dim) + 40
    store = torch.empty(pages, page, heads, dim, dtype=BF16, device="cuda")
    last = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda")
    store[-40:] = torch.randn(40, page, heads, dim, device="cuda").to(BF16)
    keys, far = 40 * page - 3, 2 ** 31 + 64
    q, k, v = (torch.randn(2, n, dim, device="cuda").to(BF16) for n in (heads * group, heads, heads))
    near = store[-40:].clone()
    args = ints([keys, keys - 2]), ints([0, 1, 2])
    want = hqb.TreeAttention(hqb.PagedCache(near, near), heads * group, 2, 2, 1, 4000)(
        q, k, v, (last - (pages - 40)).expand(2, -1).contiguous(), *args)
    wide = []
    for t in (q, k, v, want):
        wide.append(torch.empty(far + t[0].numel(), dtype=BF16, device="cuda").as_strided(t.shape, (far, dim, 1)))
        wide[-1].copy_(t)
    wide[3].zero_()
    attend = hqb.TreeAttention(hqb.PagedCache(store, store), heads * group, 2, 2, 1, 4000)
    attend(*wide[:3], last.expand(2, -1).contiguous(), *args, out=wide[3])
    assert torch.equal(wide[3], want) and attend.ws.error_flags() == 0


@pytest.mark.parametrize("tokens,far", [(2, 2 ** 31 + 64), (600, 2 ** 23 + 64)])
def test_lora_rows_past_32_bits(tokens, far):
    x, a, b, ranks, scales, ids, base = make_lora(tokens, tokens, 256, 128, 3, 64, F16, F32)
    ids[-1] = 0
    want, tol = lora_reference(x, a, b, ranks, scales, ids, base, F32)
    xs = torch.empty(far * (tokens - 1) + 256, dtype=F16, device="cuda").as_strided(x.shape, (far, 1))
    ys = torch.empty(far * (tokens - 1) + 128, dtype=F32, device="cuda").as_strided(base.shape, (far, 1))
    xs.copy_(x), ys.copy_(base)
    s = hqb.LoraSet(a, b, ranks, scales)
    s.apply(xs, ids, base=ys, out=ys)
    assert bool(((ys.double() - want).abs() <= tol).all()) and s.error_flags() == 0


@pytest.mark.parametrize("tokens,rank,cols,rows", [
    (3, 64, 64, 2 ** 18), (600, 64, 64, 2 ** 18), (600, 63, 64, 2 ** 18), (3, 63, 64, 2 ** 18), (3, 64, 2 ** 18, 64), (600, 64, 2 ** 18, 64)])
def test_lora_sets_past_32_bits(tokens, rank, cols, rows):
    """The last adapter's a or b begins beyond 2^32 elements."""
    adapters = 2 ** 32 // (rank * max(cols, rows)) + 2
    a = torch.empty(adapters, rank, cols, dtype=BF16, device="cuda")
    b = torch.empty(adapters, rows, rank, dtype=BF16, device="cuda")
    a[-1] = torch.randn(rank, cols, device="cuda") * cols ** -0.5
    b[-1] = torch.randn(rows, rank, device="cuda") * 0.2
    x = torch.randn(tokens, cols, device="cuda").to(BF16)
    ids = torch.full((tokens,), adapters - 1, dtype=torch.int32, device="cuda")
    y = hqb.LoraSet(a, b, max_tokens=0).apply(x, ids)
    want = hqb.LoraSet(a[-1:].clone(), b[-1:].clone(), max_tokens=0).apply(x, torch.zeros_like(ids))
    t, u = x.float() @ a[-1].float().T, U[BF16]
    size = t.abs() @ b[-1].float().abs().T
    # the same product, by kernels that may sum it in another order (the sizes choose them)
    assert bool(((y.float() - want.float()).abs() <= 2 * u * want.float().abs() + 4 * u * size).all())
    assert y.count_nonzero() > y.numel() // 2


def test_one_workspace_serves_a_stream():
    """Sets and attentions of several layers, one after the other on a stream, in one workspace."""
    layers = [make_lora(n, n, 256, 128, 4, rank, F16, F32) for n, rank in ((7, 16), (900, 64), (300, 27), (40, 8))]
    sets = [hqb.LoraSet(*t[1:5], max_tokens=0) for t in layers]
    ws = hqb.Workspace(max(s.workspace_bytes(len(t[0])) for s, t in zip(sets, layers)))
    want = [s.apply(t[0], t[5], base=t[6]) for s, t in zip(sets, layers)]
    got = [s.apply(t[0], t[5], base=t[6], workspace=ws) for s, t in zip(sets, layers)]
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and ws.error_flags() == 0
    steps = [make_attention(i, [900, 2000], [n, 3], hq, 2, 64, 16, F16) for i, (n, hq) in enumerate(((1, 2), (30, 16), (2, 4)))]
    shared = hqb.Workspace(64 << 20)
    outs = []
    for own in (True, False):
        attends = [hqb.TreeAttention(hqb.PagedCache(s["kc"], s["vc"]), s["q"].shape[1], 2, len(s["q"]), s["most"], 2000,
                                     workspace=None if own else lambda need: shared) for s in steps]
        outs.append([f(s["q"], s["k"], s["v"], s["tables"], ints(s["ctx"]), ints(s["starts"]), s["mask"]) for f, s in zip(attends, steps)])
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and shared.error_flags() == 0


def test_operators_take_steps_without_tokens():
    ops = torch.ops.harpq_b200
    import harpq_b200_ops  # noqa: F401

    s = make_attention(12, [40], [2], 4, 2, 64, 16, F16)
    x, a, b, ranks, scales, ids, base = make_lora(7, 4, 64, 32, 2, 8, F16, F16)
    before = s["kc"].clone()
    ops.cache_append(s["kc"], s["vc"], s["k"][:0], s["v"][:0], ints([]))
    assert torch.equal(s["kc"], before)
    out = ops.tree_attention(s["q"][:0], s["k"][:0], s["v"][:0], s["kc"], s["vc"], s["tables"], ints([40]), ints([0, 0]), None, 2, 40)
    assert out.shape == (0, 4, 64) and out.dtype == F16
    assert ops.lora(x[:0], a, b, ids[:0], ranks, scales, base[:0]).shape == (0, 32)


def test_new_results_come_from_the_memory_of_their_stream():
    """A block that the current stream has just given up may still be in use there."""
    side = torch.cuda.Stream()
    x, a, b, ranks, scales, ids, base = make_lora(7, 9, 64, 4104, 2, 8, F16, F32)
    t = make_attention(12, [40], [9], 36, 4, 64, 16, F16)
    lora, attend = hqb.LoraSet(a, b, ranks, scales), hqb.TreeAttention(hqb.PagedCache(t["kc"], t["vc"]), 36, 1, 9, 9, 40)
    args = (t["q"], t["k"], t["v"], t["tables"], ints([40]), ints([0, 9]), t["mask"])
    torch.cuda.synchronize()
    for call in (lambda s: lora.apply(x, ids, base=base, stream=s), lambda s: attend(*args, stream=s)):
        want = call(None)
        for stream in (side, side.cuda_stream):
            out = call(stream)
            side.synchronize()
            assert torch.equal(out, want)
            place, size, kind = out.data_ptr(), out.shape, out.dtype
            del out
            with torch.cuda.stream(side):
                again = torch.empty(size, dtype=kind, device="cuda")
            assert again.data_ptr() == place


def test_handles_are_freed_with_their_last_reference():
    """Not by the garbage collector: they hold large workspaces."""
    import gc
    import weakref

    x, a, b, ranks, scales, ids, base = make_lora(7, 9, 64, 32, 2, 8, F16, F32)
    t = make_attention(12, [40], [9], 4, 2, 64, 16, F16)
    gc.disable()
    try:
        cache = hqb.PagedCache(t["kc"], t["vc"])
        for make in (lambda: hqb.LoraSet(a, b, ranks, scales), lambda: hqb.TreeAttention(cache, 4, 1, 9, 9, 40),
                     lambda: hqb.PagePlan(1, 9, 16, 8, max_new=9)):
            handle = make()
            seen = weakref.ref(handle)
            del handle
            assert seen() is None
    finally:
        gc.enable()


@pytest.mark.parametrize("aside", [False, True])
def test_default_stream_has_its_own_memory(aside):
    """Its handle is 0, which PyTorch's wrapper of a handle takes for none."""
    default, device = torch.cuda.default_stream(), torch.device("cuda", torch.cuda.current_device())
    x, a, b, ranks, scales, ids, base = make_lora(7, 9, 64, 4104, 2, 8, F16, F32)
    lora = hqb.LoraSet(a, b, ranks, scales, max_tokens=0)
    with torch.cuda.stream(torch.cuda.Stream() if aside else default):
        spaces = hqb.StreamWorkspaces(device, lambda size: size)
        ws = spaces.take(1 << 24, 0)
        out = lora.apply(x, ids, base=base, stream=default)
    places = [(ws.ptr(), (1 << 24,), torch.uint8), (out.data_ptr(), out.shape, F32)]
    del spaces, ws, out
    for place, shape, kind in places:
        assert torch.empty(shape, dtype=kind, device="cuda").data_ptr() == place


# ---- errors that calls without a workspace report -------------------------------------------------


def test_errors_of_implicit_workspaces_can_be_read():
    import harpq_b200_ops

    ops, clear = torch.ops.harpq_b200, {"cache_append": 0, "tree_attention": 0, "lora": 0}
    harpq_b200_ops.serving_errors(reset=True)
    x, a, b, ranks, scales, ids, base = make_lora(7, 400, 256, 64, 2, 16, F16, F16, full=True)
    s = hqb.LoraSet(a, b, ranks, scales)
    s.apply(x, ids, base=base)
    ops.lora(x, a, b, ids, ranks, scales, base)
    assert s.error_flags() == 0 and harpq_b200_ops.serving_errors() == clear
    ids[4] = 9
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        s.apply(x, ids, base=base)
        ops.lora(x, a, b, ids, ranks, scales, base)
    assert s.error_flags(reset=True) == hqb.DEVERR_INDEX and s.error_flags() == 0
    assert harpq_b200_ops.serving_errors("cuda:0", reset=True) == {**clear, "lora": hqb.DEVERR_INDEX}
    t = make_attention(12, [40, 40], [2, 2], 4, 1, 64, 16, F16)
    ops.cache_append(t["kc"], t["vc"], t["k"], t["v"], ints([3, 10 ** 6, 4, 5]))
    ops.tree_attention(t["q"], t["k"], t["v"], t["kc"], t["vc"], t["tables"], ints([-1, 40]), ints([0, 2, 4]), t["mask"], 2, 40)
    assert harpq_b200_ops.serving_errors(reset=True) == {"cache_append": hqb.DEVERR_PAGES, "tree_attention": hqb.DEVERR_INDEX, "lora": 0}
    assert harpq_b200_ops.serving_errors() == clear


def test_errors_of_a_replay_can_be_read():
    x, a, b, ranks, scales, ids, base = make_lora(7, 40, 256, 64, 2, 16, F16, F16, full=True)
    s = hqb.LoraSet(a, b, ranks, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.apply(x, ids, base=base)
    ids[4] = 9
    graph.replay()
    assert s.error_flags() == hqb.DEVERR_INDEX
    ids[4] = 0
    graph.replay()  # clears the word first
    assert s.error_flags() == 0


# ---- refusals ------------------------------------------------------------------------------------


def test_results_that_overlap_are_refused():
    s = make_attention(12, [40], [3], 4, 2, 64, 16, F16)
    attend = hqb.TreeAttention(hqb.PagedCache(s["kc"], s["vc"]), 4, 1, 3, 3, 40)
    args = (s["q"], s["k"], s["v"], s["tables"], ints([40]), ints([0, 3]), s["mask"])
    for out in (torch.empty(1, 4, 64, dtype=F16, device="cuda").expand(3, 4, 64),
                torch.empty(3, 1, 64, dtype=F16, device="cuda").expand(3, 4, 64)):
        with pytest.raises(ValueError, match="share their place"):
            attend(*args, out=out)
    attend(*args, out=torch.empty(4, 3, 64, dtype=F16, device="cuda").transpose(0, 1))
    x, a, b, ranks, scales, ids, base = make_lora(7, 4, 64, 32, 2, 8, F16, F16)
    store = torch.zeros(6, 32, dtype=F16, device="cuda")
    lora = hqb.LoraSet(a, b, ranks, scales)
    with pytest.raises(ValueError, match="overlap"):
        lora.apply(x, ids, base=store[:4], out=store[1:5])
    lora.apply(x, ids, base=store[:4], out=store[:4])
    lora.apply(x[:2], ids[:2], base=store[:2], out=store[2:4])
