"""GPU: cases at the edges of the serving operators' contracts, each against the plain forms of
test_gpu_serving.py (whose tolerances hold here too)."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import harpq_b200 as hqb  # noqa: E402
from test_gpu_serving import BF16, F16, U, ints, make_attention, make_lora, plan_reference  # noqa: E402


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
