"""GPU: cases at the edges of the serving operators' contracts, each against the plain forms of
test_gpu_serving.py (whose tolerances hold here too)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import harpq_b200 as hqb  # noqa: E402
from test_gpu_serving import BF16, F16, ints, make_lora, plan_reference  # noqa: E402


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


# ---- memory that callers bring --------------------------------------------------------------


def test_workspaces_in_host_memory_are_refused():
    k = torch.zeros(4, 16, 2, 64, dtype=F16, device="cuda")
    with pytest.raises(ValueError):
        hqb.TreeAttention(hqb.PagedCache(k, k), 4, 1, 3, 3, 10, workspace=lambda need: hqb.Workspace(need, "cpu"))
    x, a, b, ranks, scales, ids, base = make_lora(1, 5, 64, 32, 2, 8, BF16, BF16)
    with pytest.raises(ValueError):
        hqb.LoraSet(a, b, ranks, scales).apply(x, ids, base=base, workspace=hqb.Workspace(1 << 20, "cpu"))
