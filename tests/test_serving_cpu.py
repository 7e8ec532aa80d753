"""CPU: host-side checks of the serving operators' C entry points (nothing is enqueued for a refused
call) and the fake kernels of their PyTorch operators."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

import harpq_b200 as hqb  # noqa: E402
import harpq_b200_ops  # noqa: E402, F401

AT = ctypes.addressof
INVALID, UNSUPPORTED = hqb.HQB_ERR_INVALID, hqb.HQB_ERR_UNSUPPORTED


def changed(struct, **fields):
    other = type(struct).from_buffer_copy(struct)
    for name, value in fields.items():
        setattr(other, name, value)
    return other


def a_plan():
    return hqb.PagePlanC(requests=4, page_size=16, num_pages=8, table_stride=2, token_capacity=4, free_count=3,
                         context_lens=256, new_lens=256, held=256, free_pages=256, free_head=512, tables=256, starts=256,
                         held_out=1024, free_head_out=1024)


@pytest.mark.parametrize("fields", [
    dict(starts=None), dict(context_lens=None), dict(new_lens=None), dict(page_size=0), dict(table_stride=0),
    dict(num_pages=0), dict(free_head=None), dict(free_pages=None), dict(held_out=256), dict(free_head_out=512),
    dict(free_head_out=512, free_head=512), dict(mask=256, mask_words=1), dict(mask=256, parents=256, mask_words=0),
    dict(mask=256, parents=256, mask_words=9), dict(tables=None, slots=256), dict(tables=None, free_head_out=1024),
    dict(requests=0x7FFFFFFF), dict(token_capacity=0x80000000), dict(num_pages=0x10000000)])
def test_page_plan_refusals(fields):
    assert hqb.lib().hqb_page_plan(AT(changed(a_plan(), **fields)), None) == INVALID
    assert hqb.lib().hqb_page_plan(None, None) == INVALID


def a_cache():
    return hqb.PagedCacheC(256, 256, 16 * 2 * 64, 2 * 64, 64, hqb.F16, 2, 64, 16, 8, 0)


BAD_CACHES = [dict(dtype=hqb.F32), dict(dtype=7), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0), dict(num_pages=0),
              dict(num_pages=0x8000000)]


@pytest.mark.parametrize("fields", [*BAD_CACHES, dict(k=None), dict(v=None)])
def test_cache_append_refuses_caches(fields):
    c = changed(a_cache(), **fields)
    assert hqb.lib().hqb_cache_append(AT(c), 256, 256, hqb.F16, 128, 64, 4, None, 256, 4, None, None) == INVALID


@pytest.mark.parametrize("k,v,dtype,source,slots,count", [
    (None, 256, 1, 4, 256, 4), (256, None, 1, 4, 256, 4), (256, 256, 5, 4, 256, 4), (256, 256, 1, 4, None, 4),
    (256, 256, 1, 0x80000000, 256, 4), (256, 256, 1, 4, 256, 0x80000000)])
def test_cache_append_refuses_rows(k, v, dtype, source, slots, count):
    c = a_cache()
    assert hqb.lib().hqb_cache_append(AT(c), k, v, dtype, 128, 64, source, None, slots, count, None, None) == INVALID


def an_attention():
    return hqb.AttentionC(requests=2, tokens=6, max_new=3, max_context=100, q_heads=4, table_stride=7, mask_words=1, scale=0.1,
                          starts=256, context_lens=256, tables=256, mask=256, q=256, k=256, v=256, out=256, lse=None,
                          q_token_stride=256, q_head_stride=64, kv_token_stride=128, kv_head_stride=64, out_token_stride=256,
                          out_head_stride=64)


@pytest.mark.parametrize("fields", [
    dict(max_new=0), dict(max_new=257), dict(max_new=33), dict(q_heads=0), dict(q_heads=5), dict(mask_words=0), dict(starts=None),
    dict(context_lens=None), dict(tables=None), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
    dict(tokens=0x80000000), dict(requests=0x800000), dict(max_context=0x80000000)])
def test_tree_attention_refusals(fields):
    c, a = a_cache(), changed(an_attention(), **fields)
    assert hqb.lib().hqb_tree_attention(AT(c), AT(a), 256, 1 << 40, None) == INVALID


@pytest.mark.parametrize("fields", [*BAD_CACHES, dict(k=None), dict(head_dim=257)])
def test_tree_attention_refuses_caches(fields):
    c, a = changed(a_cache(), **fields), an_attention()
    assert hqb.lib().hqb_tree_attention(AT(c), AT(a), 256, 1 << 40, None) == INVALID
    if "k" not in fields:
        assert hqb.lib().hqb_tree_attention_workspace_bytes(AT(c), AT(a), 0) == 0


def a_set():
    return hqb.LoraSetC(256, 256, None, None, 128, 64, 3, 16, hqb.F16, 0)


@pytest.mark.parametrize("fields", [dict(rows=0), dict(cols=0), dict(adapters=0), dict(max_rank=0), dict(max_rank=129),
                                    dict(dtype=hqb.F32), dict(rows=1 << 31), dict(cols=1 << 31)])
def test_lora_refuses_sets(fields):
    s = changed(a_set(), **fields)
    assert hqb.lib().hqb_lora(AT(s), 256, 64, 256, 2, None, 0, 256, hqb.F16, 128, 256, 1 << 40, None) == INVALID
    assert hqb.lib().hqb_lora_workspace_bytes(AT(s), 2, 0) == 0


def test_lora_refuses_rows():
    L, s = hqb.lib(), a_set()

    def call(x=256, xs=64, ids=256, base=None, bs=0, y=512, kind=hqb.F16, ys=128, ws=256, size=1 << 40, s=s):
        return L.hqb_lora(AT(s), x, xs, ids, 2, base, bs, y, kind, ys, ws, size, None)

    for bad in (dict(x=None), dict(ids=None), dict(y=None), dict(xs=63), dict(ys=127), dict(base=256, bs=127), dict(kind=hqb.BF16),
                dict(base=512, bs=136), dict(ws=None), dict(ws=300), dict(size=255)):
        assert call(**bad) == INVALID, bad
    assert call(s=changed(s, a=None)) == INVALID and call(s=changed(s, b=None)) == INVALID
    assert call(s=changed(s, adapters=16384)) == UNSUPPORTED


def test_lora_workspace_never_shrinks_with_tokens():
    """A workspace made for many tokens serves fewer."""
    L = hqb.lib()
    for adapters in (1, 3, 40, 700):
        for rank in (8, 32, 64, 128):
            s = changed(a_set(), adapters=adapters, max_rank=rank, cols=8192)
            sizes = [L.hqb_lora_workspace_bytes(AT(s), t, 0) for t in range(1, 3000, 7)]
            assert sizes == sorted(sizes) and sizes[0] >= 256


def test_struct_sizes_match_the_header():
    assert [ctypes.sizeof(t) for t in (hqb.PagedCacheC, hqb.PagePlanC, hqb.AttentionC, hqb.LoraSetC)] == [64, 152, 152, 64]


def test_operators_trace_with_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = torch.empty(5, 8, 64, dtype=torch.float16, device="cuda"), torch.empty(5, 2, 64, dtype=torch.float16, device="cuda")
        cache = torch.empty(9, 16, 2, 64, dtype=torch.float16, device="cuda")
        i = torch.empty(2, dtype=torch.int32, device="cuda")
        out = torch.ops.harpq_b200.tree_attention(q, k, k, cache, cache, i[None], i, i, None, 3, 100)
        assert out.shape == q.shape and out.dtype == q.dtype
        torch.ops.harpq_b200.cache_append(cache, cache.clone(), k, k, i)
        a, b = torch.empty(3, 8, 64, dtype=torch.float16, device="cuda"), torch.empty(3, 40, 8, dtype=torch.float16, device="cuda")
        y = torch.ops.harpq_b200.lora(torch.empty(4, 64, dtype=torch.float16, device="cuda"), a, b, i, None, None, None, torch.float32)
        assert y.shape == (4, 40) and y.dtype == torch.float32


def test_operators_have_no_cpu_fallback():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.harpq_b200.lora(x, torch.zeros(1, 8, 64, dtype=torch.float16), torch.zeros(1, 4, 8, dtype=torch.float16),
                                  torch.zeros(2, dtype=torch.int32))


def test_host_memory_is_refused():
    """Before any address of it reaches a kernel."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    cache = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        hqb.PagedCache(cache, cache)
    with pytest.raises(ValueError):
        hqb.LoraSet(torch.zeros(2, 8, 64, dtype=torch.float16), torch.zeros(2, 32, 8, dtype=torch.float16), max_tokens=0)
    with pytest.raises(ValueError):
        hqb.PagePlan(1, 1, 16, 8, device="cpu")
    with FakeTensorMode():
        k = torch.empty(4, 16, 2, 64, dtype=torch.float16, device="cuda:0")
        for flags in (torch.empty(1, dtype=torch.int32), torch.empty(1, device="cuda:0"), torch.empty(0, dtype=torch.int32, device="cuda:0"),
                      torch.empty(1, dtype=torch.int32, device="cuda:1")):
            with pytest.raises(ValueError):
                hqb.PagedCache(k, k, flags)


def test_the_default_stream_is_never_captured():
    number = ctypes.c_uint64(7)
    assert hqb.lib().hqb_stream_capture(None, ctypes.byref(number)) == 0 and number.value == 0
    assert hqb.lib().hqb_stream_capture(None, None) == INVALID


@pytest.mark.parametrize("name", ["hqb_page.cu", "hqb_attention.cuh", "hqb_attention.cu", "hqb_attention_tmem.cu", "hqb_lora.cu",
                                  "hqb_serve.cuh"])
def test_programmatic_dependents_read_by_plain_loads(name):
    """These kernels start while the one before them may still write their inputs: the read-only path is
    for data that does not change while a kernel runs, and its loads may move above the wait."""
    source = (hqb.PKG / "csrc" / name).read_text()
    assert "__ldg" not in source and "ld.global.nc" not in source


def test_dependents_start_after_tensor_memory_is_taken():
    """A programmatic dependent that shares an SM and takes tensor memory before its predecessor's CTA has
    would wait for that CTA, which waits for the memory."""
    found = 0
    for path in sorted((hqb.PKG / "csrc").glob("*.cu")):
        for kernel in path.read_text().split("__global__")[1:]:
            if "tmem_alloc(" in kernel:
                found += 1
                assert kernel.index("tmem_alloc(") < kernel.index("griddep_launch_dependents("), path.name
    assert found == 2


@pytest.mark.parametrize("rank", [1, 5, 27, 63, 121])
def test_lora_workspace_of_odd_ranks_never_shrinks_with_tokens(rank):
    """The laid-out rows of b join it with the token count."""
    for adapters in (1, 9, 40, 200, 700):
        s = changed(a_set(), adapters=adapters, max_rank=rank, cols=8192)
        sizes = [hqb.lib().hqb_lora_workspace_bytes(AT(s), t, 0) for t in [*range(1, 600), *range(600, 3000, 7)]]
        assert sizes == sorted(sizes) and sizes[0] >= 256
        pitch = -(-rank // 8) * 8
        assert sizes[-1] >= adapters * 128 * pitch * 2  # laid out by then
