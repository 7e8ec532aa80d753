"""PyTorch operators over the C ABI: ``torch.ops.harpq_b200.gemv`` and the serving operators
``cache_append``, ``tree_attention`` and ``lora`` (at the end of this file).

The reference lists a PyTorch custom-op wrapper over its native GEMV as planned work
(docs/RESEARCH_PLAN.md:106-107); it has no implementation to mirror.  This module
registers one through ``torch.library`` so the GEMV can sit inside PyTorch programs
(eager, CUDA graphs, and tracing through its fake kernel):

    import harpq_b200_ops  # registers the operator
    y = torch.ops.harpq_b200.gemv(x, planes, rows, cols, prefix, bias, torch.float16)

Arguments:
    x        [batch, cols] FP16 or FP32 CUDA tensor, batch 1..16
    planes   the matrix's stage planes in stage order (uint8 CUDA tensors of
             hqb_plane_bytes each, e.g. ``PlaneMatrix.planes``)
    rows, cols   the matrix's original shape
    prefix   stages to evaluate, 0..len(planes)
    bias     optional [rows] FP16 or FP32 CUDA tensor
    out_dtype    torch.float16 or torch.float32

It returns a new [batch, rows] tensor, computed by ``hqb_gemv`` on the current stream of
x's device: the same kernels and the same bits as ``PlaneMatrix.gemv``.  The operator has
only a CUDA kernel (a CPU tensor raises: there is no CPU fallback).  Its scratch workspace
is cached per (device, stream, matrix grid, batch, x dtype), so calls on different streams
never share one.
"""

import ctypes
from typing import List, Optional

import torch

import harpq_b200 as hqb

_WORKSPACES: dict = {}


def _plane_matrix(planes: List[torch.Tensor], rows: int, cols: int) -> "hqb.PlaneMatrixC":
    if not 1 <= len(planes) <= hqb.MAX_STAGES:
        raise ValueError(f"a plane matrix has 1..{hqb.MAX_STAGES} stage planes, got {len(planes)}")
    need = hqb.plane_bytes(hqb.geometry(rows, cols))
    for s, p in enumerate(planes):
        if p.dtype != torch.uint8 or not p.is_contiguous() or p.numel() < need:
            raise ValueError(f"plane {s} must be a contiguous uint8 tensor of at least {need} bytes")
    arr = (hqb.vp * hqb.MAX_STAGES)(*[p.data_ptr() for p in planes], *([None] * (hqb.MAX_STAGES - len(planes))))
    return hqb.PlaneMatrixC(rows, cols, -(-rows // hqb.TILE), -(-cols // hqb.TILE), len(planes), 0, arr)


def _workspace(m: "hqb.PlaneMatrixC", device: torch.device, stream: int, batch: int, x_dtype: int) -> "hqb.Workspace":
    key = (device.index, stream, m.grid_rows, m.grid_cols, m.stage_count, batch, x_dtype)
    ws = _WORKSPACES.get(key)
    if ws is None:
        nbytes = hqb.lib().hqb_workspace_bytes(ctypes.byref(m), batch, x_dtype, device.index)
        if nbytes == 0:
            raise ValueError("hqb_workspace_bytes rejected the matrix, batch or activation type")
        ws = _WORKSPACES[key] = hqb.Workspace(nbytes, device)
    return ws


@torch.library.custom_op("harpq_b200::gemv", mutates_args=(), device_types="cuda")
def gemv(x: torch.Tensor, planes: List[torch.Tensor], rows: int, cols: int, prefix: int,
         bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """y[b, r] = Σ_c x[b, c]·W_prefix[r, c] (+ bias[r]) over the plane matrix `planes`."""
    if x.dim() != 2 or x.shape[1] != cols:
        raise ValueError(f"x must be [batch, {cols}]")
    if out_dtype not in (torch.float16, torch.float32):
        raise ValueError("out_dtype must be torch.float16 or torch.float32")
    if any(p.device != x.device for p in planes) or (bias is not None and bias.device != x.device):
        raise ValueError("x, planes and bias must be on one device")
    x = x.contiguous()
    m = _plane_matrix(planes, rows, cols)
    xd = hqb._dtype_code(x)
    with torch.cuda.device(x.device):  # the library launches on the current device
        stream = torch.cuda.current_stream(x.device).cuda_stream
        ws = _workspace(m, x.device, stream, x.shape[0], xd)
        y = torch.empty(x.shape[0], rows, dtype=out_dtype, device=x.device)
        if bias is not None:
            bias = bias.contiguous()
        status = hqb.lib().hqb_gemv(ctypes.byref(m), prefix, x.data_ptr(), xd, x.shape[0],
                                    None if bias is None else bias.data_ptr(),
                                    hqb.F32 if bias is None else hqb._dtype_code(bias), y.data_ptr(),
                                    hqb._dtype_code(y), ws.ptr(), ws.nbytes, stream)
    hqb.check(status, "hqb_gemv")
    return y


@gemv.register_fake
def _gemv_fake(x, planes, rows, cols, prefix, bias=None, out_dtype=torch.float16):
    torch._check(x.dim() == 2 and x.shape[1] == cols, lambda: f"x must be [batch, {cols}]")
    return x.new_empty((x.shape[0], rows), dtype=out_dtype)


# ---- serving operators -------------------------------------------------------------------
#
#   cache_append(k_cache, v_cache, k, v, slots, rows)          writes into the caches
#   tree_attention(q, k, v, k_cache, v_cache, tables, context_lens, starts, mask, max_new,
#                  max_context, scale)                         -> [tokens, q_heads, dim]
#   lora(x, a, b, ids, ranks, scales, base, out_dtype)         -> [tokens, rows]
#
# The same calls and the same bits as PagedCache.append, TreeAttention and LoraSet.apply, whose
# arguments they share, without a handle to keep.  Workspaces are kept per stream and capture
# (harpq_b200.StreamWorkspaces); serving_errors() reads what their calls reported.

_SERVING_WORKSPACES: dict = {}


def _serving_workspace(kind: str, device: torch.device, stream: int, need: int) -> "hqb.Workspace":
    key = (kind, device.index)
    if key not in _SERVING_WORKSPACES:
        _SERVING_WORKSPACES[key] = hqb.StreamWorkspaces(device, lambda size: size)
    return _SERVING_WORKSPACES[key].take(need, stream)


def serving_errors(device: Optional[torch.device] = None, reset: bool = False) -> dict:
    """HQB_DEVERR_* bits of the serving operators' calls on a device (None: the current one), by operator;
    waits for the device."""
    index = torch.cuda.current_device() if device is None else hqb._device_index(torch.device(device))
    kinds = {"cache": "cache_append", "attention": "tree_attention", "lora": "lora"}
    return {name: ws.error_flags(reset) if (ws := _SERVING_WORKSPACES.get((kind, index))) is not None else 0
            for kind, name in kinds.items()}


def _serving_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, stream: int) -> "hqb.PagedCache":
    return hqb.PagedCache(k_cache, v_cache, _serving_workspace("cache", k_cache.device, stream, 256).buf.view(torch.int32)[:1])


@torch.library.custom_op("harpq_b200::cache_append", mutates_args=("k_cache", "v_cache"), device_types="cuda")
def cache_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                 rows: Optional[torch.Tensor] = None) -> None:
    """k_cache, v_cache[slots[i]] = k, v[rows[i]] (rows None: row i); negative slots and rows are skipped."""
    stream = torch.cuda.current_stream(k.device).cuda_stream
    _serving_cache(k_cache, v_cache, stream).append(k, v, slots, rows=rows)


@cache_append.register_fake
def _cache_append_fake(k_cache, v_cache, k, v, slots, rows=None):
    torch._check(k.dim() == 3 and k.shape == v.shape, lambda: "k and v must be [tokens, heads, dim]")
    torch._check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, lambda: "caches must be [pages, page_size, heads, dim]")


@torch.library.custom_op("harpq_b200::tree_attention", mutates_args=(), device_types="cuda")
def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   tables: torch.Tensor, context_lens: torch.Tensor, starts: torch.Tensor,
                   mask: Optional[torch.Tensor], max_new: int, max_context: int,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of each request's drafted nodes over its cached context and the nodes its mask shows
    (rows of no request are not written)."""
    if q.shape[0] == 0:
        return q.new_empty(q.shape)
    stream = torch.cuda.current_stream(q.device).cuda_stream
    attend = hqb.TreeAttention(_serving_cache(k_cache, v_cache, stream), q.shape[1], context_lens.numel(), q.shape[0], max_new,
                               max_context, workspace=lambda need: _serving_workspace("attention", q.device, stream, need))
    return attend(q, k, v, tables, context_lens, starts, mask, scale=scale)


@tree_attention.register_fake
def _tree_attention_fake(q, k, v, k_cache, v_cache, tables, context_lens, starts, mask, max_new, max_context, scale=None):
    torch._check(q.dim() == 3 and k.dim() == 3 and k.shape == v.shape and q.shape[0] == k.shape[0],
                 lambda: "q, k and v must be [tokens, heads, dim]")
    return q.new_empty(q.shape)


@torch.library.custom_op("harpq_b200::lora", mutates_args=(), device_types="cuda")
def lora(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, ranks: Optional[torch.Tensor] = None,
         scales: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None,
         out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """base + scales[i] * b[i] (a[i] x) per token, i = ids[token] (negative: base alone)."""
    adapters = hqb.LoraSet(a, b, ranks, scales, max_tokens=0)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    ws = _serving_workspace("lora", x.device, stream, adapters.workspace_bytes(x.shape[0]))
    return adapters.apply(x, ids, base=base, y_dtype=out_dtype, workspace=ws)


@lora.register_fake
def _lora_fake(x, a, b, ids, ranks=None, scales=None, base=None, out_dtype=None):
    torch._check(x.dim() == 2 and a.dim() == 3 and x.shape[1] == a.shape[2], lambda: "x must be [tokens, cols]")
    kind = out_dtype or (base.dtype if base is not None else x.dtype)
    return x.new_empty((x.shape[0], b.shape[1]), dtype=kind)
