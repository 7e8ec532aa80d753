"""Python binding of the C ABI in include/harpq_b200.h (ctypes over libharpq_b200.so).

Device memory is held in torch tensors (allocation, streams and events only); every
computation runs in the library's sm_100a kernels.  There is no fallback: importing
this module without the built library, or calling it without a CUDA device, raises.

    import harpq_b200 as hqb
    m = hqb.PlaneMatrix.from_stages(rows, cols, codes, fp16_scale_bits)  # repack on device
    y = m.gemv(x, prefix=2)                        # x: [batch, cols] FP16/FP32 CUDA tensor
    w = m.decode(prefix=2)                         # dense FP32, bit-exact decode
"""

from __future__ import annotations

import contextlib
import ctypes
import importlib.util
from pathlib import Path
from typing import Sequence

import torch

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "lib" / "libharpq_b200.so"
BIND_PATH = PKG / "lib" / "harpq_b200_bind.so"

F32, F16, BF16 = 0, 1, 2  # BF16: serving operators only
FLAG_PDL, FLAG_SIMT, FLAG_RING, FLAG_TCGEN05, FLAG_STREAMK, FLAG_ROWBLOCK = 1, 2, 4, 8, 16, 32
FLAG_F16MMA = 64  # keep the GEMV kernels on FP16-fragment MMAs (no int8 activation limbs)
FLAG_BULK = 128  # bulk-copy kernel (batch <= 2, raw x): default for large layers, forced by this flag
RAW_GENERIC, RAW_REQUIRE_FAST = 1, 2  # hqb_raw_gemv_ex: per-element FMA kernel / int8 raw-layout kernel only
I8_LIMBS = 4
TILE = 128
RECORD_BYTES = 4352
MAX_STAGES = 4
MAX_BATCH = 16
DEVERR_SCALE, DEVERR_DEPTH, DEVERR_TIMEOUT, DEVERR_LAUNCH, DEVERR_PAGES, DEVERR_INDEX = 1, 2, 4, 8, 16, 32
MAX_NODES, MAX_HEAD_DIM, MAX_RANK = 256, 256, 128
HQB_OK, HQB_ERR_INVALID, HQB_ERR_UNSUPPORTED = 0, 1, 801
NOALLOC_SCRATCH_BYTES = 4 << 20
ERR_SCRATCH_LIMIT = 20001

u64, u32, i32, vp = ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int, ctypes.c_void_p


class Geometry(ctypes.Structure):
    _fields_ = [(n, u64) for n in ("original_rows", "original_columns", "padded_rows", "padded_columns",
                                   "tile_rows", "tile_columns", "group_size")]


class RawStage(ctypes.Structure):
    _fields_ = [("packed_codes", vp), ("packed_code_bytes", u64), ("scale_fp16_bits", vp), ("scale_count", u64)]


class CopyC(ctypes.Structure):
    _fields_ = [("dst", ctypes.c_void_p), ("src", ctypes.c_void_p), ("bytes", ctypes.c_uint64)]


class RawStageF32(ctypes.Structure):
    _fields_ = [("packed_codes", vp), ("packed_code_bytes", u64), ("scales", vp), ("scale_count", u64)]


class PlaneMatrixC(ctypes.Structure):
    _fields_ = [("rows", u64), ("cols", u64), ("grid_rows", u32), ("grid_cols", u32), ("stage_count", u32),
                ("reserved", u32), ("planes", vp * MAX_STAGES)]


class GemvCallC(ctypes.Structure):
    _fields_ = [("m", vp), ("prefix", u32), ("x_dtype", i32), ("depth", vp), ("depth_plan", vp), ("x", vp),
                ("batch", u32), ("x_prepared", i32), ("bias", vp), ("bias_dtype", i32), ("y_dtype", i32), ("y", vp),
                ("flags", u32), ("reserved", u32)]


class LaunchInfo(ctypes.Structure):
    _fields_ = [("launches", u32), ("int8_limbs", u32), ("grid", u32), ("block", u32), ("smem_bytes", u32),
                ("reserved", u32), ("kernel", ctypes.c_char * 40)]


MAX_PEERS = 8


class GatherC(ctypes.Structure):
    _fields_ = [("world", u32), ("rank", u32), ("slot_rows", u64), ("peer_y", vp * MAX_PEERS),
                ("peer_flags", vp * MAX_PEERS)]


class PagedCacheC(ctypes.Structure):
    _fields_ = [("k", vp), ("v", vp), ("page_stride", u64), ("token_stride", u64), ("head_stride", u64),
                ("dtype", i32), ("kv_heads", u32), ("head_dim", u32), ("page_size", u32), ("num_pages", u32),
                ("reserved", u32)]


class PagePlanC(ctypes.Structure):
    _fields_ = [*[(n, u32) for n in ("requests", "page_size", "num_pages", "table_stride", "token_capacity",
                                     "free_count", "mask_words", "parent_count")],
                *[(n, vp) for n in ("context_lens", "new_lens", "held", "free_pages", "free_head", "parents", "tables",
                                    "starts", "token_request", "positions", "slots", "held_out", "free_head_out",
                                    "mask", "flags")]]


class AttentionC(ctypes.Structure):
    _fields_ = [*[(n, u32) for n in ("requests", "tokens", "max_new", "max_context", "q_heads", "table_stride",
                                     "mask_words")], ("scale", ctypes.c_float),
                *[(n, vp) for n in ("starts", "context_lens", "tables", "mask", "q", "k", "v", "out", "lse")],
                *[(n, u64) for n in ("q_token_stride", "q_head_stride", "kv_token_stride", "kv_head_stride",
                                     "out_token_stride", "out_head_stride")]]


class LoraSetC(ctypes.Structure):
    _fields_ = [("a", vp), ("b", vp), ("ranks", vp), ("scales", vp), ("rows", u64), ("cols", u64), ("adapters", u32),
                ("max_rank", u32), ("dtype", i32), ("reserved", u32)]


EXPORTS = {
    "hqb_version": (i32, []),
    "hqb_status_string": (ctypes.c_char_p, [i32]),
    "hqb_plane_bytes": (u64, [ctypes.POINTER(Geometry)]),
    "hqb_repack_stage": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStage), vp, vp, vp]),
    "hqb_xfrag_bytes": (u64, [u64, u32, i32]),
    "hqb_prepare_x": (i32, [vp, i32, u64, u32, vp, vp]),
    "hqb_workspace_bytes": (u64, [ctypes.POINTER(PlaneMatrixC), u32, i32, i32]),
    "hqb_workspace_init": (i32, [vp, u64, vp]),
    "hqb_workspace_error": (i32, [vp, ctypes.POINTER(i32), vp]),
    "hqb_stream_capture": (i32, [vp, ctypes.POINTER(u64)]),
    "hqb_depth_plan_bytes": (u64, [u32]),
    "hqb_depth_plan": (i32, [vp, u32, u32, u32, vp, vp, vp]),
    "hqb_gemv": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, i32, u32, vp, i32, vp, i32, vp, u64, vp]),
    "hqb_gemv_mixed": (i32, [ctypes.POINTER(PlaneMatrixC), vp, vp, vp, i32, u32, vp, i32, vp, i32, vp, u64, vp]),
    "hqb_gemv_ex": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, vp, vp, i32, u32, i32, vp, i32, vp, i32, vp, u64,
                          u32, vp]),
    "hqb_gemv_noalloc": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, i32, u32, vp, i32, vp, i32, vp]),
    "hqb_gemv_batch": (i32, [ctypes.POINTER(GemvCallC), u32, vp, u64, vp]),
    "hqb_step_create": (i32, [ctypes.POINTER(GemvCallC), u32, vp, u64, ctypes.POINTER(vp)]),
    "hqb_step_create_grouped": (i32, [ctypes.POINTER(GemvCallC), u32, vp, u64, ctypes.POINTER(vp)]),
    "hqb_step_create_io": (i32, [ctypes.POINTER(GemvCallC), u32, vp, u64, ctypes.POINTER(CopyC), u32,
                                 ctypes.POINTER(CopyC), u32, i32, ctypes.POINTER(vp)]),
    "hqb_gemv_grouped": (i32, [ctypes.POINTER(GemvCallC), u32, vp, u64, vp]),
    "hqb_step_launch": (i32, [vp, vp]),
    "hqb_step_destroy": (i32, [vp]),
    "hqb_gemv_query": (i32, [ctypes.POINTER(PlaneMatrixC), u32, i32, i32, u32, i32, u32, ctypes.POINTER(LaunchInfo)]),
    "hqb_peer_alloc": (i32, [u64, ctypes.POINTER(vp), vp]),
    "hqb_peer_open": (i32, [vp, ctypes.POINTER(vp)]),
    "hqb_peer_close": (i32, [vp]),
    "hqb_peer_free": (i32, [vp]),
    "hqb_gemv_gather": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, i32, u32, vp, i32, i32, ctypes.POINTER(GatherC),
                              vp, u64, u32, vp]),
    "hqb_gather_wait": (i32, [vp, u32, vp, vp, vp]),
    "hqb_gather_wait_ex": (i32, [vp, u32, vp, vp, u64, vp]),
    "hqb_gemv_noalloc_flags": (i32, [ctypes.POINTER(i32), i32, vp]),
    "hqb_gemv_noalloc_reset": (i32, [vp]),
    "hqb_gemv_noalloc_scratch": (i32, [ctypes.POINTER(vp)]),
    "hqb_decode_planes": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, vp, u64, vp]),
    "hqb_prefill_workspace_bytes": (u64, [ctypes.POINTER(PlaneMatrixC)]),
    "hqb_prefill_gemm": (i32, [ctypes.POINTER(PlaneMatrixC), u32, vp, i32, u32, vp, i32, vp, i32, vp, u64, vp]),
    "hqb_page_plan": (i32, [vp, vp]),
    "hqb_cache_append": (i32, [vp, vp, vp, i32, u64, u64, u32, vp, vp, u32, vp, vp]),
    "hqb_tree_attention_workspace_bytes": (u64, [vp, vp, i32]),
    "hqb_tree_attention": (i32, [vp, vp, vp, u64, vp]),
    "hqb_lora_workspace_bytes": (u64, [vp, u32, i32]),
    "hqb_lora": (i32, [vp, vp, u64, vp, u32, vp, u64, vp, i32, u64, vp, u64, vp]),
    "hqb_raw_gemv": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStage), u32, u32, vp, u64, vp, u64, vp, u64,
                           vp]),
    "hqb_raw_gemv_ex": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStage), u32, u32, vp, u64, vp, u64, vp,
                              u64, u32, vp]),
    "hqb_raw_dequantize_stage": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStageF32), u32, u32, vp, vp]),
    "hqb_raw_dequantize_prefix": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStageF32), u32, u32, vp, vp]),
    "hqb_raw_linear_ordered": (i32, [ctypes.POINTER(Geometry), ctypes.POINTER(RawStageF32), u32, u32, vp, u64, vp,
                                     vp, vp]),
}

_lib = None


class HQBError(RuntimeError):
    def __init__(self, status: int, what: str):
        msg = lib().hqb_status_string(status).decode() if _lib is not None else str(status)
        super().__init__(f"{what}: status {status} ({msg})")
        self.status = status


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(f"{LIB_PATH} is missing: build it with __graft_entry__.build()")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in EXPORTS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


_bind_module = None


def bind():
    """The CPython module of the serving operators' calls (csrc/hqb_bind.cpp)."""
    global _bind_module
    if _bind_module is None:
        lib()
        if not BIND_PATH.exists():
            raise ImportError(f"{BIND_PATH} is missing: build it with __graft_entry__.build()")
        spec = importlib.util.spec_from_file_location("harpq_b200_bind", str(BIND_PATH))
        _bind_module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_bind_module)
    return _bind_module


def check(status: int, what: str) -> None:
    if status != 0:
        raise HQBError(status, what)


def _stream(stream) -> int | None:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float16:
        return F16
    if t.dtype == torch.float32:
        return F32
    raise TypeError(f"unsupported dtype {t.dtype}; use float16 or float32")


def geometry(rows: int, cols: int, tile: Sequence[int] = (TILE, TILE), group: int = TILE) -> Geometry:
    pr = -(-rows // tile[0]) * tile[0]
    pc = -(-cols // tile[1]) * tile[1]
    return Geometry(rows, cols, pr, pc, tile[0], tile[1], group)


def plane_bytes(g: Geometry) -> int:
    return lib().hqb_plane_bytes(ctypes.byref(g))


def xfrag_bytes(cols: int, batch: int, x_dtype: int) -> int:
    return lib().hqb_xfrag_bytes(cols, batch, x_dtype)


def prepare_x(x: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Prepared activations for hqb_gemv_ex(x_prepared=1); shareable across matrices."""
    x = x.contiguous()
    batch, cols = x.shape
    n = xfrag_bytes(cols, batch, _dtype_code(x))
    if n == 0:
        raise ValueError("invalid activation shape/dtype")
    if out is None:
        out = torch.empty(n, dtype=torch.uint8, device=x.device)
    check(lib().hqb_prepare_x(_ptr(x), _dtype_code(x), cols, batch, _ptr(out), _stream(stream)), "hqb_prepare_x")
    return out


class Workspace:
    """Caller-owned scratch of launches, cleared once at allocation: as much as a GEMV needs (all of
    it), or the first `clear` bytes (the serving operators: the error word's)."""

    def __init__(self, nbytes: int, device=None, stream=None, clear: int | None = None):
        if clear is None:
            self.buf = torch.zeros(max(256, nbytes), dtype=torch.uint8, device=device or "cuda")
        else:
            self.buf = torch.empty(max(256, nbytes), dtype=torch.uint8, device=device or "cuda")
            self.buf[:clear].zero_()
        self.nbytes = self.buf.numel()

    def ptr(self) -> int:
        return self.buf.data_ptr()

    def error_flags(self, stream=None) -> int:
        out = ctypes.c_int(0)
        check(lib().hqb_workspace_error(self.ptr(), ctypes.byref(out), _stream(stream)), "hqb_workspace_error")
        return out.value

    def reset(self, stream=None) -> None:
        check(lib().hqb_workspace_init(self.ptr(), self.nbytes, _stream(stream)), "hqb_workspace_init")


class DepthPlan:
    """Per-tile depth map (uint8 [grid_rows, grid_cols]) and its device schedule."""

    def __init__(self, depth: torch.Tensor, stage_count: int, stream=None):
        if depth.dtype != torch.uint8 or depth.dim() != 2:
            raise TypeError("depth must be a uint8 [grid_rows, grid_cols] tensor")
        self.depth = depth.contiguous()
        self.grid_rows, self.grid_cols = self.depth.shape
        self.plan = torch.empty(self.grid_rows + 1, dtype=torch.int32, device=depth.device)
        self.flags = torch.zeros(1, dtype=torch.int32, device=depth.device)
        check(lib().hqb_depth_plan(_ptr(self.depth), self.grid_rows, self.grid_cols, stage_count, _ptr(self.plan),
                                   _ptr(self.flags), _stream(stream)), "hqb_depth_plan")


class PlaneMatrix:
    """A device-resident progressive matrix in the plane layout (one buffer per stage)."""

    def __init__(self, rows: int, cols: int, device=None):
        self.rows, self.cols = rows, cols
        self.geom = geometry(rows, cols)
        self.grid_rows, self.grid_cols = -(-rows // TILE), -(-cols // TILE)
        self.device = torch.device(device or "cuda")
        self.planes: list[torch.Tensor] = []
        self.repack_flags = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._ws: dict = {}

    @property
    def stage_count(self) -> int:
        return len(self.planes)

    def add_stage(self, codes: torch.Tensor, fp16_scale_bits: torch.Tensor, stream=None) -> None:
        """Repack one newly resident stage (reference layout, on device) into a new plane."""
        if self.stage_count >= MAX_STAGES:
            raise ValueError("a progressive matrix holds at most four stages")
        codes = codes.contiguous()
        bits = fp16_scale_bits.contiguous()
        plane = torch.empty(plane_bytes(self.geom), dtype=torch.uint8, device=self.device)
        st = RawStage(codes.data_ptr(), codes.numel(), bits.data_ptr(), bits.numel())
        check(lib().hqb_repack_stage(ctypes.byref(self.geom), ctypes.byref(st), _ptr(plane), _ptr(self.repack_flags),
                                     _stream(stream)), "hqb_repack_stage")
        self.planes.append(plane)

    @classmethod
    def stack(cls, mats: Sequence["PlaneMatrix"]) -> "PlaneMatrix":
        """Row-stacked matrix of matrices with equal column counts.  Matrices that share
        their input (q|k|v, gate|up) then run as one GEMV launch.  Tile records are
        tile-row major, so stacking is concatenation of the plane buffers.  Member i's
        outputs are rows [row_offsets[i], row_offsets[i] + member_rows[i]) of the result
        (split_rows).  Offsets are multiples of 128: a member whose row count is not a
        multiple of 128 keeps its zero padding rows inside the stack.  The stack holds
        the stages that every member holds."""
        if not mats:
            raise ValueError("nothing to stack")
        cols = mats[0].cols
        if any(m.cols != cols for m in mats):
            raise ValueError("stacked matrices need equal column counts")
        offsets, r = [], 0
        for m in mats:
            offsets.append(r)
            r += m.grid_rows * TILE
        out = cls(offsets[-1] + mats[-1].rows, cols, device=mats[0].device)
        stages = min(m.stage_count for m in mats)
        out.planes = [torch.cat([m.planes[s] for m in mats]) for s in range(stages)]
        out.row_offsets = offsets
        out.member_rows = [m.rows for m in mats]
        return out

    def split_rows(self, y: torch.Tensor) -> list[torch.Tensor]:
        """Views of each member's outputs in a stacked matrix's result [..., rows]."""
        offsets = getattr(self, "row_offsets", [0])
        rows = getattr(self, "member_rows", [self.rows])
        return [y[..., o:o + n] for o, n in zip(offsets, rows)]

    @classmethod
    def from_stages(cls, rows: int, cols: int, codes: Sequence[torch.Tensor], fp16_scale_bits: Sequence[torch.Tensor],
                    stream=None) -> "PlaneMatrix":
        m = cls(rows, cols, device=codes[0].device)
        for c, s in zip(codes, fp16_scale_bits):
            m.add_stage(c, s, stream)
        return m

    def c_struct(self) -> PlaneMatrixC:
        """The C view of this matrix, built once per set of planes (kept while they are)."""
        key = tuple(p.data_ptr() for p in self.planes)
        cached = getattr(self, "_c", None)
        if cached is None or cached[0] != key:
            arr = (vp * MAX_STAGES)(*key, *([None] * (MAX_STAGES - len(key))))
            cached = (key, PlaneMatrixC(self.rows, self.cols, self.grid_rows, self.grid_cols, len(key), 0, arr))
            self._c = cached
        return cached[1]

    def workspace_bytes(self, batch: int, x_dtype: int = F16) -> int:
        dev = self.device.index if self.device.index is not None else torch.cuda.current_device()
        return lib().hqb_workspace_bytes(ctypes.byref(self.c_struct()), batch, x_dtype, dev)

    def workspace(self, batch: int, x_dtype: int = F16) -> Workspace:
        key = (batch, x_dtype)
        if key not in self._ws:
            self._ws[key] = Workspace(self.workspace_bytes(batch, x_dtype), self.device)
        return self._ws[key]

    def gemv(self, x: torch.Tensor, prefix: int | None = None, bias: torch.Tensor | None = None,
             out: torch.Tensor | None = None, y_dtype=torch.float16, depth: DepthPlan | None = None,
             workspace: Workspace | None = None, x_prepared: torch.Tensor | None = None, flags: int = 0,
             stream=None) -> torch.Tensor:
        """y[b, r] = Σ_c x[b, c]·W[r, c] (+ bias) at a uniform prefix or a depth map."""
        if x.dim() == 1:
            x = x.unsqueeze(0)
        x = x.contiguous()
        batch = x.shape[0]
        if x.shape[1] != self.cols:
            raise ValueError("x has the wrong number of columns")
        xd = _dtype_code(x)
        if out is None:
            out = torch.empty(batch, self.rows, dtype=y_dtype, device=self.device)
        ws = workspace or self.workspace(batch, xd)
        prefix = self.stage_count if prefix is None else prefix
        src = x if x_prepared is None else x_prepared
        status = lib().hqb_gemv_ex(ctypes.byref(self.c_struct()), prefix, None if depth is None else _ptr(depth.depth),
                                   None if depth is None else _ptr(depth.plan), _ptr(src), xd, batch,
                                   0 if x_prepared is None else 1, _ptr(bias),
                                   F32 if bias is None else _dtype_code(bias), _ptr(out), _dtype_code(out), ws.ptr(),
                                   ws.nbytes, flags, _stream(stream))
        check(status, "hqb_gemv_ex")
        return out

    def launch_info(self, batch: int, x_dtype: int, prefix: int, mixed: bool = False, flags: int = 0,
                    x_prepared: bool = False) -> LaunchInfo:
        """What one gemv() call enqueues on this device (the library's own choice, hqb_gemv_query)."""
        info = LaunchInfo()
        with torch.cuda.device(self.device):
            check(lib().hqb_gemv_query(ctypes.byref(self.c_struct()), prefix, 1 if mixed else 0, x_dtype, batch,
                                       1 if x_prepared else 0, flags, ctypes.byref(info)), "hqb_gemv_query")
        return info

    def uses_int8_limbs(self, batch: int, x_dtype: int, prefix: int, mixed: bool = False, flags: int = 0,
                        x_prepared: bool = False) -> bool:
        """Whether the GEMV kernel of one gemv() call multiplies int8 activation limbs."""
        return bool(self.launch_info(batch, x_dtype, prefix, mixed, flags, x_prepared).int8_limbs)

    def gemv_kernel(self, batch: int, x_dtype: int, prefix: int, mixed: bool = False, flags: int = 0,
                    x_prepared: bool = False) -> str:
        """Name of the GEMV kernel one gemv() call runs."""
        return self.launch_info(batch, x_dtype, prefix, mixed, flags, x_prepared).kernel.decode()

    def gemv_launches(self, batch: int, x_dtype: int, prefix: int, mixed: bool = False, flags: int = 0,
                      x_prepared: bool = False) -> int:
        """Kernels one gemv() call launches (activation preparation, GEMV, split-row fix-up)."""
        return int(self.launch_info(batch, x_dtype, prefix, mixed, flags, x_prepared).launches)

    def gemv_gather(self, x: torch.Tensor, gather: "Gather", prefix: int | None = None,
                    bias: torch.Tensor | None = None, workspace: Workspace | None = None, flags: int = 0,
                    stream=None) -> None:
        """This rank's row shard of the layer, its outputs written into every rank's
        gathered buffer (gather.out after gather.wait())."""
        if x.dim() == 1:
            x = x.unsqueeze(0)
        x = x.contiguous()
        batch = x.shape[0]
        xd = _dtype_code(x)
        ws = workspace or self.workspace(batch, xd)
        prefix = self.stage_count if prefix is None else prefix
        check(lib().hqb_gemv_gather(ctypes.byref(self.c_struct()), prefix, _ptr(x), xd, batch, _ptr(bias),
                                    F32 if bias is None else _dtype_code(bias),
                                    F16 if gather.y_dtype == torch.float16 else F32, ctypes.byref(gather.c),
                                    ws.ptr(), ws.nbytes, flags, _stream(stream)), "hqb_gemv_gather")

    def prefill(self, x: torch.Tensor, prefix: int, bias: torch.Tensor | None = None,
                y_dtype: torch.dtype = torch.float16, workspace: torch.Tensor | None = None,
                out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """Large-batch product (hqb_prefill_gemm): FP16 x [batch][cols] -> y [batch][rows];
        the selected stages decoded into FP16 weights in `workspace` (a uint8 device tensor of
        prefill_workspace_bytes(), allocated here when not given), then a cuBLAS GEMM."""
        x = x if x.dim() == 2 else x.unsqueeze(0)
        if not x.is_contiguous():
            raise ValueError("x must be contiguous")
        y = out if out is not None else torch.empty(x.shape[0], self.rows, dtype=y_dtype, device=x.device)
        if workspace is None:
            workspace = torch.empty(self.prefill_workspace_bytes(), dtype=torch.uint8, device=x.device)
        check(lib().hqb_prefill_gemm(ctypes.byref(self.c_struct()), prefix, _ptr(x), _dtype_code(x), x.shape[0],
                                     _ptr(bias), F32 if bias is None else _dtype_code(bias), _ptr(y), _dtype_code(y),
                                     _ptr(workspace), workspace.numel(), _stream(stream)), "hqb_prefill_gemm")
        return y

    def prefill_workspace_bytes(self) -> int:
        return int(lib().hqb_prefill_workspace_bytes(ctypes.byref(self.c_struct())))

    def decode(self, prefix: int | None = None, depth: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        out = torch.empty(self.rows, self.cols, dtype=torch.float32, device=self.device)
        prefix = self.stage_count if prefix is None else prefix
        check(lib().hqb_decode_planes(ctypes.byref(self.c_struct()), prefix, _ptr(depth), _ptr(out), out.numel(),
                                      _stream(stream)), "hqb_decode_planes")
        return out


class Step:
    """A fixed list of GEMV calls (plane matrix, x, prefix, out, flags) on one stream with one
    workspace: the decode step's GEMVs for one host call.  graph=True (default) captures them
    once into a CUDA graph (hqb_step_create) and run() launches it; graph=False runs them
    through hqb_gemv_batch.  independent=True (no call reads another's output) runs them as
    one grouped kernel launch where they share its form (hqb_gemv_grouped).  Buffers are bound at construction; refill x and read out in
    place."""

    def __init__(self, calls, workspace: Workspace, graph: bool = True, independent: bool = False,
                 inputs=(), outputs=()):
        """inputs: (device tensor, pinned host tensor) copied host -> device before the GEMVs;
        outputs: (pinned host tensor, device tensor) copied device -> host after them; both
        are captured into the step's graph (hqb_step_create_io)."""
        self.calls = list(calls)
        self.handle = None
        self.independent = independent
        self.ws = workspace
        arr = (GemvCallC * len(self.calls))()
        self._keep = []
        for i, (pm, x, prefix, out, flags) in enumerate(self.calls):
            x = x if x.dim() == 2 else x.unsqueeze(0)
            if not x.is_contiguous() or not out.is_contiguous():
                raise ValueError("Step buffers must be contiguous")
            ms = pm.c_struct()
            self._keep.append(ms)
            arr[i] = GemvCallC(ctypes.addressof(ms), prefix, _dtype_code(x), None, None, x.data_ptr(), x.shape[0], 0,
                               None, F32, _dtype_code(out), out.data_ptr(), flags, 0)
        self.arr = arr
        if (inputs or outputs) and not graph:
            raise ValueError("input/output copies need graph=True")
        if graph:
            h = vp()
            if inputs or outputs:
                for dst, src in [*inputs, *outputs]:
                    if dst.numel() * dst.element_size() != src.numel() * src.element_size():
                        raise ValueError("copy sizes differ")
                    if not (dst.is_contiguous() and src.is_contiguous()):
                        raise ValueError("copy buffers must be contiguous")
                    host = src if src.device.type == "cpu" else dst
                    if not host.is_pinned():
                        raise ValueError("host buffers of a step must be pinned")
                self._io = [*inputs, *outputs]
                h2d = (CopyC * max(1, len(inputs)))(*[CopyC(d.data_ptr(), s_.data_ptr(), d.numel() * d.element_size())
                                                      for d, s_ in inputs])
                d2h = (CopyC * max(1, len(outputs)))(*[CopyC(d.data_ptr(), s_.data_ptr(), d.numel() * d.element_size())
                                                       for d, s_ in outputs])
                check(lib().hqb_step_create_io(arr, len(self.calls), self.ws.ptr(), self.ws.nbytes, h2d, len(inputs),
                                               d2h, len(outputs), 1 if independent else 0, ctypes.byref(h)),
                      "hqb_step_create_io")
            else:
                create = lib().hqb_step_create_grouped if independent else lib().hqb_step_create
                check(create(arr, len(self.calls), self.ws.ptr(), self.ws.nbytes, ctypes.byref(h)), "hqb_step_create")
            self.handle = h.value

    def run(self, stream=None) -> None:
        if self.handle is not None:
            check(lib().hqb_step_launch(self.handle, _stream(stream)), "hqb_step_launch")
        else:
            run = lib().hqb_gemv_grouped if self.independent else lib().hqb_gemv_batch
            check(run(self.arr, len(self.calls), self.ws.ptr(), self.ws.nbytes, _stream(stream)), "hqb_gemv_batch")

    def close(self) -> None:
        if self.handle is not None:
            lib().hqb_step_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RawMatrix:
    """Stages in the reference's own device layout (any tile geometry)."""

    def __init__(self, geom: Geometry, codes: Sequence[torch.Tensor], fp16_scale_bits: Sequence[torch.Tensor] = (),
                 scales_f32: Sequence[torch.Tensor] = ()):
        self.geom = geom
        self.codes = [c.contiguous() for c in codes]
        self.bits = [b.contiguous() for b in fp16_scale_bits]
        self.f32 = [s.contiguous() for s in scales_f32]

    def _stages(self):
        arr = (RawStage * MAX_STAGES)()
        for i, (c, b) in enumerate(zip(self.codes, self.bits)):
            arr[i] = RawStage(c.data_ptr(), c.numel(), b.data_ptr(), b.numel())
        return arr

    def _stages_f32(self):
        arr = (RawStageF32 * MAX_STAGES)()
        for i, (c, s) in enumerate(zip(self.codes, self.f32)):
            arr[i] = RawStageF32(c.data_ptr(), c.numel(), s.data_ptr(), s.numel())
        return arr

    def gemv(self, x: torch.Tensor, prefix: int, bias: torch.Tensor | None = None, stream=None,
             flags: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """LaunchProgressiveGemv semantics (hqb_raw_gemv_ex); flags RAW_GENERIC / RAW_REQUIRE_FAST."""
        y = out if out is not None else torch.empty(self.geom.original_rows, dtype=torch.float32, device=x.device)
        check(lib().hqb_raw_gemv_ex(ctypes.byref(self.geom), self._stages(), len(self.codes), prefix, _ptr(x),
                                    x.numel(), _ptr(bias), 0 if bias is None else bias.numel(), _ptr(y), y.numel(),
                                    flags, _stream(stream)), "hqb_raw_gemv_ex")
        return y

    def dequantize_prefix(self, prefix: int, stream=None) -> torch.Tensor:
        out = torch.empty(self.geom.original_rows, self.geom.original_columns, dtype=torch.float32,
                          device=self.codes[0].device)
        check(lib().hqb_raw_dequantize_prefix(ctypes.byref(self.geom), self._stages_f32(), len(self.codes), prefix,
                                              _ptr(out), _stream(stream)), "hqb_raw_dequantize_prefix")
        return out

    def dequantize_stage(self, stage: int, stream=None) -> torch.Tensor:
        out = torch.empty(self.geom.original_rows, self.geom.original_columns, dtype=torch.float32,
                          device=self.codes[0].device)
        check(lib().hqb_raw_dequantize_stage(ctypes.byref(self.geom), self._stages_f32(), len(self.codes), stage,
                                             _ptr(out), _stream(stream)), "hqb_raw_dequantize_stage")
        return out

    def linear_ordered(self, x: torch.Tensor, prefix: int, bias: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        x = x.contiguous().reshape(-1, self.geom.original_columns)
        y = torch.empty(x.shape[0], self.geom.original_rows, dtype=torch.float32, device=x.device)
        check(lib().hqb_raw_linear_ordered(ctypes.byref(self.geom), self._stages_f32(), len(self.codes), prefix,
                                           _ptr(x), x.shape[0], _ptr(bias), _ptr(y), _stream(stream)),
              "hqb_raw_linear_ordered")
        return y


# ---- serving operators: paged cache, drafted trees, adapters ------------------------------

_SERVING_DTYPES = {torch.float16: F16, torch.bfloat16: BF16}
_ROW_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
# The calls below go through bind(), which checks the tensors and fills the argument structure in
# one step and answers _UNFIT where an argument does not fit; the methods here then say which.
_UNFIT = -1


def _device_index(device: torch.device) -> int:
    return torch.cuda.current_device() if device.index is None else device.index


def _raw_stream(stream) -> int | None:
    """A stream argument as the number that bind() takes; None: the device's current one."""
    return None if stream is None else _stream(stream) or 0


def _ints(name: str, t: torch.Tensor, n: int, device: int) -> None:
    """Refuses what is no contiguous int32 tensor of n elements on GPU `device`."""
    if t.dtype is not torch.int32 or t.numel() != n or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements on GPU {device}, "
                         f"got {list(t.shape)} {t.dtype} on {t.device}")


def _on_stream(stream: int, device: torch.device):
    """Makes a stream, by its handle, the device's current one for a while."""
    if stream == torch.cuda.current_stream(device).cuda_stream:
        return contextlib.nullcontext()
    # (an ExternalStream of handle 0 would be a new stream, not the default one)
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device))


def _result(shape: tuple, dtype: torch.dtype, device: torch.device, stream) -> torch.Tensor:
    """A call's new result, from the memory of the stream that writes it: another stream's could still
    be in use there."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with _on_stream(_raw_stream(stream), device):
        return torch.empty(shape, dtype=dtype, device=device)


def _on_gpu(name: str, t: torch.Tensor) -> None:
    """Refuses host memory: its address means nothing to a kernel."""
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a GPU, got {t.device}")


def _own_workspace(ws: Workspace, device: int) -> Workspace:
    """A workspace that a caller brings, refused where it is not on GPU `device`."""
    if ws.buf.get_device() != device:
        raise ValueError(f"the workspace must be on GPU {device}, got {ws.buf.device}")
    return ws


def _table(name: str, t: torch.Tensor, rows: int, device: int) -> None:
    """Refuses what is no int32 matrix of `rows` rows."""
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got {list(t.shape)}")
    _ints(name, t, t.numel(), device)


class StreamWorkspaces:
    """The workspaces of calls that bring none: one a stream, grown in powers of two.

    A call under capture gets one that belongs to its capture, from its graph's memory pool, whose
    error word each replay clears: the graph may be replayed on any stream, beside eager calls and
    other graphs.  The newest capture's is held here, for its error word; the graph keeps the memory
    of all of them."""

    def __init__(self, device: torch.device, bytes_of):
        self.device, self.bytes_of = device, bytes_of  # bytes_of(size): what calls up to `size` need
        self._index, self._capture = _device_index(device), bind().capture
        self.eager: dict = {}
        self.captured: dict = {}
        self.kept: dict = {}

    def given(self, ws: Workspace, stream: int) -> Workspace:
        """A workspace that a caller brings: one that a capture uses is kept, whatever replaces it here."""
        if self._capture(self._index, stream):
            self.kept[ws.ptr()] = ws
        return ws

    def take(self, size: int, stream: int) -> Workspace:
        """A workspace for a call of `size` on a stream."""
        capture = self._capture(self._index, stream)
        if capture:
            last = self.captured.get(stream)
            if last is None or last[0] != capture or size > last[1].size:
                last = self.captured[stream] = (capture, self._make(size, stream, None))
            return last[1]
        ws = self.eager.get(stream)
        if ws is None or size > ws.size:
            ws = self.eager[stream] = self._make(size, stream, ws)
        return ws

    def error_flags(self, reset: bool = False) -> int:
        """The HQB_DEVERR_* bits of the calls so far, all streams', and of the newest captures' last
        replays; waits for the device."""
        bits = 0
        with torch.cuda.device(self.device):
            torch.cuda.synchronize()
            for stream, ws in [*self.eager.items(), *((s, ws) for s, (_, ws) in self.captured.items())]:
                bits |= ws.error_flags(stream)
                if reset:
                    check(lib().hqb_workspace_init(ws.ptr(), 256, stream), "hqb_workspace_init")
        return bits

    def _make(self, size: int, stream: int, smaller: Workspace | None) -> Workspace:
        size = 1 << (size - 1).bit_length()
        # on the stream that uses it: the allocator then reuses it in that order
        with _on_stream(stream, self.device):
            ws = Workspace(self.bytes_of(size), self.device, clear=256)
            if smaller is not None:
                ws.buf[:256].copy_(smaller.buf[:256])  # the error word
        ws.size = size
        return ws


class PagePlan:
    """One decode step's lengths as addresses (hqb_page_plan), in buffers that are kept between
    steps: starts [requests + 1], requests and positions [tokens] (entries past the step's last
    token are -1) and flags [1] (HQB_DEVERR_* bits, OR-ed); of a build with tables also slots
    [tokens], held [requests] and free_head [1], of a build with parents mask [tokens, words] (with
    max_new > 0: trees of up to that many nodes).  These four are None after a build that left them
    out; before the first one they are the buffers."""

    def __init__(self, requests: int, tokens: int, page_size: int, num_pages: int, max_new: int = 0, device=None):
        if requests < 1 or tokens < 1 or page_size < 1 or num_pages < 1:
            raise ValueError("requests, tokens, page_size and num_pages must be positive")
        if not 0 <= max_new <= MAX_NODES:
            raise ValueError(f"max_new must be 0..{MAX_NODES}")
        self.page_size, self.num_pages, self.words = page_size, num_pages, -(-max_new // 32)
        self.batch, self.tokens = requests, tokens
        # one buffer, so that a step's metadata is one copy where it is wanted on the host
        sizes = [requests + 1, tokens, tokens, tokens, requests, 1, 1, tokens * self.words]
        parts = torch.zeros(sum(sizes), dtype=torch.int32, device=device or "cuda").split(sizes)
        self.starts, self.requests, self.positions, self._slots, self._held, self._free_head, self.flags, mask = parts
        self._mask = mask.view(tokens, self.words) if self.words else None
        self._paged = self._tree = True
        _on_gpu("a plan's buffers", self.starts)
        self.device = self.starts.device
        self._index = _device_index(self.device)
        at = [t.data_ptr() for t in parts]
        self._args = PagePlanC(requests=requests, page_size=page_size, num_pages=num_pages, token_capacity=tokens,
                               starts=at[0], token_request=at[1], positions=at[2], flags=at[6])
        self._at = ctypes.addressof(self._args)
        self._outputs = (at[3], at[4], at[5], at[7], self.words)
        self._call = bind().page_plan

    def build(self, context_lens: torch.Tensor, new_lens: torch.Tensor, held: torch.Tensor | None = None,
              tables: torch.Tensor | None = None, free_pages: torch.Tensor | None = None,
              free_head: torch.Tensor | None = None, parents: torch.Tensor | None = None, stream=None) -> "PagePlan":
        """Fills the buffers.  tables [requests, columns] (with free_pages and free_head) also gives the
        new tokens pages and slots, writing new columns into it; parents (one a token, in token
        order; a token past their end counts as a root, with HQB_DEVERR_INDEX) gives tree positions
        and masks.  held and free_head are the counts before the
        step (a previous plan's, not this one's buffers)."""
        status = self._call(self._at, self._index, _raw_stream(stream), context_lens, new_lens, held, tables, free_pages,
                            free_head, parents, *self._outputs)
        if status:
            if status == _UNFIT:
                self._refuse(context_lens, new_lens, held, tables, free_pages, free_head, parents)
            check(status, "hqb_page_plan")
        self._paged, self._tree = tables is not None, parents is not None
        return self

    @property
    def slots(self) -> torch.Tensor | None:
        return self._slots if self._paged else None

    @property
    def held(self) -> torch.Tensor | None:
        return self._held if self._paged else None

    @property
    def free_head(self) -> torch.Tensor | None:
        return self._free_head if self._paged else None

    @property
    def mask(self) -> torch.Tensor | None:
        return self._mask if self._tree else None

    def _refuse(self, context_lens, new_lens, held, tables, free_pages, free_head, parents) -> None:
        n, device = self.batch, self._index
        _ints("context_lens", context_lens, n, device)
        _ints("new_lens", new_lens, n, device)
        if held is not None:
            _ints("held", held, n, device)
        if tables is not None:
            if free_pages is None or free_head is None:
                raise ValueError("tables need free_pages and free_head")
            _table("tables", tables, n, device)
            _ints("free_pages", free_pages, free_pages.numel(), device)
            _ints("free_head", free_head, 1, device)
        if parents is not None:
            if not self.words:
                raise ValueError("parents need a plan with max_new > 0")
            _ints("parents", parents, parents.numel(), device)


class PagedCache:
    """A paged cache over two device tensors k, v [pages, page_size, heads, dim] (FP16 or BF16;
    any strides with adjacent elements within a head, the same for both: a cache that stores
    heads before tokens is passed as its transpose(1, 2)).  flags [1] int32 collects the
    HQB_DEVERR_* bits of append() (made here when not given)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, flags: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be [pages, page_size, heads, dim] tensors of one shape, layout, type and device")
        if k.dtype not in _SERVING_DTYPES:
            raise TypeError(f"unsupported dtype {k.dtype}; use float16 or bfloat16")
        if k.stride(3) != 1 and k.shape[3] > 1:
            raise ValueError("a head's elements must be adjacent")
        _on_gpu("k and v", k)
        if flags is not None:
            _ints("flags", flags, 1, _device_index(k.device))
        self.k, self.v = k, v
        self.num_pages, self.page_size, self.heads, self.dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self.c = PagedCacheC(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), _SERVING_DTYPES[k.dtype],
                             self.heads, self.dim, self.page_size, self.num_pages, 0)
        self.flags = torch.zeros(1, dtype=torch.int32, device=k.device) if flags is None else flags
        self._at, self._flags = ctypes.addressof(self.c), self.flags.data_ptr()
        self._index = _device_index(self.device)
        self._call = bind().cache_append

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rows: torch.Tensor | None = None,
               stream=None) -> None:
        """Writes rows of k and v [tokens, heads, dim] (FP16, BF16 or FP32) into the cache's slots
        [count]: row rows[i], or i, goes to slots[i]; negative ones are skipped, and so are ones out
        of range (see flags)."""
        status = self._call(self._at, self._index, _raw_stream(stream), k, v, slots, rows, self._flags)
        if status:
            if status == _UNFIT:
                self._refuse(k, v, slots, rows)
            check(status, "hqb_cache_append")

    def _refuse(self, k, v, slots, rows) -> None:
        if k.dim() != 3 or k.shape[1] != self.heads or k.shape[2] != self.dim or v.shape != k.shape:
            raise ValueError(f"k and v must be [tokens, {self.heads}, {self.dim}]")
        if k.dtype not in _ROW_DTYPES or v.dtype is not k.dtype:
            raise TypeError("k and v must share a type: float16, bfloat16 or float32")
        if (v.stride() != k.stride() or (k.stride(2) != 1 and self.dim > 1) or k.get_device() != self._index
                or v.get_device() != self._index):
            raise ValueError("k and v must share strides (adjacent elements within a head) and the cache's device")
        _ints("slots", slots, slots.numel(), self._index)
        if rows is not None:
            _ints("rows", rows, slots.numel(), self._index)
        raise ValueError("more slots than rows")


class TreeAttention:
    """Attention of drafted trees over a paged cache (hqb_tree_attention) for steps of up to
    `requests` requests, `tokens` tokens in all, max_new nodes and about max_context cached
    tokens a request; holds the call's workspace, cleared on the stream that is current here (or
    takes one: workspace(bytes) gives it, and attentions that follow one another on a stream may
    share it), so calls that overlap need one each."""

    def __init__(self, cache: PagedCache, q_heads: int, requests: int, tokens: int, max_new: int, max_context: int,
                 workspace=None):
        if q_heads < 1 or q_heads % cache.heads != 0:
            raise ValueError("q_heads must be a multiple of the cache's heads")
        if not 1 <= max_new <= MAX_NODES:
            raise ValueError(f"max_new must be 1..{MAX_NODES}")
        if not 1 <= cache.dim <= MAX_HEAD_DIM:
            raise ValueError(f"the head dimension must be 1..{MAX_HEAD_DIM}")
        if requests < 1 or tokens < 1 or max_context < 0:
            raise ValueError("requests and tokens must be positive")
        self.cache, self.q_heads, self.requests, self.tokens = cache, q_heads, requests, tokens
        self.max_new, self.max_context = max_new, max_context
        self._args = AttentionC(requests=requests, tokens=tokens, max_new=max_new, max_context=max_context, q_heads=q_heads)
        self._at = ctypes.addressof(self._args)
        need = lib().hqb_tree_attention_workspace_bytes(cache._at, self._at, cache._index)
        if need == 0:
            raise ValueError("hqb_tree_attention_workspace_bytes rejected the shape")
        self.ws = Workspace(need, cache.device, clear=256) if workspace is None else _own_workspace(workspace(need), cache._index)
        self._ws, self._ws_bytes = self.ws.ptr(), self.ws.nbytes
        self._scale = cache.dim ** -0.5
        self._call = bind().tree_attention

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor,
                 context_lens: torch.Tensor, starts: torch.Tensor, mask: torch.Tensor | None = None,
                 scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                 stream=None) -> torch.Tensor:
        """out [tokens, q_heads, dim] for q [tokens, q_heads, dim] and the step's own k, v
        [tokens, heads, dim]; request r owns tokens starts[r] .. starts[r + 1] and reads the
        first context_lens[r] cached tokens of its row of tables [requests, columns].  mask
        [tokens, words]: bit j of a node's row shows it node j of its request (None: the nodes
        up to itself).  scale None: dim ** -0.5.  lse [tokens, q_heads] FP32 gets the logarithm of
        the sum of weights.  Rows of no request are not written."""
        c = self.cache
        if out is None:
            out = _result((q.shape[0], self.q_heads, c.dim), c.dtype, c.device, stream)
        status = self._call(c._at, self._at, self._ws, self._ws_bytes, c._index, _raw_stream(stream), q, k, v, tables,
                            context_lens, starts, mask, self._scale if scale is None else scale, out, lse)
        if status:
            if status == _UNFIT:
                self._refuse(q, k, v, tables, context_lens, starts, mask, out, lse)
            check(status, "hqb_tree_attention")
        return out

    def _refuse(self, q, k, v, tables, context_lens, starts, mask, out, lse) -> None:
        c, tokens, requests = self.cache, q.shape[0], context_lens.numel()
        for name, t, heads in (("q", q, self.q_heads), ("k", k, c.heads), ("v", v, c.heads), ("out", out, self.q_heads)):
            if tuple(t.shape) != (tokens, heads, c.dim):
                raise ValueError(f"{name} must be [{tokens}, {heads}, {c.dim}], got {list(t.shape)}")
            if t.dtype is not c.dtype or t.get_device() != c._index:
                raise TypeError(f"{name} must have the cache's type and device")
            if t.stride(2) != 1 and c.dim > 1:
                raise ValueError(f"{name}: a head's elements must be adjacent")
        if k.stride() != v.stride():
            raise ValueError("k and v must share strides")
        if any(n > 1 and step == 0 for n, step in zip(out.shape, out.stride())):
            raise ValueError("out: elements must not share their place (an expanded tensor)")
        if requests > self.requests or tokens > self.tokens:
            raise ValueError(f"built for {self.requests} requests and {self.tokens} tokens, got {requests} and {tokens}")
        _table("tables", tables, requests, c._index)
        _ints("context_lens", context_lens, requests, c._index)
        _ints("starts", starts, requests + 1, c._index)
        if mask is not None:
            _table("mask", mask, mask.shape[0], c._index)
            if mask.shape[0] < tokens or mask.shape[1] * 32 < self.max_new:
                raise ValueError(f"mask must be [{tokens}, {-(-self.max_new // 32)}] or larger")
        raise ValueError(f"lse must be a contiguous float32 [{tokens}, {self.q_heads}] tensor")


class LoraSet:
    """Low-rank adapters stacked in two device tensors: a [adapters, max_rank, cols] and b
    [adapters, rows, max_rank] (FP16 or BF16), with ranks [adapters] int32 (None: max_rank each)
    and scales [adapters] FP32 (None: 1).  Workspaces are kept per stream and capture (see
    StreamWorkspaces); the constructing stream's is made at once, for up to max_tokens tokens (0:
    when it is first needed)."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, ranks: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None, max_tokens: int = 8192):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError("a must be [adapters, max_rank, cols] and b [adapters, rows, max_rank]")
        if a.dtype != b.dtype or a.dtype not in _SERVING_DTYPES:
            raise TypeError("a and b must share a type: float16 or bfloat16")
        if not a.is_contiguous() or not b.is_contiguous() or a.device != b.device:
            raise ValueError("a and b must be contiguous and on one device")
        _on_gpu("a and b", a)
        self.adapters, self.max_rank, self.cols = a.shape
        self.rows = b.shape[1]
        if self.adapters < 1 or self.rows < 1 or self.cols < 1:
            raise ValueError("a set has at least one adapter, row and column")
        if not 1 <= self.max_rank <= MAX_RANK:
            raise ValueError(f"max_rank must be 1..{MAX_RANK}")
        if ranks is not None:
            _ints("ranks", ranks, self.adapters, _device_index(a.device))
        if scales is not None and (scales.dtype != torch.float32 or tuple(scales.shape) != (self.adapters,)
                                   or not scales.is_contiguous() or scales.device != a.device):
            raise ValueError(f"scales must be a contiguous float32 [{self.adapters}] tensor")
        self.a, self.b, self.ranks, self.scales = a, b, ranks, scales
        self.dtype, self.device = a.dtype, a.device
        self.c = LoraSetC(a.data_ptr(), b.data_ptr(), _ptr(ranks), _ptr(scales), self.rows, self.cols, self.adapters,
                          self.max_rank, _SERVING_DTYPES[a.dtype], 0)
        self._at, self._index = ctypes.addressof(self.c), _device_index(a.device)
        self._call = bind().lora
        c, index = self.c, self._index  # (not self: a cycle would keep the set's memory)
        self._workspaces = StreamWorkspaces(self.device, lambda tokens: lib().hqb_lora_workspace_bytes(ctypes.byref(c), tokens, index))
        self._ws = self._workspaces.eager
        if max_tokens > 0:
            self.workspace(max_tokens, torch.cuda.current_stream(a.device).cuda_stream)

    def workspace_bytes(self, tokens: int) -> int:
        return lib().hqb_lora_workspace_bytes(self._at, tokens, self._index)

    def error_flags(self, reset: bool = False) -> int:
        """HQB_DEVERR_* bits of the set's calls that brought no workspace (see StreamWorkspaces)."""
        return self._workspaces.error_flags(reset)

    def workspace(self, tokens: int, stream: int) -> Workspace:
        """The stream's workspace, or under capture the capture's, grown to what `tokens` tokens need."""
        return self._workspaces.take(tokens, stream)

    def apply(self, x: torch.Tensor, ids: torch.Tensor, base: torch.Tensor | None = None,
              out: torch.Tensor | None = None, y_dtype: torch.dtype | None = None, workspace: Workspace | None = None,
              stream=None) -> torch.Tensor:
        """base + scale_i * b_i (a_i x) per token, i = ids[token] (negative: base alone) (hqb_lora).
        x [tokens, cols]; base [tokens, rows] (None: zeros) and the result share a type, the
        set's or FP32.  out=base adds in place, e.g. to the output of a projection's gemv()."""
        if out is None:
            kind = y_dtype or (base.dtype if base is not None else x.dtype)
            out = _result((x.shape[0], self.rows), kind, self.device, stream)
        s = torch._C._cuda_getCurrentRawStream(self._index) if stream is None else _raw_stream(stream)
        if workspace is None:
            ws = self._workspaces.take(x.shape[0], s)
        else:
            ws = self._workspaces.given(_own_workspace(workspace, self._index), s)
        status = self._call(self._at, ws.ptr(), ws.nbytes, self._index, s, x, ids, base, out)
        if status:
            if status == _UNFIT:
                self._refuse(x, ids, base, out)
            check(status, "hqb_lora")
        return out

    def _refuse(self, x, ids, base, out) -> None:
        tokens = x.shape[0]
        for name, t, cols, kinds in (("x", x, self.cols, (self.dtype,)), ("out", out, self.rows, (self.dtype, torch.float32)),
                                     ("base", base, self.rows, (out.dtype,))):
            if t is None:
                continue
            if tuple(t.shape) != (tokens, cols) or t.get_device() != self._index:
                raise ValueError(f"{name} must be [{tokens}, {cols}] on {self.device}, got {list(t.shape)}")
            if t.dtype not in kinds:
                raise TypeError(f"{name} must be {' or '.join(map(str, kinds))}, got {t.dtype}")
            if (t.stride(1) != 1 and cols > 1) or (t.stride(0) < cols and tokens > 1):
                raise ValueError(f"{name}: a row's elements must be adjacent, and rows must not overlap")
        _ints("ids", ids, tokens, self._index)
        raise ValueError("base must be out itself or not overlap it")


# ---- output-row sharding across ranks --------------------------------------------------

def shard_rows(rows: int, world: int, rank: int) -> tuple[int, int]:
    """Tile-row aligned contiguous output rows of one rank: (first row, row count).

    Whole 128-row tiles are dealt out as evenly as possible, so every rank's shard is
    itself a valid plane matrix and the ranks' slices tile [0, rows) exactly."""
    if world < 1 or not 0 <= rank < world:
        raise ValueError("invalid rank/world")
    tiles = -(-rows // TILE)
    t0, t1 = tiles * rank // world, tiles * (rank + 1) // world
    r0, r1 = t0 * TILE, min(t1 * TILE, rows)
    return r0, max(0, r1 - r0)


def shard_pad_rows(rows: int, world: int) -> int:
    """Per-rank slot size of the gathered output (the largest shard, whole tiles)."""
    return -(-(-(-rows // TILE)) // world) * TILE


def slice_stage_rows(codes, bits, cols: int, r0: int, nrows: int):
    """Row-shard one matrix's reference-layout stages (codes row-major, scales
    tile-row major): returns the (codes, fp16 bits) slices of rows [r0, r0+nrows)."""
    kpad = -(-cols // TILE) * TILE
    per_row = kpad // 4
    nt = -(-nrows // TILE)
    c = [x[r0 * per_row:(r0 + nt * TILE) * per_row] for x in codes]
    per_tile_row = (kpad // TILE) * TILE
    t0 = r0 // TILE
    b = [x[t0 * per_tile_row:(t0 + nt) * per_tile_row] for x in bits]
    return c, b


# ---------------------------------------------------------------------------------------
# output-row shards across the GPUs of one node: fused all-gather over peer memory

class _DeviceView:
    """Raw device memory seen as a torch tensor (CUDA array interface, no copy)."""

    def __init__(self, ptr: int, shape, typestr: str):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3, "strides": None}


class PeerBuffer:
    """A device buffer of `nbytes` (zero-initialised) that every rank of a torch.distributed
    group maps: rank r's copy is peers[r] (peers[rank] is the local one).  Collective:
    every rank constructs it in the same order."""

    def __init__(self, nbytes: int, group=None):
        import torch.distributed as dist

        self.world = dist.get_world_size(group)
        self.rank = dist.get_rank(group)
        local = vp()
        handle = ctypes.create_string_buffer(64)
        check(lib().hqb_peer_alloc(nbytes, ctypes.byref(local), handle), "hqb_peer_alloc")
        handles = [None] * self.world
        dist.all_gather_object(handles, bytes(handle.raw), group=group)
        self.local = local.value
        self.peers = []
        self._opened = []
        for r, h in enumerate(handles):
            if r == self.rank:
                self.peers.append(self.local)
                continue
            ptr = vp()
            check(lib().hqb_peer_open(ctypes.create_string_buffer(h, 64), ctypes.byref(ptr)), "hqb_peer_open")
            self.peers.append(ptr.value)
            self._opened.append(ptr.value)
        self.nbytes = nbytes

    def close(self):
        for ptr in self._opened:
            lib().hqb_peer_close(ptr)
        self._opened = []
        if self.local:
            lib().hqb_peer_free(self.local)
            self.local = None


class Gather:
    """Gathered output of a row-sharded layer: [batch][world * slot_rows] of y_dtype on every
    rank, filled by PlaneMatrix.gemv_gather on all ranks; wait() orders later work in the
    stream after every rank's slice has arrived."""

    def __init__(self, slot_rows: int, batch: int = 1, y_dtype=torch.float16, group=None):
        self.slot_rows, self.batch = slot_rows, batch
        self.y_dtype = y_dtype
        esize = 2 if y_dtype == torch.float16 else 4
        self.ybuf = PeerBuffer(batch * slot_rows * _world(group) * esize, group)
        self.flags = PeerBuffer(4 * MAX_PEERS, group)
        self.epoch = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.device_flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.world, self.rank = self.ybuf.world, self.ybuf.rank
        c = GatherC()
        c.world, c.rank, c.slot_rows = self.world, self.rank, slot_rows
        for r in range(self.world):
            c.peer_y[r] = self.ybuf.peers[r]
            c.peer_flags[r] = self.flags.peers[r]
        self.c = c
        self.out = torch.as_tensor(_DeviceView(self.ybuf.local, (batch, self.world * slot_rows),
                                               "<f2" if esize == 2 else "<f4"), device="cuda")

    def wait(self, stream=None):
        check(lib().hqb_gather_wait(self.flags.local, self.world, _ptr(self.epoch), _ptr(self.device_flags),
                                    _stream(stream)), "hqb_gather_wait")

    def close(self):
        self.ybuf.close()
        self.flags.close()


def _world(group=None) -> int:
    import torch.distributed as dist

    return dist.get_world_size(group)
