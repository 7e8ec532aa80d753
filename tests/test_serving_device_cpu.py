"""CPU: the serving operators' binding, and the GEMV operator, make their tensors' GPU current around
the library's calls.

PyTorch's device switch is replaced by one that records (tests/native/recording_device_guard.cpp),
in a process of its own; fake tensors stand in for tensors on a second GPU, so nothing is launched."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

REPO = Path(__file__).resolve().parents[1]

PROGRAM = """
import ctypes, sys
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import harpq_b200 as hqb

bind = hqb.bind()
guard = ctypes.CDLL(sys.argv[1])
guard.record_devices()
with FakeTensorMode():
    i = torch.empty(1, dtype=torch.int32, device="cuda:1")
    x = torch.empty(1, 8, dtype=torch.float16, device="cuda:1")
    h = x[None]
plan = hqb.PagePlanC(requests=1, page_size=16, num_pages=8, token_capacity=1)
cache = hqb.PagedCacheC(256, 256, 128, 8, 8, hqb.F16, 1, 8, 16, 8, 0)
attention = hqb.AttentionC(requests=1, tokens=1, max_new=1, max_context=1, q_heads=1)
adapters = hqb.LoraSetC(256, 256, None, None, 8, 8, 1, 8, hqb.F16, 0)
at = ctypes.addressof
calls = {
    "page_plan": (at(plan), 1, 0, i, i, None, None, None, None, None, 0, 0, 0, 0, 0),
    "cache_append": (at(cache), 1, 0, h, h, i, None, 256),
    "tree_attention": (at(cache), at(attention), 256, 256, 1, 0, h, h, h, i[None], i, i, None, 1.0, h, None),
    "lora": (at(adapters), 256, 256, 1, 0, x, i, None, x),
}
log = ctypes.POINTER(ctypes.c_int)()
for name, args in calls.items():
    before = guard.recorded_devices(ctypes.byref(log))
    try:
        getattr(bind, name)(*args)
    except RuntimeError:  # a fake tensor has no address
        pass
    print(name, log[before:guard.recorded_devices(ctypes.byref(log))])
"""


def test_binding_makes_the_tensors_device_current(tmp_path):
    from torch.utils import cpp_extension

    so = tmp_path / "guard.so"
    torch_lib = Path(torch.__file__).parent / "lib"
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-fPIC", "-shared",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    *[a for d in cpp_extension.include_paths() for a in ("-isystem", d)],
                    str(REPO / "tests" / "native" / "recording_device_guard.cpp"), "-o", str(so), "-L", str(torch_lib), "-lc10"],
                   check=True, timeout=300)
    run = subprocess.run([sys.executable, "-c", PROGRAM, str(so)], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": str(REPO / "harp-q_b200"), "CUDA_VISIBLE_DEVICES": ""})
    assert run.returncode == 0, run.stderr
    assert run.stdout.split("\n")[:-1] == [f"{name} [1, 0]" for name in ("page_plan", "cache_append", "tree_attention", "lora")]


def test_gemv_operator_makes_its_inputs_device_current(monkeypatch):
    import harpq_b200 as hqb
    import harpq_b200_ops

    inside, seen = [], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *_):
            inside.pop()

    class Library:
        @staticmethod
        def hqb_gemv(*_):
            seen.append(list(inside))
            return 0

    planes = [torch.zeros(hqb.plane_bytes(hqb.geometry(128, 128)), dtype=torch.uint8)]
    x, stream = torch.zeros(2, 128, dtype=torch.float16), type("Stream", (), {"cuda_stream": 7})
    scratch = type("Scratch", (), {"ptr": lambda self: 256, "nbytes": 256})()
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    monkeypatch.setattr(harpq_b200_ops, "_plane_matrix", lambda *_: hqb.PlaneMatrixC())
    monkeypatch.setattr(harpq_b200_ops, "_workspace", lambda *_: scratch)
    monkeypatch.setattr(hqb, "lib", lambda: Library)
    harpq_b200_ops.gemv._init_fn(x, planes, 128, 128, 1)
    assert seen == [[x.device]]
