"""A CUDA error that an entry point has reported does not stay behind for the program's next CUDA call (torch asks for
the last error after its own launches and would raise it there)."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

# A launch into a stream whose capture has been given up is refused by the runtime: nothing reaches the GPU.
CODE = """
import ctypes, torch
from rsna_knee_efficiency_b200 import _native as nat, ops
runtime = ctypes.CDLL("libcudart.so.12")                 # the one that the library and torch share
x = torch.ones(4, 64, device="cuda")
y = torch.zeros_like(x)
refused = left = None
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            torch.cuda.synchronize()                     # not allowed here: the capture is over
        except RuntimeError:
            pass
        runtime.cudaGetLastError()
        try:
            ops.layer_norm(x, None, None, y)
        except nat.Dn8Error as e:
            refused = str(e)
        left = runtime.cudaPeekAtLastError()
except RuntimeError:
    pass
assert refused and "Capture" in refused, refused
assert left == 0, left
ops.layer_norm(x, None, None, y)
assert (y == 0).all()
"""


def test_reported_errors_are_not_left_behind():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env={**os.environ, "PYTHONPATH": str(ROOT)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
