"""Layer norm at the widths between 512 and 4096, where a row belongs to 128 or 512 threads, in 16-bit vectors and
in single elements: against the 64-bit restatement, in a process of its own, and from two host threads."""
from __future__ import annotations

import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import _native as nat
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, F32, gen, randn

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
WIDTHS = [520, 632, 640, 704, 768, 784, 792, 1000, 1024, 1064, 1664, 2048, 2056, 4096]


def both_directions(M, C, t, to):
    g = gen(C)
    x, r = randn(g, M, C, dtype=t), randn(g, M, C, dtype=t)
    w, b = 1 + 0.2 * randn(g, C), randn(g, C)
    y, h = torch.empty(M, C, dtype=to, device=DEV), torch.empty_like(x)
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    ops.layer_norm(x, w, b, y, 1e-5, r, h, mean, rstd)
    wh, wy, wm, wr, tol, tm, tr = ref.layer_norm(x, w, b, 1e-5, r)
    assert torch.equal(h.double(), wh)
    ref.close(y, wy, tol * 1.01 + ref.u(to) * wy.abs(), f"y {C}")
    ref.close(mean, wm, tm, f"mean {C}")
    ref.close(rstd, wr, tr, f"rstd {C}")
    dy, ds = randn(g, M, C, dtype=to), randn(g, M, C, dtype=t)
    dx, dw, db = torch.empty_like(x), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.layer_norm_backward(dy, h, w, mean, rstd, dx, dw, db, dsum=ds)
    wx, ww, wb, tx, tw, tb = ref.layer_norm_backward(dy, h, w, mean, rstd, ds)
    ref.close(dx, wx, tx * 1.01 + ref.u(t) * wx.abs(), f"dx {C}")
    ref.close(dw, ww, tw, f"dw {C}")
    ref.close(db, wb, tb, f"db {C}")


def test_widths_in_a_process_of_its_own():
    """The widths whose backward pass asks for a little more shared memory than a launch has by default, before any
    other width has run: what a call may use must not depend on the calls before it."""
    code = ("import test_gpu_context_widths as t\n"
            "for C in (632, 640, 704, 768, 784):\n"
            "    for dt in (t.BF16, t.F16):\n"
            "        t.both_directions(37, C, dt, dt)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT / "tests", env={**os.environ, "PYTHONPATH": str(ROOT)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("t,to", [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(C, t, to):
    both_directions(301, C, t, to)


@pytest.mark.parametrize("direction,widths", [("forward", (5200, 8000)), ("backward", (1064, 1664))])
def test_two_widths_from_several_host_threads(direction, widths):
    """Widths of one kernel instance that ask for different amounts of shared memory, called from four host threads
    at the C entry (which lets go of Python's lock): no call is refused for what another thread asks."""
    lib, refused, go = nat.lib(), [], threading.Barrier(4, timeout=60)

    def work(C):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x, y = (torch.ones(8, C, dtype=BF16, device=DEV) for _ in range(2))
            mean, rstd = torch.zeros(8, device=DEV), torch.ones(8, device=DEV)
            if direction == "forward":
                fn = lib.dn8_layer_norm
                a = nat.LayerNormArgs(x=x.data_ptr(), y=y.data_ptr(), rows=8, x_stride=C, y_stride=C, C=C, eps=1e-5)
            else:
                fn = lib.dn8_layer_norm_bwd
                a = nat.LayerNormBwdArgs(dy=x.data_ptr(), x=x.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr(),
                                         dx=y.data_ptr(), rows=8, dy_stride=C, x_stride=C, dx_stride=C, C=C)
            a.x_type = a.y_type = nat.DN8_BF16
            s.synchronize()
            go.wait()
            refused.append(sum(fn(a, s.cuda_stream) != nat.DN8_OK for _ in range(20000)))
            s.synchronize()
    switch = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    threads = [threading.Thread(target=work, args=(C,)) for C in widths * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    sys.setswitchinterval(switch)
    assert refused == [0] * 4
