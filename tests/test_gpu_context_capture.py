"""Capture through autograd is refused in the backward pass too: a forward pass that ran eagerly, its gradient asked for
inside a capture of the same stream. Each case in a process of its own (a capture that torch cannot carry through may
end the process)."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CODE = """
import torch
from rsna_knee_efficiency_b200 import context
s = torch.cuda.Stream()
x = torch.randn(40, 4, 64, device="cuda").bfloat16().requires_grad_()
cu = torch.tensor([0, 40], dtype=torch.int32).cuda()
pos = torch.zeros(40, 1, dtype=torch.int32).cuda()
def run():
    if "{what}" == "layer_norm":
        return context.layer_norm(x.view(40, 256), None, None)
    if "{what}" == "rope":
        return context.rope(x, x, pos, (8,))[0]
    return context.attention(x, x, x, cu, cu)
kept = run()                                             # another eager graph of the same leaf, on another stream
seed = torch.ones_like(kept)
torch.cuda.synchronize()
with torch.cuda.stream(s):
    out = run()
s.synchronize()
refused = ""
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
        out.backward(seed)
except RuntimeError as e:
    refused = str(e)
assert "cannot be captured" in refused, refused
x.grad = None
kept.backward(seed)
torch.cuda.synchronize()
assert x.grad.isfinite().all()
"""


@pytest.mark.parametrize("what", ["layer_norm", "rope", "attention"])
def test_backward_inside_a_capture(what):
    r = subprocess.run([sys.executable, "-c", CODE.replace("{what}", what)], cwd=ROOT, env={**os.environ, "PYTHONPATH": str(ROOT)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])
