"""What a kernel of a context head reports on the GPU reaches the program: the head's error word, read by `check`, by the
study runner's, and by the sharded study loop before it gives logits out. (Offsets outside the tensors stand for a
wait that was given up: both set the word, and neither reads or writes out of range.)"""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_b200 import _native as nat
from rsna_knee_efficiency_b200 import infer
from rsna_knee_efficiency_b200.context import ContextHead
from test_gpu_study import IMG, SLICES, _packs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def beyond(lay):
    """The layout with its last study's end far behind the tokens."""
    cu = lay["cu_k"].clone()
    cu[-1] += 100000
    return {**lay, "cu_k": cu}


@pytest.mark.parametrize("grad", [False, True])
def test_head(grad):
    torch.manual_seed(1)
    m = ContextHead(c=64, n_out=3, width=64, heads=2, window=4).to(DEV)
    m.check()                                                # (no call yet: nothing to report)
    feats, pos = torch.randn(20, 64, device=DEV), torch.zeros(20, 2, dtype=torch.int32, device=DEV)
    lay = m.layout([12, 8], DEV)
    with torch.set_grad_enabled(grad):
        good = m(feats, lay, pos)
        m.check()
        assert "err" not in m.state_dict() and not list(m.buffers()) and m.err.device == torch.device(DEV)
        bad = m(feats, beyond(lay), pos)
    with pytest.raises(nat.Dn8Error, match="code 4"):
        m.check()
    m.check()                                                # the word is read once
    if grad:
        bad.sum().backward()                                 # the backward pass reports too
        with pytest.raises(nat.Dn8Error):
            m.check()
    assert torch.equal(m(feats, lay, pos).detach(), good.detach())
    m.check()


def test_study_loop():
    studies = 2
    packs = [p for p, _, _ in _packs(studies * (SLICES - 2))]
    runner = infer.StudyRunner(packs, 0, studies, SLICES, context=[ContextHead(n_out=2) for _ in packs])
    vols = torch.from_numpy(infer.make_volumes(studies, img=IMG, slices=SLICES, seed=5)).pin_memory()
    want = infer.run_shard(runner, vols)
    good = runner.layouts[1]
    runner.layouts[1] = beyond(good)
    runner.run(vols.cuda())
    with pytest.raises(nat.Dn8Error, match="ContextHead"):
        runner.check()
    with pytest.raises(nat.Dn8Error, match="ContextHead"):
        infer.run_shard(runner, vols)
    runner.layouts[1] = good
    assert torch.equal(infer.run_shard(runner, vols), want)


def test_first_call_in_inference_mode_or_in_a_capture():
    torch.manual_seed(2)
    feats, pos = torch.randn(20, 64, device=DEV), torch.zeros(20, 2, dtype=torch.int32, device=DEV)
    m = ContextHead(c=64, n_out=3, width=64, heads=2).to(DEV)
    bad = beyond(m.layout([12, 8], DEV))
    with torch.inference_mode():
        m(feats, bad, pos)
    with pytest.raises(nat.Dn8Error):
        m.check()
    m.check()
    n = ContextHead(c=64, n_out=3, width=64, heads=2).to(DEV)
    m(feats, m.layout([20], DEV), pos)                       # (the libraries' own first calls)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n(feats, bad, pos)
    for _ in range(2):
        graph.replay()
        with pytest.raises(nat.Dn8Error):
            n.check()
        n.check()
