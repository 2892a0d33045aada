"""The study loop with context heads and the flip of test-time augmentation: a head sees every study's windows, then the
same windows flipped, at the same positions; a slot that a study lacks is masked in both."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import infer
from rsna_knee_efficiency_b200.context import ContextHead
from test_gpu_context_head import GAIN, ROUNDINGS
from test_gpu_study import IMG, SLICES, _packs

pytestmark = pytest.mark.gpu


def test_flipped_windows():
    studies = 2
    packs = [p for p, _, _ in _packs(2 * studies * (SLICES - 2))]
    torch.manual_seed(3)
    heads = [ContextHead(n_out=6, window=5) for _ in packs]
    runner = infer.StudyRunner(packs, 0, studies, SLICES, flip_tta=True, context=heads)
    vols = torch.from_numpy(infer.make_volumes(studies, img=IMG, slices=SLICES, seed=9)).cuda()
    present = torch.tensor([[True, False], [True, True]]).cuda()
    for have in (None, present):
        got = runner.run(vols, have).clone()
        runner.check()
        want = torch.zeros_like(got)
        for k, h in enumerate(heads):
            w = torch.from_numpy(runner.windows[k]).int().cuda()
            n = len(w)
            pos = torch.stack([w // (SLICES - 2), w % (SLICES - 2)], 1).repeat(2, 1)
            for s in range(studies):
                feats = runner.encoders[k].out[s * 2 * n:(s + 1) * 2 * n]
                keep = None if have is None else have[s][pos[:, 0].long()]
                with torch.no_grad():
                    want[s] += h(feats, [2 * n], pos, keep)[0] / len(heads)
        # (one study alone or two together: the library's matrix products may add in another order)
        torch.testing.assert_close(got, want, rtol=0, atol=ROUNDINGS * GAIN * ref.u(torch.bfloat16) * float(want.abs().max()))
