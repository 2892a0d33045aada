"""The sharded study loop with context heads and studies that lack a crop window: the logits of each batch run by itself,
the last one padded; what the missing window's volume holds does not matter."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_b200 import infer
from rsna_knee_efficiency_b200.context import ContextHead
from test_gpu_study import IMG, SLICES, _packs

pytestmark = pytest.mark.gpu


def test_missing_windows_in_the_sharded_loop():
    batch, n = 2, 5
    packs = [p for p, _, _ in _packs(batch * (SLICES - 2))]
    torch.manual_seed(2)
    runner = infer.StudyRunner(packs, 0, batch, SLICES, context=[ContextHead(n_out=3, window=6) for _ in packs])
    vols = torch.from_numpy(infer.make_volumes(n, img=IMG, slices=SLICES, seed=21)).pin_memory()
    present = torch.tensor([[True, True], [True, False], [False, True], [True, True], [False, True]])
    got = infer.run_shard(runner, vols, present=present)
    for rows in ([0, 1], [2, 3], [4, 4]):
        want = runner.run(vols[:, rows].cuda(), present[rows].cuda()).cpu()
        assert torch.equal(got[rows], want)
    assert torch.equal(infer.run_shard(runner, vols, rank=1, world=2, present=present.cuda()), got[3:])
    other = vols.clone()
    for s in range(n):
        other[~present[s], s] = 255 - other[~present[s], s]
    assert torch.equal(infer.run_shard(runner, other.pin_memory(), present=present), got)
    assert not torch.equal(infer.run_shard(runner, other.pin_memory()), infer.run_shard(runner, vols))
