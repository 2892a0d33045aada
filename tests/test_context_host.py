"""The host side of the study loop around context heads, without a GPU."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_b200 import infer
from test_host import _FakeRunner


def test_run_shard_checks_before_it_gives_logits_out():
    class Failing(_FakeRunner):
        def check(self):
            assert self.calls == 3                           # once, behind the last batch
            raise RuntimeError("device error")
    with pytest.raises(RuntimeError, match="device error"):
        infer.run_shard(Failing(3), infer.make_volumes(7, img=16, slices=4, seed=3))


class Masked(_FakeRunner):
    """Logits that tell which windows `present` named."""

    def run(self, vols, present=None):
        return super().run(vols) if present is None else super().run(vols) * 0 + present @ torch.tensor([1.0, 2.0])[:, None]


@pytest.mark.parametrize("rank,world,studies", [(0, 1, None), (1, 2, None), (0, 2, [6, 0, 0, 3, 1]), (1, 2, [6, 0, 0, 3, 1]),
                                                (2, 3, [4])])
def test_run_shard_passes_the_windows_that_studies_have(rank, world, studies):
    vols = infer.make_volumes(7, img=16, slices=4, seed=3)
    present = torch.tensor([[n & 1, n >> 1 & 1] for n in range(7)]).bool()

    class Runner(Masked):
        def run(self, v, p):
            assert p.shape == (3, 2) and p.dtype == torch.bool
            return super().run(v, p.float())
    out = infer.run_shard(Runner(3), vols, rank, world, studies, present)
    order = list(range(7)) if studies is None else studies
    start, end = infer.shard(len(order), world, rank)
    want = torch.tensor([float(n & 3) for n in order[start:end]])[:, None].expand(-1, 4)
    assert torch.equal(out, want)
    for bad in (present[:6], present.t(), present.int()):
        with pytest.raises(ValueError, match="present"):
            infer.run_shard(Runner(3), vols, rank, world, studies, bad)
