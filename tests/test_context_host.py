"""The host side of the study loop around context heads, without a GPU."""
from __future__ import annotations

import pytest

from rsna_knee_efficiency_b200 import infer
from test_host import _FakeRunner


def test_run_shard_checks_before_it_gives_logits_out():
    class Failing(_FakeRunner):
        def check(self):
            assert self.calls == 3                           # once, behind the last batch
            raise RuntimeError("device error")
    with pytest.raises(RuntimeError, match="device error"):
        infer.run_shard(Failing(3), infer.make_volumes(7, img=16, slices=4, seed=3))
