"""Sizes beyond what the C structures of the context operators hold: refused at the C entry, before any CUDA call."""
from __future__ import annotations

from rsna_knee_efficiency_b200 import _native as nat


def test_rows_too_long():
    lib = nat.lib()
    for C in ((1 << 29), (1 << 30), (1 << 31) - 1):
        assert lib.dn8_layer_norm(nat.LayerNormArgs(x=4096, y=4096, rows=2, C=C, eps=1e-5), None) == nat.DN8_EINVAL
        a = nat.LayerNormBwdArgs(dy=4096, x=4096, mean=4096, rstd=4096, dx=4096, rows=2, C=C)
        assert lib.dn8_layer_norm_bwd(a, None) == nat.DN8_EINVAL
        assert lib.dn8_layer_norm_bwd_work(C) == -1
    assert lib.dn8_layer_norm_bwd_work((1 << 29) - 1) > 0
