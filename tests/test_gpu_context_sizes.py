"""Sizes and limits that need more than 32 bits are refused; their upper bits are not dropped on the way to the C
entry."""
from __future__ import annotations

import pytest
import torch

from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, i32

pytestmark = pytest.mark.gpu
WIDE = (1 << 32) + 8                                         # (its lower 32 bits: 8)


def test_rows_too_long():
    x = torch.empty(1, WIDE, dtype=BF16, device=DEV)
    s = torch.zeros(1, device=DEV)
    with pytest.raises(ValueError, match="2\\^29"):
        ops.layer_norm(x, None, None, x)
    with pytest.raises(ValueError, match="2\\^29"):
        ops.layer_norm_backward(x, x, None, s, s, x)
    q = x.view(1, 1, WIDE)
    with pytest.raises(ValueError):
        ops.rope(q, None, i32([[1]]), q, None, (4,))
    with pytest.raises(ValueError):
        ops.attention(q, q, q, q, i32([0, 1]), i32([0, 1]))


def test_limits_that_would_wrap():
    q = torch.ones(5, 2, 64, dtype=BF16, device=DEV)
    out, cu = torch.empty_like(q), i32([0, 5])
    for bad in (dict(left=-(1 << 32)), dict(right=-(1 << 32)), dict(sinks=-(1 << 32)), dict(left=-(1 << 32) + 3), dict(sinks=-2)):
        with pytest.raises(ValueError):
            ops.attention(q, q, q, out, cu, cu, **bad)
    for sections in (((1 << 32) + 4,), (-1, 4), (4, (1 << 32)), (33,)):
        with pytest.raises(ValueError):
            ops.rope(q, None, torch.zeros(5, len(sections), dtype=torch.int32, device=DEV), out, None, sections)
