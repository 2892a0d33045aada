"""Keys that only the window hides from every query of their sequence (what an evicted part of a cache is) may hold
anything: the outputs and gradients are those of a call without it, bit for bit."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, attention_case, i32, randn, run_attention

pytestmark = pytest.mark.gpu

CASES = [  # queries, keys, head size, left, right, first tokens, type: row kernel, tiles, borders inside and between tiles
    (1, 700, 64, 20, -1, 0, BF16), (1, 700, 128, 20, 0, 3, F16), (3, 900, 64, 100, 0, 33, BF16), (1, 513, 128, 0, 0, 0, BF16),
    (200, 700, 64, 40, 0, 0, BF16), (200, 700, 128, 40, 30, 3, F16), (300, 900, 64, 100, -1, 130, BF16), (129, 1000, 128, 64, 0, 128, BF16),
    (130, 386, 64, 0, 0, 5, F16), (150, 5000, 64, 300, 0, 4, BF16)]


@pytest.mark.parametrize("nq,nk,D,left,right,sinks,t", CASES)
@pytest.mark.parametrize("kept", [1.0, 0.8])
def test_keys_that_the_window_hides(nq, nk, D, left, right, sinks, t, kept):
    g, q, k, v, cq, ck, _, mask = attention_case(nq + nk, [nq, 2, nq], [nk, 40, nk], 4, 2, D, t, left, right, sinks, keep=kept)
    seen = torch.zeros(ck[-1], dtype=torch.bool, device=DEV)
    for b in range(3):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        seen[ck[b]:ck[b + 1]] = ref.visible(torch.arange(n, device=DEV), n, m, left, right, sinks, None, DEV).any(0)
    assert int((~seen).sum()) > 100                          # (hidden by the window alone)
    dout = randn(g, *q.shape, dtype=t)

    def everything():
        out, lse = run_attention(q, k, v, cq, ck, None, mask)
        grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
        ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), **mask)
        return out, lse, *grads
    clean = everything()
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, **mask)
    ref.close(clean[0], o, to, "out")
    want = ref.attention(q, k, v, cq, ck, dout=dout, out=clean[0], lse=clean[1], **mask)
    for a, w, tol, name in zip(clean[2:], want[:3], want[3:], ("dq", "dk", "dv")):
        ref.close(a, w, tol, name)
    val = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(t).min], device=DEV).to(t)
    for x in (k, v):
        x[~seen] = val[torch.randint(0, 4, (int((~seen).sum()), *x.shape[1:]), generator=g, device=DEV)]
    for a, b, name in zip(clean, everything(), ("out", "lse", "dq", "dk", "dv")):
        assert torch.equal(a, b), name
