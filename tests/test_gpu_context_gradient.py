"""Attention's gradient against differences along the gradient itself: with d = sign(gradient) the directional derivative
is the sum of all its magnitudes, so that no part of dq, dk or dv can be off without showing."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, attention_case, i32, randn, run_attention

pytestmark = pytest.mark.gpu


def loss(q, k, v, dout, G, scale, ok):
    Q, K, V = q.transpose(0, 1), k.transpose(0, 1).repeat_interleave(G, 0), v.transpose(0, 1).repeat_interleave(G, 0)
    S = (Q @ K.transpose(1, 2) * scale).masked_fill(~ok, -torch.inf)
    P = torch.where(ok.any(1)[None, :, None], S.softmax(2), 0.0).nan_to_num(0.0)
    return ((P @ V).transpose(0, 1) * dout.double()).sum()


@pytest.mark.parametrize("nq,nk,Hq,Hk,D,t,left,right,sinks,keep", [
    (37, 37, 2, 1, 16, F16, 9, 4, 2, 0.8), (150, 150, 4, 2, 64, F16, -1, 0, 0, 1.0), (150, 290, 2, 2, 128, F16, 60, 20, 5, 0.9),
    (1, 200, 4, 1, 64, F16, -1, -1, 0, 1.0), (300, 300, 4, 4, 40, BF16, 70, -1, 3, 0.8), (5, 40, 6, 2, 128, BF16, 8, 0, 1, 1.0)])
def test_derivative_along_the_gradient(nq, nk, Hq, Hk, D, t, left, right, sinks, keep):
    g, q, k, v, cq, ck, _, mask = attention_case(nq + D, [nq], [nk], Hq, Hk, D, t, left, right, sinks, keep=keep)
    out, lse = run_attention(q, k, v, cq, ck, None, mask)
    dout = randn(g, *q.shape, dtype=t)
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), **mask)
    ok = ref.visible(torch.arange(nq, device=DEV), nq, nk, left, right, sinks, mask["keep"], DEV)
    # The bounds on dq, dk, dv are for the given out and lse; what those are off by moves the gradients by the
    # difference of two 64-bit passes.
    o64, l64, _, _ = ref.attention(q, k, v, cq, ck, **mask)
    given = ref.attention(q, k, v, cq, ck, dout=dout, out=out, lse=lse, **mask)
    exact = ref.attention(q, k, v, cq, ck, dout=dout, out=o64, lse=l64, **mask)
    base = [x.double() for x in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = exact[i].sign()
        total = float(exact[i].abs().sum())
        s = 1e-5                                             # central differences: error of order s^2
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + s * d, base[i] - s * d
        num = float(loss(*hi, dout, Hq // Hk, D ** -0.5, ok) - loss(*lo, dout, Hq // Hk, D ** -0.5, ok)) / (2 * s)
        assert abs(num - total) <= 1e-6 * total, name        # the formulas
        got = float((grads[i].double() * d).sum())
        tol = float((given[i + 3] + (given[i] - exact[i]).abs()).sum()) + 1e-6 * total
        assert tol <= (0.02 if t is F16 else 0.16) * total   # (8 times the roundoff, 8 times the bound: a test worth its name)
        assert abs(num - got) <= tol, (name, num, got, tol)
