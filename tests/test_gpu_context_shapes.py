"""Layer norms of narrow rows (several to a warp) and interleaved pairs that do not fill a vector, against the
64-bit restatements."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, F32, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,C,t,to", [(1, 8, BF16, BF16), (3001, 8, F32, F16), (4099, 31, BF16, BF16), (777, 64, F32, BF16),
                                      (5000, 65, F16, F16), (33, 100, F32, F32), (999, 128, F16, F16), (130, 128, F32, F32),
                                      (257, 129, BF16, BF16), (6000, 136, BF16, BF16)])
@pytest.mark.parametrize("res", [False, True])
def test_narrow_layer_norm(M, C, t, to, res):
    g = gen(M + C)
    x = randn(g, M, C, dtype=t) - 2
    r = randn(g, M, C, dtype=t) if res else None
    w, b = 1 + 0.2 * randn(g, C), randn(g, C)
    y, s = torch.empty(M, C, dtype=to, device=DEV), torch.empty_like(x) if res else None
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    ops.layer_norm(x, w, b, y, 1e-5, r, s, mean, rstd)
    h, wy, wm, wr, tol, tm, tr = ref.layer_norm(x, w, b, 1e-5, r)
    ref.close(y, wy, tol + ref.u(to) * wy.abs() + ref.eta(to), "y")
    ref.close(mean, wm, tm, "mean")
    ref.close(rstd, wr, tr, "rstd")
    if res:
        assert torch.equal(s.double(), h)
    hs = s if res else x
    dy, ds = randn(g, M, C, dtype=to), randn(g, M, C, dtype=t) if res else None
    dx, dw, db = torch.empty_like(x), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.layer_norm_backward(dy, hs, w, mean, rstd, dx, dw, db, ds)
    wdx, wdw, wdb, tx, tw, tb = ref.layer_norm_backward(dy, hs, w, mean, rstd, ds)
    ref.close(dx, wdx, tx + ref.u(t) * wdx.abs() + ref.eta(t), "dx")
    ref.close(dw, wdw, tw, "dw")
    ref.close(db, wdb, tb, "db")
    again = [torch.empty_like(z) for z in (dx, dw, db)]
    ops.layer_norm_backward(dy, hs, w, mean, rstd, *again, ds)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


@pytest.mark.parametrize("M,C,t,to", [(300, 2, BF16, BF16), (77, 514, F16, F16), (40, 2050, F32, F16), (9, 8194, F32, F32), (5, 18002, BF16, BF16),
                                      (64, 130, F32, BF16), (33, 515, BF16, BF16), (21, 1537, F32, F32), (3, 4100, F16, F16)])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("wt", [F32, F16])
def test_layer_norm_by_pairs(M, C, t, to, res, wt):
    g = gen(M * C + 1)
    wide = randn(g, M, C + 3, dtype=t)               # rows an odd number of elements apart: single elements again
    for x in (randn(g, M, C, dtype=t), wide[:, 1:C + 1], wide[:, 2:C + 2]):
        r = randn(g, M, C, dtype=t) if res else None
        w, b = (1 + 0.2 * randn(g, C)).to(wt), randn(g, C, dtype=wt)
        y, s = torch.empty(M, C, dtype=to, device=DEV), torch.empty(M, C, dtype=t, device=DEV) if res else None
        ops.layer_norm(x, w, b, y, 1e-5, r, s)
        h, wy, _, _, tol, _, _ = ref.layer_norm(x, w, b, 1e-5, r)
        ref.close(y, wy, tol + ref.u(to) * wy.abs() + ref.eta(to), "y")
        if res:
            assert torch.equal(s.double(), h)


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("T,Hq,Hk,D,sec,per_axis", [
    (1, 1, 0, 8, (1,), False), (53, 8, 2, 64, (1, 30), True), (700, 4, 1, 32, (1, 11, 1, 2), True), (19, 3, 3, 80, (39,), False),
    (5, 2, 1, 512, (60, 68), False), (2000, 1, 1, 128, (64,), False), (7, 2, 2, 20, (3, 2), True)])
@pytest.mark.parametrize("inverse", [False, True])
def test_interleaved_rope(t, T, Hq, Hk, D, sec, per_axis, inverse):
    g = gen(T + D)
    q, k = randn(g, T, Hq, D, dtype=t), randn(g, T, Hk, D, dtype=t) if Hk else None
    pos = torch.randint(-(1 << 20), 1 << 20, (T, len(sec)), generator=g, device=DEV, dtype=torch.int32)
    if 2 * sum(sec) < D:
        q[:, :, 2 * sum(sec)] = float("inf")         # behind the pairs anything is copied
    qo, ko = torch.empty_like(q), torch.empty_like(k) if Hk else None
    ops.rope(q, k, pos, qo, ko, sec, 10000.0, per_axis, True, inverse)
    P2 = 2 * sum(sec)
    for x, y in ((q, qo), (k, ko)):
        if x is None:
            continue
        assert torch.equal(y[:, :, P2:], x[:, :, P2:])
        want, tol = ref.rope(x[:, :, :P2], pos, sec, 10000.0, per_axis, True, inverse)
        ref.close(y[:, :, :P2], want, tol + ref.u(t) * want.abs(), "rope")
    if Hk:                                           # in place
        ops.rope(q, k, pos, q, k, sec, 10000.0, per_axis, True, inverse)
        assert torch.equal(q, qo) and torch.equal(k, ko)
