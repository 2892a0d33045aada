"""The context operators under torch's autograd: what a second differentiation, changed masks, unused outputs,
expanded gradients and missing parameters do."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import context
from test_gpu_context_ops import BF16, DEV, F16, gen, i32, randn

pytestmark = pytest.mark.gpu


def inputs(T=40, Hq=4, Hk=2, D=32):
    g = gen(T)
    return [randn(g, T, h, D, dtype=BF16).requires_grad_() for h in (Hq, Hk, Hk)] + [i32([0, 25, T])]


def test_changed_masks_are_noticed():
    for name in ("keep", "len_k"):
        q, k, v, cu = inputs()
        mask = dict(keep=torch.ones(40, dtype=torch.bool, device=DEV)) if name == "keep" else dict(len_k=i32([20, 15]))
        out = context.attention(q, k, v, cu, cu, **mask)
        mask[name][0] = 0
        with pytest.raises(RuntimeError, match="modified"):
            out.float().sum().backward()


def test_second_derivatives_are_refused():
    q, k, v, cu = inputs()
    out = context.attention(q, k, v, cu, cu)
    dq, = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()
    x, w = randn(gen(2), 10, 64).requires_grad_(), torch.ones(64, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(context.layer_norm(x, w, None).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("weight,bias", [(None, F16), (F16, F16), (torch.float32, None), (None, None)])
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm_parameters(weight, bias, res):
    g = gen(5)
    x = randn(g, 30, 72).requires_grad_()
    r = randn(g, 30, 72).requires_grad_() if res else None
    w = None if weight is None else (1 + 0.1 * randn(g, 72)).to(weight).requires_grad_()
    b = None if bias is None else randn(g, 72, dtype=bias).requires_grad_()
    y = context.layer_norm(x, w, b, res=r)
    y, h = y if res else (y, x)
    dy = randn(g, 30, 72)
    (y * dy).sum().backward()                        # (the sum's own gradient: zero)
    hd = h.detach()
    _, _, m, rs, *_ = ref.layer_norm(hd, w, b, 1e-5)
    wx, ww, wb, tx, tw, tb = ref.layer_norm_backward(dy, hd, w, m, rs)
    # (the kernel's own statistics: fp32 roundings of mean and rstd, each 2^-24 relative, as in the bounds)
    ref.close(x.grad, wx, 2 * tx + 4 * ref.U32 * wx.abs(), "dx")
    if res:
        assert torch.equal(r.grad, x.grad)
    if w is not None:
        assert w.grad.dtype == weight
        ref.close(w.grad, ww, 2 * tw + ref.u(weight) * ww.abs() + 8 * ref.U32 * 30 * dy.abs().max(), "dw")
    if b is not None:
        assert b.grad.dtype == bias
        ref.close(b.grad, wb, tb + ref.u(bias) * wb.abs(), "db")


def test_expanded_and_partly_used_gradients():
    """The gradient of a plain sum is one element expanded; an output that nothing uses has none."""
    q, k, v, cu = inputs()
    pos = torch.randint(0, 50, (40, 2), device=DEV, dtype=torch.int32)
    qr, kr = context.rope(q, k, pos, (8, 8))
    qr.sum().backward()
    assert q.grad.isfinite().all() and (k.grad == 0).all()
    q.grad = k.grad = None
    context.attention(q, k, v, cu, cu).sum().backward()
    got = [t.grad.clone() for t in (q, k, v)]
    for t in (q, k, v):
        t.grad = None
    out = context.attention(q, k, v, cu, cu)
    out.backward(torch.ones_like(out))
    assert all(torch.equal(a, t.grad) for a, t in zip(got, (q, k, v)))
    with torch.no_grad():
        assert torch.equal(context.attention(q, k, v, cu, cu), out)
