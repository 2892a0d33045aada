"""The context transformer's operators on the GPU against 64-bit restatements (tests/context_ref.py,
which derives the bounds): types, odd sizes, strides, masks that leave rows empty, gradients."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


# ---- layer norm ----
LN = [(1, 1, F32, F32), (3, 7, F32, BF16), (5, 64, BF16, BF16), (24, 1664, F32, BF16), (33, 513, F16, F16),
      (301, 512, BF16, BF16), (17, 1663, F32, F32), (9, 2048, F32, F16), (1200, 72, BF16, BF16), (4, 4104, F16, F16),
      (3, 9001, BF16, BF16), (2, 20000, F32, F32), (2, 40000, BF16, BF16)]


@pytest.mark.parametrize("M,C,t,to", LN)
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm(M, C, t, to, res):
    g = gen(M * C)
    x = randn(g, M, C, dtype=t) + 3
    r = randn(g, M, C, dtype=t) if res else None
    w, b = 1 + 0.2 * randn(g, C), randn(g, C)
    y, s = torch.empty(M, C, dtype=to, device=DEV), torch.empty_like(x) if res else None
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    ops.layer_norm(x, w, b, y, 1e-5, r, s, mean, rstd)
    h, wy, wm, wr, tol, tm, tr = ref.layer_norm(x, w, b, 1e-5, r)
    if res:
        assert torch.equal(s.double(), h)
    ref.close(y, wy, tol * 1.01 + ref.u(to) * wy.abs(), "y")
    ref.close(mean, wm, tm, "mean")
    ref.close(rstd, wr, tr, "rstd")


@pytest.mark.parametrize("M,C,t,to", LN)
@pytest.mark.parametrize("res", [False, True])
def test_layer_norm_backward(M, C, t, to, res):
    g = gen(M + C)
    x = randn(g, M, C, dtype=t) + 1
    dy = randn(g, M, C, dtype=to)
    ds = randn(g, M, C, dtype=t) if res else None
    w = 1 + 0.2 * randn(g, C)
    _, _, m, r, *_ = ref.layer_norm(x, w, None, 1e-5)
    mean, rstd = m.float(), r.float()
    dx, dw, db = torch.empty_like(x), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db, dsum=ds)
    wx, ww, wb, tx, tw, tb = ref.layer_norm_backward(dy, x, w, mean, rstd, ds)
    ref.close(dx, wx, tx * 1.01 + ref.u(t) * wx.abs(), "dx")
    ref.close(dw, ww, tw, "dw")
    ref.close(db, wb, tb, "db")
    again = torch.empty_like(dw)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, again, db, dsum=ds)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("C", [96, 97])
def test_layer_norm_strides_parameters_in_place(C):
    g = gen(C)
    big = randn(g, 40, 3 * C + 8, dtype=BF16)
    x, r = big[:, :C], big[:, C:2 * C]
    w, b = randn(g, C, dtype=BF16), randn(g, C, dtype=BF16)
    _, wy, _, _, tol, _, _ = ref.layer_norm(x, w, b, 1e-3, r)
    h = (x.double() + r.double()).to(BF16)
    rest = big[:, 2 * C:].clone()
    ops.layer_norm(x, w, b, r, 1e-3, r, x)          # y over res, sum over x
    assert torch.equal(x, h) and torch.equal(big[:, 2 * C:], rest)
    ref.close(r, wy, tol * 1.01 + ref.u(BF16) * wy.abs())
    # no weight, no bias, no statistics; and an empty matrix
    y = torch.empty_like(h)
    ops.layer_norm(h, None, None, y)
    _, wy, _, _, tol, _, _ = ref.layer_norm(h, None, None, 1e-5)
    ref.close(y, wy, tol * 1.01 + ref.u(BF16) * wy.abs())
    e = torch.empty(0, C, device=DEV)
    ops.layer_norm(e, None, None, e)
    dw = torch.full((C,), 7.0, device=DEV)
    v = torch.empty(0, device=DEV)
    ops.layer_norm_backward(e, e, None, v, v, e, dw)
    assert (dw == 0).all()                          # a sum over no rows


def test_layer_norm_constant_rows():
    x = torch.full((4, 512), 1000.0, device=DEV)
    y = torch.empty_like(x)
    ops.layer_norm(x, None, None, y)
    assert (y == 0).all()                           # no cancellation noise blown up by 1 / sqrt(eps)


def test_layer_norm_gradient_against_differences():
    g = gen(5)
    M, C, eps = 6, 40, 1e-5
    x, w, b, dy = randn(g, M, C), randn(g, C), randn(g, C), randn(g, M, C)
    y, mean, rstd = torch.empty_like(x), torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    ops.layer_norm(x, w, b, y, eps, mean=mean, rstd=rstd)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ops.layer_norm_backward(dy, x, w, mean, rstd, dx, dw, db)

    def loss(x_, w_, b_):
        return (ref.layer_norm(x_, w_, b_, eps)[1] * dy.double()).sum()
    for t, grad, put in ((x, dx, lambda v: loss(v, w, b)), (w, dw, lambda v: loss(x, v, b)), (b, db, lambda v: loss(x, w, v))):
        d = randn(g, *t.shape).double()
        s = 1e-5                                     # central differences: error of order s^2
        num = (put(t.double() + s * d) - put(t.double() - s * d)) / (2 * s)
        got = (grad.double() * d).sum()
        assert abs(float(num - got)) <= 1e-4 * float((grad.double() * d).abs().sum())


# ---- rotary positions ----
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("T,Hq,Hk,D,sec,per_axis,inter", [
    (1, 1, 0, 2, (1,), False, False), (52, 8, 8, 64, (8, 24), True, False), (17, 4, 2, 80, (5, 6, 7), False, True),
    (300, 16, 4, 64, (8, 12, 12), False, False), (9, 3, 1, 128, (16, 16, 16, 16), True, True),
    (1, 32, 8, 128, (64,), False, False), (5, 2, 2, 256, (64, 64), False, False), (7, 2, 1, 36, (0, 9), True, False)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(t, T, Hq, Hk, D, sec, per_axis, inter, inverse):
    g = gen(T * D)
    q, k = randn(g, T, Hq, D, dtype=t), randn(g, T, Hk, D, dtype=t) if Hk else None
    pos = torch.randint(-(1 << 20), 1 << 20, (T, len(sec)), generator=g, device=DEV, dtype=torch.int32)
    pos[0] = 0
    qo, ko = torch.empty_like(q), torch.empty_like(k) if Hk else None
    ops.rope(q, k, pos, qo, ko, sec, 10000.0, per_axis, inter, inverse)
    for x, y in ((q, qo), (k, ko)):
        if x is None:
            continue
        want, tol = ref.rope(x, pos, sec, 10000.0, per_axis, inter, inverse)
        ref.close(y, want, tol + ref.u(t) * want.abs(), "rope")
        assert torch.equal(y[0], x[0])               # position 0


def test_rope_strides_in_place_and_back():
    g = gen(3)
    qkv = randn(g, 37, 12, 64, dtype=BF16)
    q, k = qkv[:, :8], qkv[:, 8:10]
    keep, orig = qkv[:, 10:].clone(), qkv.clone()
    pos = torch.randint(0, 500, (37, 2), generator=g, device=DEV, dtype=torch.int32)
    wq, tq = ref.rope(orig[:, :8], pos, (16, 16), 100.0, False, False, False)
    ops.rope(q, k, pos, q, k, (16, 16), base=100.0)
    ref.close(q, wq, tq + ref.u(BF16) * wq.abs())
    assert torch.equal(qkv[:, 10:], keep)
    # heads-first memory, odd offsets (single elements)
    y = torch.empty(8, 37, 65, dtype=BF16, device=DEV)[:, :, 1:].transpose(0, 1)
    ops.rope(orig[:, :8], None, pos, y, None, (16, 16), base=100.0)
    assert torch.equal(y, q)
    x = randn(g, 11, 2, 64)
    p = torch.randint(0, 1 << 30, (11, 1), generator=g, device=DEV, dtype=torch.int32)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.rope(x, None, p, a, None, (32,))
    ops.rope(a, None, p, b, None, (32,), inverse=True)
    # both turns use the same cos and sin, off by at most 7 u from a rotation, and round a few times
    assert float((b - x).abs().max()) <= 40 * ref.U32 * float(x.abs().max()) * 2
    e = torch.empty(0, 2, 64, device=DEV)
    ops.rope(e, None, torch.empty(0, 1, dtype=torch.int32, device=DEV), e, None, (32,))


# ---- attention ----
def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def attention_case(seed, lens_q, lens_k, Hq, Hk, D, t, left, right, sinks, keep=1.0, slots=None, spread=1.0):
    g = gen(seed)
    cq, ck = offsets(lens_q), offsets(slots or lens_k)
    q, k, v = (randn(g, cq[-1], Hq, D, dtype=t, scale=spread), randn(g, ck[-1], Hk, D, dtype=t, scale=spread),
               randn(g, ck[-1], Hk, D, dtype=t))
    kp = None if keep >= 1 else torch.rand(ck[-1], generator=g, device=DEV) < keep
    mask = dict(left=left, right=right, sinks=sinks, keep=kp)
    return g, q, k, v, cq, ck, (lens_k if slots else None), mask


def run_attention(q, k, v, cq, ck, len_k, mask, **kw):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attention(q, k, v, out, i32(cq), i32(ck), len_k=None if len_k is None else i32(len_k), lse=lse, err=err, **mask, **kw)
    assert int(err) == 0
    return out, lse


CASES = [
    # lens_q, lens_k, Hq, Hk, D, type, left, right, sinks, keep, slots
    ([1], [1], 1, 1, 8, BF16, -1, -1, 0, 1.0, None),
    ([5, 0, 3], [5, 0, 3], 2, 1, 64, BF16, -1, -1, 0, 1.0, None),
    ([52] * 5, [52] * 5, 8, 8, 64, BF16, -1, -1, 4, 0.7, None),
    ([129, 1, 127, 128], [129, 1, 127, 128], 4, 4, 64, F16, -1, 0, 0, 1.0, None),
    ([700, 300], [700, 300], 4, 2, 64, BF16, 100, 60, 5, 1.0, None),
    ([1000], [1000], 2, 2, 128, F16, 0, 0, 0, 1.0, None),
    ([1000], [1000], 2, 1, 128, BF16, 3, 0, 2, 0.5, None),           # windows that the mask empties
    ([513], [513], 8, 1, 40, F16, 200, -1, 0, 0.9, None),
    ([300], [300], 2, 2, 32, BF16, 17, 300, 130, 1.0, None),
    ([40, 17, 260], [100, 900, 130], 2, 2, 80, BF16, -1, 0, 0, 1.0, None),      # chunks behind a cache; more queries than keys
    ([40, 17, 260], [100, 900, 130], 4, 2, 64, F16, 64, 0, 4, 1.0, None),
    ([1] * 6, [1, 31, 32, 33, 1000, 4000], 8, 2, 128, BF16, -1, 0, 0, 1.0, [40, 31, 64, 33, 1500, 4096]),
    ([1] * 6, [1, 31, 0, 33, 1000, 4000], 8, 8, 64, F16, 500, 0, 4, 0.8, [40, 31, 64, 33, 1500, 4096]),
    ([4] * 3, [6000, 2000, 10], 4, 4, 64, BF16, -1, -1, 0, 1.0, None),          # pooling queries
    ([12], [9000], 4, 1, 64, F16, -1, -1, 0, 0.5, None),
    ([2000], [2000], 4, 1, 128, BF16, -1, -1, 0, 1.0, None),
    ([2000, 1500], [2000, 1500], 4, 2, 64, F16, 256, 256, 16, 0.95, None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][0]}x{len(c[0])}-{c[1][0]}-h{c[2]}.{c[3]}-d{c[4]}-w{c[6]}.{c[7]}.{c[8]}")
def test_attention(case):
    *base, slots = case
    _, q, k, v, cq, ck, len_k, mask = attention_case(len(str(case)), *base, slots=slots)
    out, lse = run_attention(q, k, v, cq, ck, len_k, mask)
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, len_k=len_k, **mask)
    ref.close(out, o, to, "out")
    ref.close(lse, ls, tl, "lse")
    out2, _ = run_attention(q, k, v, cq, ck, len_k, mask)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][0]}x{len(c[0])}-{c[1][0]}-h{c[2]}.{c[3]}-d{c[4]}-w{c[6]}.{c[7]}.{c[8]}")
def test_attention_backward(case):
    *base, slots = case
    g, q, k, v, cq, ck, len_k, mask = attention_case(len(str(case)), *base, slots=slots)
    out, lse = run_attention(q, k, v, cq, ck, len_k, mask)
    dout = randn(g, *q.shape, dtype=q.dtype)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    args = (i32(cq), i32(ck))
    lk = None if len_k is None else i32(len_k)
    ops.attention_backward(dout, q, k, v, out, lse, *grads, *args, len_k=lk, **mask)
    want = ref.attention(q, k, v, cq, ck, len_k=len_k, dout=dout, out=out, lse=lse, **mask)
    for i, name in enumerate(("dq", "dk", "dv")):
        w, tol = want[i], want[i + 3]
        if slots and i:                              # rows of a slot behind its length stay as they were
            rows = torch.zeros(len(w), dtype=torch.bool, device=DEV)
            for b, n in enumerate(len_k):
                rows[ck[b]:ck[b] + n] = True
            assert (grads[i][~rows] == 7).all()
            ref.close(grads[i][rows], w[rows], tol[rows], name)
        else:
            ref.close(grads[i], w, tol, name)
    again = [torch.empty_like(t) for t in (q, k, v)]
    ops.attention_backward(dout, q, k, v, out, lse, *again, *args, len_k=lk, **mask)
    rows = grads[1] != 7
    assert torch.equal(again[0], grads[0]) and torch.equal(again[1][rows], grads[1][rows])


@pytest.mark.parametrize("D,left,nq,nk", [(64, -1, 200, 200), (128, 40, 300, 300), (64, -1, 3, 500), (64, 20, 1, 700)])
def test_attention_masked_places_hold_anything(D, left, nq, nk):
    """NaN and infinities in masked keys, behind a sequence and in another sequence change nothing."""
    g, q, k, v, cq, ck, _, mask = attention_case(D + nk, [nq, nq], [nk, nk], 4, 2, D, BF16, left, 0, 3, keep=0.6)
    mask["keep"][nk - 30:nk] = False
    mask["keep"][:3] = False                         # the first tokens too
    pad = 70
    big = lambda t, n: torch.cat([t, torch.zeros(n, *t.shape[1:], dtype=t.dtype, device=DEV)])
    q, k, v = big(q, pad), big(k, pad), big(v, pad)
    mask["keep"] = torch.cat([mask["keep"], torch.ones(pad, dtype=torch.bool, device=DEV)])
    dout = randn(g, *q.shape, dtype=BF16)

    def everything():
        out, lse = run_attention(q, k, v, cq, ck, None, mask)
        grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
        ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), **mask)
        return out, lse, *grads
    clean = everything()
    bad = ~mask["keep"]
    bad[ck[-1]:] = True
    val = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min], device=DEV).to(BF16)
    n = int(bad.sum())
    for t in (k, v):
        t[bad] = val[torch.randint(0, 4, (n, *t.shape[1:]), generator=g, device=DEV)]
    q[cq[-1]:] = float("nan")
    dout[cq[-1]:] = float("nan")
    for a, b in zip(clean, everything()):
        assert torch.equal(a, b)
    for t in (clean[0], clean[2]):
        assert (t[cq[-1]:] == 7).all()               # rows behind the last sequence
    # a whole sequence of NaN beside a good one (whose masked keys, now visible, are finite again)
    mask["keep"] = None
    k[bad], v[bad] = 0.5, 0.5
    q[:cq[1]], k[:ck[1]], v[:ck[1]], dout[:cq[1]] = (float("nan"),) * 4
    for t, cu in zip(everything(), (cq, cq, cq, ck, ck)):
        assert not torch.isnan(t[cu[1]:cu[2]]).any()


def test_attention_all_masked():
    g, q, k, v, cq, ck, _, mask = attention_case(9, [150, 3], [150, 400], 2, 2, 64, BF16, -1, -1, 0)
    mask["keep"] = torch.zeros(ck[-1], dtype=torch.uint8, device=DEV)
    out, lse = run_attention(q, k, v, cq, ck, None, mask)
    assert (out == 0).all() and (lse == -torch.inf).all()
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    ops.attention_backward(randn(g, *q.shape, dtype=BF16), q, k, v, out, lse, *grads, i32(cq), i32(ck), **mask)
    assert all((t == 0).all() for t in grads)


def test_attention_strided_views_and_large_scores():
    g = gen(77)
    T, H, D = 333, 4, 64
    qkv = randn(g, T, 3, H, D, dtype=BF16, scale=4.0)
    q, k, v = qkv.unbind(1)
    hf = torch.empty(H, T, D, dtype=BF16, device=DEV).transpose(0, 1)      # heads-first output
    lse = torch.empty(T, H, device=DEV)
    ops.attention(q, k, v, hf, i32([0, T]), i32([0, T]), left=50, right=50, lse=lse)
    o, ls, to, tl = ref.attention(q, k, v, [0, T], [0, T], left=50, right=50)
    ref.close(hf, o, to)
    ref.close(lse, ls, tl)
    dqkv = torch.empty_like(qkv)
    dout = randn(g, T, H, D, dtype=BF16)
    ops.attention_backward(dout, q, k, v, hf, lse, *dqkv.unbind(1), i32([0, T]), i32([0, T]), left=50, right=50)
    want = ref.attention(q, k, v, [0, T], [0, T], left=50, right=50, dout=dout, out=hf, lse=lse)
    for i in range(3):
        ref.close(dqkv[:, i], want[i], want[i + 3])


def test_attention_gradient_against_differences():
    g, q, k, v, cq, ck, _, mask = attention_case(4, [37], [37], 2, 1, 16, F16, 9, 4, 2, keep=0.8)
    out, lse = run_attention(q, k, v, cq, ck, None, mask)
    dout = randn(g, *q.shape, dtype=F16)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), **mask)
    f = [q.double(), k.double(), v.double()]

    def _loss(a, dout, mask):
        Q, K, V = a[0].transpose(0, 1), a[1].transpose(0, 1).repeat_interleave(2, 0), a[2].transpose(0, 1).repeat_interleave(2, 0)
        ok = ref.visible(torch.arange(37, device=DEV), 37, 37, mask["left"], mask["right"], mask["sinks"], mask["keep"], DEV)
        S = (Q @ K.transpose(1, 2) * 0.25).masked_fill(~ok, -torch.inf)
        P = torch.where(ok.any(1)[None, :, None], S.softmax(2), 0.0).nan_to_num(0.0)
        return ((P @ V).transpose(0, 1) * dout.double()).sum()
    for i in range(3):
        d = randn(g, *f[i].shape).double()
        s = 1e-5
        hi, lo = list(f), list(f)
        hi[i], lo[i] = f[i] + s * d, f[i] - s * d
        num = (_loss(hi, dout, mask) - _loss(lo, dout, mask)) / (2 * s)
        got = (grads[i].double() * d).sum()
        # every gradient element is off by a few roundings of 16 bits (P, dS, out, the result)
        assert abs(float(num - got)) <= 8 * ref.u(F16) * float((grads[i].double() * d).abs().sum() + (dout.double().abs().sum()))


def test_attention_offsets_outside_the_tensors():
    """A sequence that leaves the tensors counts as empty and is reported; the others are computed."""
    g, q, k, v, cq, ck, _, mask = attention_case(8, [20, 30], [20, 30], 2, 2, 64, BF16, -1, -1, 0)
    want, _ = run_attention(q, k, v, cq, ck, None, mask)
    for bad_q, bad_k, lk in (([0, 20, 51], ck, None), (cq, [0, 20, 5000], None), ([0, 20, -7], ck, None), (cq, ck, [20, 31]),
                             (cq, ck, [20, -1])):
        out, lse = torch.full_like(q, 7.0), torch.zeros(50, 2, device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.attention(q, k, v, out, i32(bad_q), i32(bad_k), len_k=None if lk is None else i32(lk), err=err, lse=lse)
        assert int(err) == 4
        assert torch.equal(out[:20], want[:20])
        grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
        err.zero_()
        ops.attention_backward(q, q, k, v, out, lse, *grads, i32(bad_q), i32(bad_k), len_k=None if lk is None else i32(lk), err=err)
        assert int(err) == 4


@pytest.mark.parametrize("what", ["capture", "stream"])
def test_attention_captured_and_on_another_stream(what):
    """A captured call replays on new contents; a call given a stream runs there, workspace included."""
    g, q, k, v, cq, ck, _, mask = attention_case(6, [3, 2], [5000, 7000], 4, 2, 64, BF16, -1, -1, 0)
    cu_q, cu_k = i32(cq), i32(ck)
    out, lse = torch.zeros_like(q), torch.zeros(5, 4, device=DEV)
    x, w = randn(g, 64, 256), randn(g, 256)
    y, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)
    mean, rstd = torch.empty(64, device=DEV), torch.empty(64, device=DEV)
    grads = [torch.zeros_like(t) for t in (q, k, v)]

    def calls(stream=None):
        ops.attention(q, k, v, out, cu_q, cu_k, lse=lse, stream=stream)
        ops.attention_backward(q, q, k, v, out, lse, *grads, cu_q, cu_k, stream=stream)
        ops.layer_norm(x, w, None, y, mean=mean, rstd=rstd, stream=stream)
        ops.layer_norm_backward(y, x, w, mean, rstd, dx, dw, stream=stream)
    calls()
    want = [t.clone() for t in (out, lse, *grads, y, dx, dw)]
    for t in (out, lse, *grads, y, dx, dw):
        t.zero_()
    torch.cuda.synchronize()
    if what == "stream":
        s = torch.cuda.Stream()
        calls(s)
        s.synchronize()
    else:
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for gr in graphs:                            # two graphs of the same call: workspaces of their own
            with torch.cuda.graph(gr):
                calls()
        s = torch.cuda.Stream()
        graphs[0].replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[1].replay()
        torch.cuda.synchronize()
    for a, b in zip(want, (out, lse, *grads, y, dx, dw)):
        assert torch.equal(a, b)
