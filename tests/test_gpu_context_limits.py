"""Calls of the context operators at the edges of what they take: rows beyond 32-bit offsets, workspaces that
the caller gives, streams side by side, captured calls whose walks are cut, other scales, refusals."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import _native as nat
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, attention_case, gen, i32, randn, run_attention

pytestmark = pytest.mark.gpu


def gradients(dout, q, k, v, out, lse, cq, ck, mask, **kw):
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), err=err, **mask, **kw)
    assert int(err) == 0
    return grads


def test_rows_beyond_32_bits():
    """Rows 61440 elements apart: the last ones lie 8.6 GB behind the first."""
    g = gen(1)
    rows, far = 70000, 61440
    buf = torch.empty(rows, far, dtype=BF16, device=DEV)
    buf[:, :512] = randn(g, rows, 512, dtype=BF16)
    assert (rows - 1) * far > 1 << 31
    k, v, q, o = (buf[:, x:x + 128].view(rows, 2, 64) for x in (0, 128, 256, 384))
    # single tokens and pooling queries (row kernel), then a tile of queries, over the last keys
    for nq, nk in ((3, 69000), (300, 5000)):
        cq, ck = [0, nq], [rows - nk, rows]
        qs = q[rows - nq:]
        out, lse = o[rows - nq:], torch.empty(nq, 2, device=DEV)
        ops.attention(qs, k, v, out, i32(cq), i32(ck), lse=lse)
        want, wl, to, tl = ref.attention(qs.contiguous(), k[rows - nk:].contiguous(), v[rows - nk:].contiguous(), cq, [0, nk])
        ref.close(out, want, to, "out")
        ref.close(lse, wl, tl, "lse")
    nq = nk = 400
    cq = [rows - nq, rows]
    lse = torch.empty(rows, 2, device=DEV)
    ops.attention(q, k, v, o, i32(cq), i32(cq), lse=lse, right=0)
    dout = randn(g, nq, 2, 64, dtype=BF16)
    s = slice(rows - nq, rows)
    want = ref.attention(q[s].contiguous(), k[s].contiguous(), v[s].contiguous(), [0, nq], [0, nk], right=0, dout=dout,
                         out=o[s].contiguous(), lse=lse[s].contiguous())
    dfull = torch.zeros(rows, 2, 64, dtype=BF16, device=DEV)
    dfull[s] = dout
    dq, dk, dv = (buf[:, x:x + 128].view(rows, 2, 64) for x in (512, 640, 768))
    buf[:, 512:896] = 7
    ops.attention_backward(dfull, q, k, v, o, lse, dq, dk, dv, i32(cq), i32(cq), right=0)
    for got, w, tol in zip((dq, dk, dv), want[:3], want[3:]):
        ref.close(got[s], w, tol)
        assert (got[:rows - nq] == 7).all()
    # rope and layer norm over the same rows
    pos = torch.randint(0, 100000, (rows, 1), generator=g, device=DEV, dtype=torch.int32)
    ops.rope(q, None, pos, dq, None, (32,))
    w, tol = ref.rope(q[-50:].contiguous(), pos[-50:], (32,), 10000.0, False, False, False)
    ref.close(dq[-50:], w, tol + ref.u(BF16) * w.abs())
    x, y = buf[:, :128], buf[:, 640:768]
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    ops.layer_norm(x, None, None, y, mean=mean, rstd=rstd)
    _, w, _, _, tol, _, _ = ref.layer_norm(x[-50:].contiguous(), None, None, 1e-5)
    ref.close(y[-50:], w, tol + ref.u(BF16) * w.abs())
    dx = buf[:, 768:896]
    ops.layer_norm_backward(y, x, None, mean, rstd, dx)
    w, _, _, tol, _, _ = ref.layer_norm_backward(y[-50:].contiguous(), x[-50:].contiguous(), None, mean[-50:], rstd[-50:])
    ref.close(dx[-50:], w, tol * 1.01 + ref.u(BF16) * w.abs())


@pytest.mark.parametrize("lens_q,lens_k,Hq,Hk,D,t", [([1] * 5, [9, 1, 700, 0, 3001], 6, 2, 72, F16), ([200, 3], [200, 3], 2, 2, 8, BF16),
                                                     ([12, 1], [4000, 12], 8, 2, 24, F16), ([700], [700], 2, 1, 104, BF16)])
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scales_and_odd_head_sizes(lens_q, lens_k, Hq, Hk, D, t, scale):
    g, q, k, v, cq, ck, _, mask = attention_case(D, lens_q, lens_k, Hq, Hk, D, t, -1, -1, 0)
    out, lse = run_attention(q, k, v, cq, ck, None, mask, scale=scale)
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, scale=scale, **mask)
    ref.close(out, o, to, "out")
    ref.close(lse, ls, tl, "lse")
    dout = randn(g, *q.shape, dtype=t)
    got = gradients(dout, q, k, v, out, lse, cq, ck, mask, scale=scale)
    want = ref.attention(q, k, v, cq, ck, scale=scale, dout=dout, out=out, lse=lse, **mask)
    for a, w, tol, name in zip(got, want[:3], want[3:], ("dq", "dk", "dv")):
        ref.close(a, w, tol, name)


# few rows, a cut walk, the first tokens' shares, an uncut walk
CALLS = [([1, 2], [5000, 7000], 4, 2, 64, -1, -1, 0), ([700], [4100], 4, 1, 64, -1, 0, 0), ([5000], [5000], 8, 8, 64, 100, 0, 5),
         ([300, 200], [300, 200], 8, 8, 128, -1, -1, 0)]


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_given_workspaces(call):
    lens_q, lens_k, Hq, Hk, D, left, right, sinks = call
    g, q, k, v, cq, ck, _, mask = attention_case(2, lens_q, lens_k, Hq, Hk, D, BF16, left, right, sinks)
    out, lse = run_attention(q, k, v, cq, ck, None, mask)
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, **mask)
    ref.close(out, o, to, "out")
    dout = randn(g, *q.shape, dtype=BF16)
    grads = gradients(dout, q, k, v, out, lse, cq, ck, mask)
    for a, w, tol in zip(grads, *[ref.attention(q, k, v, cq, ck, dout=dout, out=out, lse=lse, **mask)[x:x + 3] for x in (0, 3)]):
        ref.close(a, w, tol)
    # full of NaN: nothing is read before it is written
    work = torch.full((256 << 20,), 0xFF, dtype=torch.uint8, device=DEV)
    out2, lse2 = run_attention(q, k, v, cq, ck, None, mask, work=work)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    work.fill_(0xFF)
    assert all(torch.equal(a, b) for a, b in zip(grads, gradients(dout, q, k, v, out, lse, cq, ck, mask, work=work)))
    with pytest.raises(ValueError):
        gradients(dout, q, k, v, out, lse, cq, ck, mask, work=work[:16])
    with pytest.raises(ValueError):
        gradients(dout, q, k, v, out, lse, cq, ck, mask, work=work[1:])


def test_streams_side_by_side():
    """Two programs on two streams, with calls of every kind, end with what each gives alone."""
    made = []
    for n, (lens_q, lens_k, Hq, Hk, D, left, right, sinks) in enumerate(CALLS):
        g, q, k, v, cq, ck, _, mask = attention_case(n, lens_q, lens_k, Hq, Hk, D, F16, left, right, sinks)
        out, lse = run_attention(q, k, v, cq, ck, None, mask)
        dout = randn(g, *q.shape, dtype=F16)
        made.append((q, k, v, i32(cq), i32(ck), mask, out, lse, dout, gradients(dout, q, k, v, out, lse, cq, ck, mask)))
    x, w = randn(gen(9), 3000, 512, dtype=BF16), randn(gen(8), 512)
    torch.cuda.synchronize()
    streams, kept = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(6):
        for s, order in zip(streams, (made, made[::-1])):
            with torch.cuda.stream(s):
                for q, k, v, cq, ck, mask, out, lse, dout, grads in order:
                    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
                    ops.attention(q, k, v, o2, cq, ck, lse=l2, **mask)
                    g2 = [torch.empty_like(t) for t in grads]
                    ops.attention_backward(dout, q, k, v, o2, l2, *g2, cq, ck, **mask)
                    kept.append((out, o2, lse, l2, grads, g2))
                y, mean, rstd = torch.empty_like(x), torch.empty(3000, device=DEV), torch.empty(3000, device=DEV)
                ops.layer_norm(x, w, w, y, mean=mean, rstd=rstd)
                dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
                ops.layer_norm_backward(y, x, w, mean, rstd, dx, dw, db)
                kept.append((y, dx, dw))
    torch.cuda.synchronize()
    norms = [k for k in kept if len(k) == 3]
    assert all(torch.equal(a, b) for n in norms for a, b in zip(n, norms[0]))
    for out, o2, lse, l2, grads, g2 in (k for k in kept if len(k) == 6):
        assert torch.equal(out, o2) and torch.equal(lse, l2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


@pytest.mark.parametrize("call", CALLS, ids=str)
def test_captured_cut_calls_read_lengths_when_they_run(call):
    """A graph of a call on cache slots, replayed after the lengths have changed."""
    lens_q, lens_k, Hq, Hk, D, left, right, sinks = call
    g, q, k, v, cq, ck, _, mask = attention_case(4, lens_q, lens_k, Hq, Hk, D, BF16, left, right, sinks)
    cu_q, cu_k, ln = i32(cq), i32(ck), i32(lens_k)
    out, lse, err = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    dout, grads = randn(g, *q.shape, dtype=BF16), [torch.zeros_like(t) for t in (q, k, v)]

    def run():
        ops.attention(q, k, v, out, cu_q, cu_k, len_k=ln, lse=lse, err=err, **mask)
        ops.attention_backward(dout, q, k, v, out, lse, *grads, cu_q, cu_k, len_k=ln, err=err, **mask)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lens in (lens_k, [1] * len(lens_k), [n - n // 3 for n in lens_k], [0] * len(lens_k)):
        ln.copy_(i32(lens))
        graph.replay()
        assert int(err) == 0
        ow, lw, to, tl = ref.attention(q, k, v, cq, ck, len_k=lens, **mask)
        ref.close(out, ow, to, "out")
        ref.close(lse, lw, tl, "lse")
        want = ref.attention(q, k, v, cq, ck, len_k=lens, dout=dout, out=out, lse=lse, **mask)
        live = torch.cat([torch.arange(c, c + n, device=DEV) for c, n in zip(ck, lens)])
        ref.close(grads[0], want[0], want[3], "dq")
        for i in (1, 2):
            ref.close(grads[i][live], want[i][live], want[i + 3][live], "dk, dv")


def test_refusals():
    g, q, k, v, cq, ck, _, mask = attention_case(1, [5], [5], 2, 2, 64, BF16, -1, -1, 0)
    out, cu = torch.empty_like(q), i32(cq)
    bad = [
        dict(q=q.float()), dict(k=k.half()), dict(out=out[:4]), dict(k=k[:, :1]), dict(v=v[:4]), dict(q=q.cpu()), dict(cu_q=cu.long()),
        dict(cu_q=cu.cpu()), dict(cu_k=i32([0, 2, 5])), dict(k=k[:1].expand(5, 2, 64)), dict(q=q[:, :, ::2]), dict(left=-2),
        dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(keep=torch.ones(4, dtype=torch.bool, device=DEV)),
        dict(keep=torch.ones(5, device=DEV)), dict(len_k=i32([1, 2])), dict(lse=torch.empty(5, 3, device=DEV)),
        dict(lse=torch.empty(5, 2, device=DEV, dtype=F16)), dict(err=torch.zeros(1, device=DEV)),
        dict(q=torch.empty(5, 2, 65, dtype=BF16, device=DEV)[:, :, 1:]),
    ]
    for change in bad:
        a = dict(q=q, k=k, v=v, out=out, cu_q=cu, cu_k=cu)
        a.update(change)
        with pytest.raises((ValueError, TypeError, nat.Dn8Error)):
            ops.attention(**a)
    want = run_attention(q, k, v, cq, ck, None, mask)[0]
    assert want.isfinite().all()                     # the context is as it was
    far = dict(left=1 << 40, right=1 << 30, sinks=1 << 35)      # limits beyond every length are none
    assert torch.equal(want, run_attention(q, k, v, cq, ck, None, far)[0])
