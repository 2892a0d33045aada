"""Attention whose walks are cut into shares: few heads over long sequences, some tens of queries over long
caches, in both directions, against the 64-bit restatement."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, attention_case, i32, randn, run_attention

pytestmark = pytest.mark.gpu

CASES = [
    # lens_q, lens_k, Hq, Hk, D, type, left, right, sinks, keep, slots
    ([5000], [5000], 1, 1, 80, BF16, -1, -1, 1, 0.8, None),
    ([3022, 28], [3022, 28], 8, 2, 80, BF16, 479, -1, 4, 1.0, None),
    ([1, 2900, 4], [1, 2900, 4], 8, 4, 128, F16, -1, 0, 0, 1.0, None),
    ([2000], [9000], 1, 1, 64, F16, -1, 0, 0, 1.0, None),
    ([300], [20000], 4, 1, 128, F16, 2500, 0, 130, 0.9, None),           # a chunk behind a long cache
    ([300, 1], [9000, 3], 2, 2, 64, BF16, 2500, 100, 700, 1.0, None),    # shares that begin among the first tokens
    ([12] * 6, [20, 1, 3312, 16114, 0, 777], 8, 2, 64, BF16, -1, -1, 4, 1.0, [23, 1, 4000, 16200, 5, 800]),
    ([33] * 3, [4100, 16, 6000], 2, 2, 128, BF16, -1, -1, 0, 0.7, [4200, 16, 6100]),
    ([700] * 3, [130, 5000, 0], 2, 2, 64, BF16, -1, 0, 0, 1.0, None),    # queries before the first key see nothing
    ([1500] * 2, [1500] * 2, 2, 1, 32, F16, 300, 20, 5, 0.6, None),
]
IDS = [f"{c[0][0]}x{len(c[0])}-{max(c[1])}-h{c[2]}.{c[3]}-d{c[4]}-w{c[6]}.{c[7]}.{c[8]}" for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_cut_attention(case):
    *base, slots = case
    _, q, k, v, cq, ck, len_k, mask = attention_case(len(str(case)), *base, slots=slots)
    out, lse = run_attention(q, k, v, cq, ck, len_k, mask)
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, len_k=len_k, **mask)
    ref.close(out, o, to, "out")
    ref.close(lse, ls, tl, "lse")
    for _ in range(3):
        again, lse2 = run_attention(q, k, v, cq, ck, len_k, mask)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_cut_attention_backward(case):
    *base, slots = case
    g, q, k, v, cq, ck, len_k, mask = attention_case(len(str(case)), *base, slots=slots)
    out, lse = run_attention(q, k, v, cq, ck, len_k, mask)
    dout = randn(g, *q.shape, dtype=q.dtype)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    lk = None if len_k is None else i32(len_k)
    want = ref.attention(q, k, v, cq, ck, len_k=len_k, dout=dout, out=out, lse=lse, **mask)
    live = torch.ones(len(k), dtype=torch.bool, device=DEV)
    if slots:                                        # rows of a slot behind its length stay as they were
        live[:] = False
        for b, n in enumerate(len_k):
            live[ck[b]:ck[b] + n] = True
    first = None
    for _ in range(3):
        grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
        ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), len_k=lk, err=err, **mask)
        assert int(err) == 0
        for i, name in enumerate(("dq", "dk", "dv")):
            rows = live if i else slice(None)
            ref.close(grads[i][rows], want[i][rows], want[i + 3][rows], name)
            if i:
                assert (grads[i][~live] == 7).all()
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, grads))
        first = grads


def test_cut_attention_offsets_that_go_back():
    """Offsets that go back over rows ask for more shares than there is room for: reported, inside the workspace."""
    _, q, k, v, _, _, _, _ = attention_case(5, [2000], [2000], 1, 1, 64, BF16, -1, -1, 0)
    bad = i32([0, 2000] * 6)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = torch.empty_like(q), torch.empty(2000, 1, device=DEV)
    ops.attention(q, k, v, out, bad, bad, lse=lse, err=err)
    assert int(err) == 4
    err.zero_()
    good = i32([0, 2000])
    ops.attention(q, k, v, out, good, good, lse=lse, err=err)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    ops.attention_backward(q, q, k, v, out, lse, *grads, bad, bad, err=err)
    assert int(err) == 4


def many(n, seed, most):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most, (n,), generator=g).tolist()


# batches around the number of sequences that a block keeps at hand, with a long one among the short ones
MANY = [(many(128, 1, 90), None, 2, 1, 64, -1, -1), (many(129, 2, 90), None, 2, 2, 64, 30, 0), (many(300, 3, 70), None, 1, 1, 128, -1, 0),
        (many(200, 4, 20) + [900], many(200, 5, 50) + [9000], 1, 1, 64, -1, -1), ([1] * 140, many(139, 6, 300) + [12000], 4, 1, 64, -1, 0),
        ([700] + [0] * 150, [5000] + [3] * 150, 2, 1, 64, -1, -1)]


@pytest.mark.parametrize("lens_q,lens_k,Hq,Hk,D,left,right", MANY, ids=[f"{len(m[0])}-{m[2]}.{m[3]}-d{m[4]}" for m in MANY])
def test_many_sequences(lens_q, lens_k, Hq, Hk, D, left, right):
    g, q, k, v, cq, ck, _, mask = attention_case(len(lens_q), lens_q, lens_k or lens_q, Hq, Hk, D, BF16, left, right, 0)
    out, lse = run_attention(q, k, v, cq, ck, None, mask)
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, **mask)
    ref.close(out, o, to, "out")
    ref.close(lse, ls, tl, "lse")
    dout = randn(g, *q.shape, dtype=BF16)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    ops.attention_backward(dout, q, k, v, out, lse, *grads, i32(cq), i32(ck), err=err, **mask)
    assert int(err) == 0
    want = ref.attention(q, k, v, cq, ck, dout=dout, out=out, lse=lse, **mask)
    for a, w, tol, name in zip(grads, want[:3], want[3:], ("dq", "dk", "dv")):
        ref.close(a, w, tol, name)
