"""What a call has written is there for the very next kernel, in a captured graph too: calls with few rows whose second
kernel has nothing to add up, and calls of many pieces of one key tile."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, F16, attention_case, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,nq,nk,Hq,Hk,D", [(24, 4, 52, 4, 4, 64), (8, 1, 500, 8, 2, 128), (40, 3, 52, 8, 2, 64)])
@pytest.mark.parametrize("captured", [False, True])
def test_reader_behind_a_call_that_is_not_cut(n, nq, nk, Hq, Hk, D, captured):
    """Pooling queries of many short studies: no walk is long enough to be cut, so the kernel that adds shares up has
    nothing to do. `out` is cleared before the call and copied right behind it, many times in a row."""
    _, q, k, v, cq, ck, _, mask = attention_case(n, [nq] * n, [nk] * n, Hq, Hk, D, BF16, -1, -1, 0)
    cu_q, cu_k, times = i32(cq), i32(ck), 20
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    seen = [torch.zeros_like(q) for _ in range(times)]
    seen_lse = [torch.zeros_like(lse) for _ in range(times)]

    def run():
        for o2, l2 in zip(seen, seen_lse):
            out.fill_(7.0)
            lse.fill_(7.0)
            ops.attention(q, k, v, out, cu_q, cu_k, lse=lse, **mask)
            torch.mul(out, 1.0, out=o2)
            torch.mul(lse, 1.0, out=l2)
    run()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for t in (*seen, *seen_lse):
            t.zero_()
        for _ in range(5):
            graph.replay()
    o, ls, to, tl = ref.attention(q, k, v, cq, ck, **mask)
    ref.close(seen[0], o, to, "out")
    ref.close(seen_lse[0], ls, tl, "lse")
    assert all(torch.equal(a, seen[0]) for a in seen) and all(torch.equal(a, seen_lse[0]) for a in seen_lse)


@pytest.mark.parametrize("D,lens_q,lens_k,mask", [
    (64, [100] * 1500, [100] * 1500, dict(left=-1, right=0, sinks=0)), (128, [128, 65] * 600, [128, 65] * 600, dict(left=-1, right=-1, sinks=0)),
    (64, [200, 1, 90] * 400, [100, 128, 3] * 400, dict(left=-1, right=-1, sinks=0)),
    (64, [128, 90, 140] * 400, [128, 0, 140] * 400, dict(left=20, right=20, sinks=2))])
def test_pieces_of_one_key_tile_one_after_the_other(D, lens_q, lens_k, mask):
    """Thousands of pieces of one key tile each, dozens per SM (empty ones between them in the last case): the sums that
    two warps hand to each other belong to this piece, not to the next one, every time."""
    _, q, k, v, cq, ck, _, _ = attention_case(D + len(lens_q), lens_q, lens_k, 4, 4, D, F16, -1, -1, 0)
    cu_q, cu_k = i32(cq), i32(ck)
    out, lse = torch.full_like(q, 7.0), torch.empty(q.shape[:2], device=DEV)
    ops.attention(q, k, v, out, cu_q, cu_k, lse=lse, **mask)
    n = 9                                                    # the first sequences, some in the middle, the last ones
    for at in (0, len(lens_q) // 2, len(lens_q) - n):
        sq, sk = slice(cq[at], cq[at + n]), slice(ck[at], ck[at + n])
        o, ls, to, tl = ref.attention(q[sq], k[sk], v[sk], [x - cq[at] for x in cq[at:at + n + 1]],
                                      [x - ck[at] for x in ck[at:at + n + 1]], **mask)
        ref.close(out[sq], o, to, "out")
        ref.close(lse[sq], ls, tl, "lse")
    for _ in range(30):
        o2, l2 = torch.full_like(q, 7.0), torch.empty_like(lse)
        ops.attention(q, k, v, o2, cu_q, cu_k, lse=l2, **mask)
        assert torch.equal(o2, out) and torch.equal(l2, lse)
