"""What a call has written is there for the very next kernel, in a captured graph too: calls with few rows whose second
kernel has nothing to add up."""
from __future__ import annotations

import pytest
import torch

import context_ref as ref
from rsna_knee_efficiency_b200 import ops
from test_gpu_context_ops import BF16, DEV, attention_case, i32

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
