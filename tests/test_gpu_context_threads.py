"""Two host threads, a stream each, calling every operator at the same time: each gets what it gets alone."""
from __future__ import annotations

import threading

import pytest
import torch

from rsna_knee_efficiency_b200 import ops
from test_gpu_context_limits import CALLS
from test_gpu_context_ops import BF16, DEV, attention_case, gen, i32, randn

pytestmark = pytest.mark.gpu


def program(n):
    """(inputs, a function that runs every operator on them and returns the outputs)"""
    calls = []
    for x, (lens_q, lens_k, Hq, Hk, D, left, right, sinks) in enumerate(CALLS[::1 if n % 2 else -1]):
        g, q, k, v, cq, ck, _, mask = attention_case(10 * n + x, lens_q, lens_k, Hq, Hk, D, BF16, left, right, sinks)
        calls.append((q, k, v, i32(cq), i32(ck), mask, randn(g, *q.shape, dtype=BF16)))
    g = gen(n)
    C = (768, 1664)[n % 2]
    x, w, pos = randn(g, 500, C, dtype=BF16), randn(g, C), torch.randint(0, 900, (500, 2), generator=g, device=DEV, dtype=torch.int32)

    def run():
        outs = []
        for q, k, v, cu_q, cu_k, mask, dout in calls:
            out, lse, grads = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV), [torch.empty_like(t) for t in (q, k, v)]
            ops.attention(q, k, v, out, cu_q, cu_k, lse=lse, **mask)
            ops.attention_backward(dout, q, k, v, out, lse, *grads, cu_q, cu_k, **mask)
            outs += [out, lse, *grads]
        y, mean, rstd = torch.empty_like(x), torch.empty(500, device=DEV), torch.empty(500, device=DEV)
        ops.layer_norm(x, w, w, y, mean=mean, rstd=rstd)
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        ops.layer_norm_backward(y, x, w, mean, rstd, dx, dw, db)
        h = torch.empty(500, C // 64, 64, dtype=BF16, device=DEV)
        ops.rope(x.view(500, C // 64, 64), None, pos, h, None, (8, 24))
        return outs + [y, dx, dw, db, h]
    return run


def test_two_host_threads():
    runs = [program(n) for n in range(2)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    failed, go = [], threading.Barrier(2, timeout=60)

    def work(n):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                go.wait()
                for _ in range(15):
                    got = runs[n]()
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[n])):
                        failed.append(n)
                s.synchronize()
        except Exception as e:                               # (an exception in a thread would pass unseen)
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[:3]
