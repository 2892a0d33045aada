"""Plain 64-bit restatements of the context transformer's operators, each with a bound on how far a
32-bit implementation that rounds where the operators say may be off (u: unit roundoffs)."""
from __future__ import annotations

import torch

U32 = 2.0 ** -24


def u(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def eta(dtype: torch.dtype) -> float:
    """Below the normal range a rounding is off by half the smallest subnormal (fp16: 2^-25), however
    small the value."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor, what: str = "") -> None:
    g = got.double()
    assert not torch.isnan(g).any(), f"{what}: NaN"
    bad = ((g - want).abs() > tol) & ~(torch.isinf(want) & (g == want))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((g - want).abs() / tol.clamp_min(1e-300))[bad].max()):.2f} x the bound at "
                           f"{bad.nonzero()[0].tolist()}")


def layer_norm(x, w, b, eps, res=None):
    """(h, y, mean, rstd, bound on y without y's own rounding, bounds on mean and rstd)."""
    h = x.double() if res is None else (x.double() + res.double()).to(x.dtype).double()
    mu = h.mean(1, keepdim=True)
    r = ((h - mu).square().mean(1, keepdim=True) + eps).rsqrt()
    xh = (h - mu) * r
    w64 = torch.ones(h.shape[1], dtype=torch.float64, device=h.device) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    # A sum of C terms: at most C / 512 (long rows) or 32 in a thread, 5 + 4 in the tree, 16 warps: K
    # roundings, each of a partial sum <= sum |h|, so |mu| is off by K u mean|h|. The variance is a
    # sum of positive terms (K u relative), r half of that and 2 ulp for rsqrt; the shift of mu enters
    # it in second order, (K u max|h| r)^2, which counts where a row is nearly constant.
    K = 64 + h.shape[1] / 256
    dmu = K * U32 * h.abs().mean(1, keepdim=True)
    dr = K * U32 + (dmu * r).square()
    tol = ((dmu + U32 * (h - mu).abs()) * r + (dr + 3 * U32) * xh.abs()) * w64.abs() + 2 * U32 * b64.abs()
    return h, xh * w64 + b64, mu[:, 0], r[:, 0], tol, dmu[:, 0] + 1e-40, (dr * r)[:, 0]


def layer_norm_backward(dy, h, w, mean, rstd, dsum=None):
    """(dx, dw, db, bounds) for the given statistics."""
    h, dy = h.double(), dy.double()
    r = rstd.double()[:, None]
    xh = (h - mean.double()[:, None]) * r
    w64 = torch.ones(h.shape[1], dtype=torch.float64, device=h.device) if w is None else w.double()
    g = dy * w64
    a, c = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - a - xh * c)
    K = 64 + h.shape[1] / 256
    ea, ec = K * U32 * g.abs().mean(1, keepdim=True), (K + 4) * U32 * (g * xh).abs().mean(1, keepdim=True)
    tol = r * (ea + xh.abs() * ec + 6 * U32 * (g.abs() + a.abs() + (xh * c).abs()))
    if dsum is not None:
        dx = dx + dsum.double()
        tol = tol + U32 * (dsum.double().abs() + dx.abs())
    # rows of a column: M / 296 in a thread at most, 8 teams, 10 + 5 in the last sum
    L = 64 + h.shape[0] / 32
    tw, tb = (L + 4) * U32 * (dy * xh).abs().sum(0), L * U32 * dy.abs().sum(0)
    return dx, (dy * xh).sum(0), dy.sum(0), tol, tw, tb


def rope(x, pos, sections, base, per_axis, interleaved, inverse):
    """(y, bound): pairs turned one after the other."""
    y, tol = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    P, j = sum(sections), 0
    for ax, n in enumerate(sections):
        for i in range(n):
            f = base ** (-(i / n)) if per_axis else base ** (-(j / P))
            ang = pos[:, ax].double() * f * (-1.0 if inverse else 1.0)
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + P)
            a, b = x[..., lo].double(), x[..., hi].double()
            y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
            # the angle: 32 roundings of 64 bits on the frequency and the product (here and there), one of
            # 32 bits on the fraction of a half turn (<= pi u); sin / cos of a half turn: 2 ulp
            da = ang.abs()[:, None] * 64 * 2.0 ** -53 + 3.2 * U32 + 4 * U32
            t = (a.abs() + b.abs()) * (da + 2 * U32)
            tol[..., lo], tol[..., hi] = t, t
            j += 1
    return y, tol


def visible(i, nq, nk, left, right, sinks, keep, device):
    p = i[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None]
    ok = torch.ones(len(i), nk, dtype=torch.bool, device=device)
    if right >= 0:
        ok = ok & (j <= p + right)
    if left >= 0:
        ok = ok & ((j >= p - left) | (j < sinks))
    return ok if keep is None else ok & keep[None].bool()


# exp2 by the special function unit or by a polynomial: relative error below 2^-17
E_EXP = 2.0 ** -17


def attention(q, k, v, cu_q, cu_k, left=-1, right=-1, sinks=0, keep=None, len_k=None, scale=None, dout=None,
              out=None, lse=None):
    """Forward: (out, lse, bound on out, bound on lse); with dout (and the forward pass's out, lse):
    (dq, dk, dv and their bounds). Offsets are lists; rows of no sequence stay zero."""
    Tq, Hq, D = q.shape
    Hk = k.shape[1]
    G, scale = Hq // Hk, D ** -0.5 if scale is None else scale
    u16, e16 = u(q.dtype), eta(q.dtype)
    dev = q.device
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)
    if dout is None:
        o, to = z(q), z(q)
        ls, tl = (torch.zeros(Tq, Hq, dtype=torch.float64, device=dev) for _ in range(2))
    else:
        dq, tq, dk, tk, dv, tv = z(q), z(q), z(k), z(k), z(v), z(v)
    for b in range(len(cu_q) - 1):
        q0, q1, k0 = cu_q[b], cu_q[b + 1], cu_k[b]
        nk = len_k[b] if len_k is not None else cu_k[b + 1] - k0
        nq = q1 - q0
        if nq == 0:
            continue
        kp = None if keep is None else keep[k0:k0 + nk]
        ok = visible(torch.arange(nq, device=dev), nq, nk, left, right, sinks, kp, dev)
        seen = ok.any(0)
        for h in range(Hq):
            Q = q[q0:q1, h].double()
            K, V = (torch.where(seen[:, None], t[k0:k0 + nk, h // G].double(), 0.0) for t in (k, v))
            S = (Q @ K.T) * scale
            # scores: D products added in 32 bits, two roundings for the scale
            dS = (D + 4) * U32 * (Q.abs() @ K.abs().T) * abs(scale)
            S = S.masked_fill(~ok, -torch.inf)
            empty = ~ok.any(1)
            if dout is None:
                L = torch.logsumexp(S, 1) if nk else torch.full((nq,), -torch.inf, dtype=torch.float64, device=dev)
                P = torch.where(ok, (S - L[:, None]).exp(), 0.0)
                # a weight is off by its score's error, the reference maximum's and the exponential's, and
                # by its rounding; 8 + nk / 64 for the sums of weights and products
                rel = 2 * (dS * ok).amax(1, keepdim=True) if nk else torch.zeros(nq, 1, dtype=torch.float64, device=dev)
                rel = rel + 2 * E_EXP + (64 + nk / 32) * U32
                smax = torch.where(ok, S.abs(), 0.0).amax(1, keepdim=True) if nk else torch.zeros_like(rel)
                rel = rel + 4 * U32 * smax
                o[q0:q1, h] = P @ V
                to[q0:q1, h] = (rel + u16 * 1.01) * (P @ V.abs()) + e16 * (ok.double() @ V.abs() + 1) + u16 * (P @ V).abs()
                ls[q0:q1, h] = torch.where(empty, -torch.inf, L)
                tl[q0:q1, h] = rel[:, 0] + 2 * U32 * torch.where(empty, 0.0, L).abs()
                continue
            L = lse[q0:q1, h].double()[:, None]
            live = ok & ~torch.isinf(L)
            P = torch.where(live, (S - L).exp(), 0.0)
            Do = torch.where(empty[:, None], 0.0, dout[q0:q1, h].double())
            O = torch.where(empty[:, None], 0.0, out[q0:q1, h].double())
            Qz = torch.where(empty[:, None], 0.0, Q)
            delta, dP = (Do * O).sum(1, keepdim=True), Do @ V.T
            G_ = P * (dP - delta) * scale
            rel = torch.where(live, dS, 0.0) + E_EXP + 4 * U32 * (S.abs().masked_fill(~live, 0.0) + L.abs().masked_fill(
                torch.isinf(L), 0.0)) + 8 * U32
            eP = P * (rel + u16 * 1.01) + live * e16
            eG = G_.abs() * (rel + u16 * 1.01 + 8 * U32) + 1.01 * P * abs(scale) * (D + 4) * U32 * (
                Do.abs() @ V.abs().T + (Do * O).abs().sum(1, keepdim=True)) + live * e16
            acc = lambda n: (64 + n / 32) * U32
            dq[q0:q1, h] = G_ @ K
            tq[q0:q1, h] = (eG + acc(nk) * G_.abs()) @ K.abs() + u16 * (G_ @ K).abs() + e16
            kr = slice(k0, k0 + nk)
            dk[kr, h // G] += G_.T @ Qz
            tk[kr, h // G] += (eG + acc(nq * G) * G_.abs()).T @ Qz.abs()
            dv[kr, h // G] += P.T @ Do
            tv[kr, h // G] += (eP + acc(nq * G) * P).T @ Do.abs()
    if dout is None:
        return o, ls, to, tl
    return dq, dk, dv, tq, tk + u16 * dk.abs() + e16, tv + u16 * dv.abs() + e16
