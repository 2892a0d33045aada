"""The operators of the study's context transformer (layer norm, rotary positions with several axes,
attention with a sliding window and first tokens that stay visible) as cases to measure: plain forms in
elementary torch operations, the framework's entry points, exact results in 64 bits and the work each needs.

A study's tokens are either its windows (2 slots x 24 triplets = 48 per study, features of 1664 channels)
or the places of the encoder's last maps (16 x 16 per image at 512 px, 24 images per view = 6144 tokens).
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _text(ints):
    return ",".join(str(n) for n in ints)


def _ints(text):
    return [int(n) for n in text.split(",")]


# ---- cases --------------------------------------------------------------------------------------
def listed():
    return [
        # the features of one view (24 images) before the head: the smallest call, latency counts
        dict(name="ln_view", op="ln", rows=24, c=1664, type="f32", out="bf16", res=False),
        # the tokens of 16 views between two sublayers: sum with the residual and its norm
        dict(name="ln_tokens", op="ln", rows=98304, c=512, type="bf16", out="bf16", res=True),
        # refit of the head on INT8 features: gradient of the input norm, 16 studies of 48 windows, odd width
        dict(name="ln_bwd_odd", op="ln_bwd", rows=769, c=1663, type="f32", out="f32", res=False),
        # training over map tokens, with the gradient that comes along the residual
        dict(name="ln_bwd_tokens", op="ln_bwd", rows=98304, c=512, type="bf16", out="bf16", res=True),
        # one study: 48 windows and 4 first tokens, positions (slot, slice)
        dict(name="rope_study", op="rope", tokens=52, hq=8, hk=8, d=64, sections="8,24", type="bf16",
             interleaved=False, per_axis=True, inverse=False, far=64),
        # map tokens of 16 views, positions (slice, row, column), grouped heads
        dict(name="rope_maps", op="rope", tokens=98304, hq=16, hk=4, d=64, sections="8,12,12", type="bf16",
             interleaved=False, per_axis=False, inverse=False, far=100000),
        # the windows of 16 studies with missing slots: many short sequences
        dict(name="attn_studies", op="attn", lens=_text([52] * 16), hq=8, hk=8, d=64, type="bf16", left=-1, right=-1,
             sinks=4, keep=0.9),
        # map tokens of four views, 2 slices to each side, grouped heads
        dict(name="attn_window", op="attn", lens="6160,6160,4113,6160", hq=16, hk=4, d=64, type="bf16", left=512,
             right=512, sinks=16, keep=1.0),
        # map tokens of four views, all earlier slices
        dict(name="attn_causal", op="attn", lens="6144,6144,6144,6144", hq=8, hk=8, d=128, type="f16", left=-1, right=0,
             sinks=0, keep=1.0),
        # pooling: 4 finding queries over all tokens of a study's two views, 16 studies
        dict(name="attn_pool", op="few", nq=4, slots=_text([12288] * 16), lens=_text([12288] * 16), hq=8, hk=8, d=64,
             type="bf16", left=-1, right=-1, sinks=0),
        # one new token of each of 8 streams over caches of different fill
        dict(name="attn_step", op="few", nq=1, slots=_text([32768] * 8),
             lens="32768,20001,777,1,16384,30011,9000,25600", hq=32, hk=8, d=128, type="bf16", left=-1,
             right=0, sinks=0),
        # training step of the window attention, ragged views, grouped heads
        dict(name="attn_bwd", op="attn_bwd", lens="6160,3907,6160,1", hq=16, hk=4, d=64, type="bf16", left=512,
             right=512, sinks=16, keep=1.0),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln", "ln_bwd", "rope", "attn", "few", "attn_bwd"])
    half = rng.choice(["bf16", "f16"])
    if op in ("ln", "ln_bwd"):
        c = _logint(rng, 16, 4096)
        if rng.random() < 0.6:
            c = max(8, c // 8 * 8)
        t = rng.choice(["f32", "bf16", "f16"])
        out = rng.choice(["f32", "bf16", "f16"]) if t == "f32" else t
        return dict(op=op, rows=min(_logint(rng, 1, 98304), 50_000_000 // c), c=c, type=t, out=out,
                    res=rng.random() < 0.5)
    if op == "rope":
        d = rng.choice([32, 64, 80, 128])
        axes = rng.choice([1, 2, 3, 4])
        left, sec = d // 2, []
        for a in range(axes):
            sec.append(left if a == axes - 1 else rng.randint(1, left - (axes - 1 - a)))
            left -= sec[-1]
        if rng.random() < 0.3 and sec[-1] > 1:
            sec[-1] -= 1
        hk = rng.choice([1, 2, 4, 8])
        hq = hk * rng.choice([1, 2, 4])
        return dict(op=op, tokens=min(_logint(rng, 1, 98304), 60_000_000 // ((hq + hk) * d)), hq=hq, hk=hk, d=d,
                    sections=_text(sec), type=rng.choice(["f32", "bf16", "f16"]), interleaved=rng.random() < 0.3,
                    per_axis=rng.random() < 0.5, inverse=rng.random() < 0.4, far=_logint(rng, 64, 1 << 20))
    hk = rng.choice([1, 2, 4])
    hq = hk * rng.choice([1, 2, 4])
    d = rng.choice([32, 64, 80, 128])
    window = rng.random() < 0.6
    lo = _logint(rng, 1, 2048) if window else -1
    right = rng.choice([0, 0, -1, lo])
    if op == "few":
        b = _logint(rng, 1, 32)
        slots = [_logint(rng, 1, 30000) for _ in range(b)]
        nq = rng.choice([1, 1, 2, 4, 12])
        lens = [rng.randint(1, s) for s in slots]
        # a finding's query sees the whole study; a new token stands at the end of its cache
        return dict(op=op, nq=nq, slots=_text(slots), lens=_text(lens), hq=hq, hk=hk, d=d, type=half,
                    left=lo if nq == 1 else -1, right=0 if nq == 1 else -1, sinks=rng.choice([0, 4, 16]))
    b = rng.randint(1, 5)
    lens = [_logint(rng, 1, 6160) for _ in range(b)]
    case = dict(op=op, lens=_text(lens), hq=hq, hk=hk, d=d, type=half, left=lo, right=right,
                sinks=rng.choice([0, 1, 4, 16, 130]), keep=1.0 if op == "attn_bwd" else rng.choice([1.0, 0.8]))
    while work(case)["flops"] > 1.6e11:
        case["lens"] = _text(n // 2 + 1 for n in _ints(case["lens"]))
    return case


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    t = TYPES[case["type"]]
    st = dict(case=case)
    if op in ("ln", "ln_bwd"):
        m, c = case["rows"], case["c"]
        to = TYPES[case["out"]]
        # features are means of rectified maps: positive, each channel at its own level
        level = torch.rand(c, generator=g, device=DEV) * 2
        st["x"] = (_randn(g, m, c) * 0.7 + level).to(t)
        st["w"] = 1 + 0.1 * _randn(g, c)
        st["b"] = 0.1 * _randn(g, c)
        if op == "ln":
            st["res"] = _randn(g, m, c).to(t) if case["res"] else None
            st["sum"] = torch.empty(m, c, dtype=t, device=DEV) if case["res"] else None
            st["y"] = torch.empty(m, c, dtype=to, device=DEV)
            st["mean"] = torch.empty(m, device=DEV)
            st["rstd"] = torch.empty(m, device=DEV)
        else:
            st["dy"] = _randn(g, m, c, scale=0.1).to(to)
            st["dsum"] = _randn(g, m, c, scale=0.1).to(t) if case["res"] else None
            h = st["x"].float()
            st["mean"] = h.mean(1)
            st["rstd"] = ((h - st["mean"][:, None]).square().mean(1) + 1e-5).rsqrt()
            st["dx"] = torch.empty(m, c, dtype=t, device=DEV)
            st["dw"] = torch.empty(c, device=DEV)
            st["db"] = torch.empty(c, device=DEV)
        return st
    if op == "rope":
        n, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        # queries and keys as a fused projection leaves them: one row per token
        qkv = _randn(g, n, hq + 2 * hk, d).to(t)
        st["q"], st["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        axes = len(_ints(case["sections"]))
        st["pos"] = torch.randint(0, case["far"], (n, axes), generator=g, device=DEV, dtype=torch.int32)
        st["qo"] = torch.empty(n, hq, d, dtype=t, device=DEV)
        st["ko"] = torch.empty(n, hk, d, dtype=t, device=DEV)
        return st
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if op == "few":
        b = len(_ints(case["slots"]))
        cq, ck = [case["nq"] * i for i in range(b + 1)], _offsets(_ints(case["slots"]))
        st["len_k"] = torch.tensor(_ints(case["lens"]), dtype=torch.int32, device=DEV)
    else:
        cq = ck = _offsets(_ints(case["lens"]))
        st["len_k"] = None
    st["cq"], st["ck"] = cq, ck
    st["cu_q"] = torch.tensor(cq, dtype=torch.int32, device=DEV)
    st["cu_k"] = st["cu_q"] if op != "few" else torch.tensor(ck, dtype=torch.int32, device=DEV)
    st["q"] = _randn(g, cq[-1], hq, d, scale=1.5).to(t)
    st["k"] = _randn(g, ck[-1], hk, d).to(t)
    st["v"] = _randn(g, ck[-1], hk, d).to(t)
    st["keep"] = None
    if case.get("keep", 1.0) < 1.0:
        keep = torch.rand(ck[-1], generator=g, device=DEV) < case["keep"]
        for s in ck[:-1]:                       # a sequence's first token is always there
            keep[s] = True
        st["keep"] = keep
    st["out"] = torch.empty(cq[-1], hq, d, dtype=t, device=DEV)
    st["lse"] = torch.empty(cq[-1], hq, device=DEV)
    if op == "attn_bwd":
        o, st["lse"] = _attention_plain(st)
        st["out"] = o.to(t)
        st["dout"] = _randn(g, cq[-1], hq, d).to(t)
        st["dq"] = torch.empty(cq[-1], hq, d, dtype=t, device=DEV)
        st["dk"] = torch.empty(ck[-1], hk, d, dtype=t, device=DEV)
        st["dv"] = torch.empty(ck[-1], hk, d, dtype=t, device=DEV)
    return st


# ---- plain forms --------------------------------------------------------------------------------
def _ln_plain(st):
    h = st["x"].float()
    if st["res"] is not None:
        h = (h + st["res"].float()).to(st["x"].dtype).float()
    mean = h.mean(1, keepdim=True)
    d = h - mean
    rstd = (d.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    r = {"y": (d * rstd * st["w"] + st["b"]).to(st["y"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if st["res"] is not None:
        r["sum"] = h.to(st["x"].dtype)
    return r


def _ln_bwd_plain(st):
    h, dy, r = st["x"].float(), st["dy"].float(), st["rstd"][:, None]
    xh = (h - st["mean"][:, None]) * r
    g = dy * st["w"]
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if st["dsum"] is not None:
        dx = dx + st["dsum"].float()
    return {"dx": dx.to(st["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _ladder(case):
    """Frequencies of the pairs in 64 bits and the axis of each."""
    sec, base = _ints(case["sections"]), 10000.0
    pairs = sum(sec)
    freq, axis = [], []
    for a, n in enumerate(sec):
        for i in range(n):
            freq.append(base ** (-i / n) if case["per_axis"] else base ** (-len(freq) / pairs))
            axis.append(a)
    return freq, axis


def _rope_plain(st):
    case = st["case"]
    freq, axis = _ladder(case)
    f = torch.tensor(freq, dtype=torch.float64, device=DEV)
    # angles of far positions lose their fraction of a turn in 32 bits
    ang = st["pos"][:, axis].double() * f
    c, s = ang.cos().float()[:, None], ang.sin().float()[:, None]
    if case["inverse"]:
        s = -s
    p = len(freq)
    out = []
    for x in (st["q"], st["k"]):
        y = x.float().clone()
        i1, i2 = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if case["interleaved"] else (slice(0, p), slice(p, 2 * p))
        a, b = x[..., i1].float(), x[..., i2].float()
        y[..., i1] = a * c - b * s
        y[..., i2] = b * c + a * s
        out.append(y.to(x.dtype))
    return {"q": out[0], "k": out[1]}


def _sequences(st):
    case = st["case"]
    for b, nk in enumerate(_ints(case["lens"])):
        yield st["cq"][b], st["cq"][b + 1], st["ck"][b], st["ck"][b] + nk


def _visible(case, i0, i1, nq, nk, keep):
    p = torch.arange(i0, i1, device=DEV)[:, None] + (nk - nq)
    j = torch.arange(nk, device=DEV)[None]
    ok = torch.ones(i1 - i0, nk, dtype=torch.bool, device=DEV)
    if case["right"] >= 0:
        ok &= j <= p + case["right"]
    if case["left"] >= 0:
        ok &= (j >= p - case["left"]) | (j < case["sinks"])
    if keep is not None:
        ok &= keep[None]
    return ok


def _heads(x, group):
    """[n, h, d] -> [h * group, n, d] in 32 bits"""
    x = x.float().transpose(0, 1)
    return x if group == 1 else x.repeat_interleave(group, 0)


def _attention_plain(st, chunk=2048):
    case = st["case"]
    group, scale = case["hq"] // case["hk"], case["d"] ** -0.5
    out = torch.zeros(st["q"].shape, device=DEV)
    lse = torch.full(st["q"].shape[:2], -math.inf, device=DEV)
    for q0, q1, k0, k1 in _sequences(st):
        k, v = _heads(st["k"][k0:k1], group), _heads(st["v"][k0:k1], group)
        keep = None if st["keep"] is None else st["keep"][k0:k1]
        for i0 in range(0, q1 - q0, chunk):
            i1 = min(q1 - q0, i0 + chunk)
            s = torch.matmul(_heads(st["q"][q0 + i0:q0 + i1], 1), k.transpose(1, 2)) * scale
            s = s.masked_fill(~_visible(case, i0, i1, q1 - q0, k1 - k0, keep), -math.inf)
            top = s.amax(2, keepdim=True).clamp_min(-1e30)
            e = torch.exp(s - top)
            z = e.sum(2, keepdim=True)
            o = torch.matmul(e, v) / z.clamp_min(1e-38)
            out[q0 + i0:q0 + i1] = o.transpose(0, 1)
            lse[q0 + i0:q0 + i1] = (top + z.log())[..., 0].transpose(0, 1)
    return out, lse


def _attention_bwd_plain(st, chunk=2048):
    case = st["case"]
    hq, hk, d = case["hq"], case["hk"], case["d"]
    group, scale = hq // hk, d ** -0.5
    dq = torch.zeros(st["q"].shape, device=DEV)
    dk = torch.zeros(st["k"].shape, device=DEV)
    dv = torch.zeros(st["v"].shape, device=DEV)
    for q0, q1, k0, k1 in _sequences(st):
        k, v = _heads(st["k"][k0:k1], group), _heads(st["v"][k0:k1], group)
        gk, gv = torch.zeros_like(k), torch.zeros_like(v)
        for i0 in range(0, q1 - q0, chunk):
            i1 = min(q1 - q0, i0 + chunk)
            rows = slice(q0 + i0, q0 + i1)
            q, do, o = _heads(st["q"][rows], 1), _heads(st["dout"][rows], 1), _heads(st["out"][rows], 1)
            s = torch.matmul(q, k.transpose(1, 2)) * scale
            p = torch.exp(s - st["lse"][rows].transpose(0, 1)[..., None])
            p = p.masked_fill(~_visible(case, i0, i1, q1 - q0, k1 - k0, None), 0.0)
            gv += torch.matmul(p.transpose(1, 2), do)
            ds = p * (torch.matmul(do, v.transpose(1, 2)) - (do * o).sum(2, keepdim=True)) * scale
            dq[rows] = torch.matmul(ds, k).transpose(0, 1)
            gk += torch.matmul(ds.transpose(1, 2), q)
        dk[k0:k1] = gk.view(hk, group, k1 - k0, d).sum(1).transpose(0, 1)
        dv[k0:k1] = gv.view(hk, group, k1 - k0, d).sum(1).transpose(0, 1)
    t = st["q"].dtype
    return {"dq": dq.to(t), "dk": dk.to(t), "dv": dv.to(t)}


# ---- one pass -----------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        if op == "ln":
            return _ln_plain(st)
        if op == "ln_bwd":
            return _ln_bwd_plain(st)
        if op == "rope":
            return _rope_plain(st)
        if op == "attn_bwd":
            return _attention_bwd_plain(st)
        out, lse = _attention_plain(st)
        return {"out": out.to(st["q"].dtype), "lse": lse}
    from rsna_knee_efficiency_b200 import ops
    if op == "ln":
        ops.layer_norm(st["x"], st["w"], st["b"], st["y"], eps=1e-5, res=st["res"], sum=st["sum"], mean=st["mean"],
                       rstd=st["rstd"])
        r = {"y": st["y"], "mean": st["mean"], "rstd": st["rstd"]}
        if st["res"] is not None:
            r["sum"] = st["sum"]
        return r
    if op == "ln_bwd":
        ops.layer_norm_backward(st["dy"], st["x"], st["w"], st["mean"], st["rstd"], st["dx"], st["dw"], st["db"],
                                dsum=st["dsum"])
        return {"dx": st["dx"], "dw": st["dw"], "db": st["db"]}
    if op == "rope":
        ops.rope(st["q"], st["k"], st["pos"], st["qo"], st["ko"], _ints(case["sections"]), base=10000.0,
                 per_axis=case["per_axis"], interleaved=case["interleaved"], inverse=case["inverse"])
        return {"q": st["qo"], "k": st["ko"]}
    mask = dict(left=case["left"], right=case["right"], sinks=case["sinks"], keep=st["keep"], len_k=st["len_k"])
    if op == "attn_bwd":
        ops.attention_backward(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"], st["dq"], st["dk"],
                               st["dv"], st["cu_q"], st["cu_k"], **mask)
        return {"dq": st["dq"], "dk": st["dk"], "dv": st["dv"]}
    ops.attention(st["q"], st["k"], st["v"], st["out"], st["cu_q"], st["cu_k"], lse=st["lse"], **mask)
    return {"out": st["out"], "lse": st["lse"]}


# ---- what a pass cannot do without --------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of a head, by the formula of the mask (a key mask's share expected)."""
    total = 0.0
    nqs = [case["nq"]] * len(_ints(case["lens"])) if case["op"] == "few" else _ints(case["lens"])
    for nq, nk in zip(nqs, _ints(case["lens"])):
        for i in range(nq):
            p = i + nk - nq
            hi = nk if case["right"] < 0 else min(nk, p + case["right"] + 1)
            lo = 0 if case["left"] < 0 else max(0, p - case["left"])
            total += max(0, hi - lo) + max(0, min(case["sinks"], lo, hi))
    return total * case.get("keep", 1.0)


def _seen_keys(case):
    """Keys that some query sees, over the sequences (a cache's unseen part need not be read)."""
    if case["op"] != "few" or case["left"] < 0:
        return sum(_ints(case["lens"]))
    return sum(min(n, case["left"] + case["nq"] + case["sinks"]) for n in _ints(case["lens"]))


def work(case):
    op = case["op"]
    e = TYPES[case["type"]].itemsize
    if op in ("ln", "ln_bwd"):
        n, m, c = case["rows"] * case["c"], case["rows"], case["c"]
        eo = TYPES[case["out"]].itemsize
        if op == "ln":
            return {"bytes": n * (e * (3 if case["res"] else 1) + eo) + 8 * m + 8 * c, "flops": 8 * n}
        return {"bytes": n * (e * (3 if case["res"] else 2) + eo) + 8 * m + 12 * c, "flops": 16 * n}
    if op == "rope":
        n = case["tokens"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * n * e + 4 * case["tokens"] * len(_ints(case["sections"])), "flops": 3 * n}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    nk = _seen_keys(case)
    nq = case["nq"] * len(_ints(case["lens"])) if op == "few" else sum(_ints(case["lens"]))
    pairs = _pairs(case) * hq
    if op == "attn_bwd":
        return {"bytes": e * d * (4 * nq * hq + 4 * nk * hk) + 4 * nq * hq, "flops": 10 * d * pairs}
    return {"bytes": e * d * (2 * nq * hq + 2 * nk * hk) + 4 * nq * hq, "flops": 4 * d * pairs}


# ---- exact results in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op in ("attn", "few", "attn_bwd") and _pairs(case) * case["hq"] * case["d"] > 4e11:
        return None
    st = prepare(case, seed)
    if op == "ln":
        x = st["x"].double()
        if st["res"] is not None:
            # the sum that is normalised is the stored one, rounded to the inputs' type
            x = (x + st["res"].double()).to(st["x"].dtype).double()
        var, mu = torch.var_mean(x, dim=1, correction=0)
        inv = 1.0 / torch.sqrt(var + 1e-5)
        y = torch.einsum("mc,m->mc", x - mu[:, None], inv) * st["w"].double() + st["b"].double()
        r = {"y": y, "mean": mu, "rstd": inv}
        if st["res"] is not None:
            r["sum"] = x
        return r
    if op == "ln_bwd":
        x, dy, w = st["x"].double(), st["dy"].double(), st["w"].double()
        mu, r, c = st["mean"].double(), st["rstd"].double(), case["c"]
        xh = torch.einsum("mc,m->mc", x - mu[:, None], r)
        a = torch.einsum("mc,c->m", dy, w) / c
        b = torch.einsum("mc,c,mc->m", dy, w, xh) / c
        dx = torch.einsum("m,mc->mc", r, dy * w - a[:, None] - xh * b[:, None])
        if st["dsum"] is not None:
            dx += st["dsum"].double()
        return {"dx": dx, "dw": torch.einsum("mc,mc->c", dy, xh), "db": dy.sum(0)}
    if op == "rope":
        pairs, out = sum(_ints(case["sections"])), []
        sign = -1.0 if case["inverse"] else 1.0
        for x in (st["q"].double(), st["k"].double()):
            y = x.clone()
            j = 0
            for a, n in enumerate(_ints(case["sections"])):
                for i in range(n):
                    step = 10000.0 ** (i / n if case["per_axis"] else j / pairs)
                    # a rotation is a product with exp(i angle)
                    turn = torch.polar(torch.ones(case["tokens"], dtype=torch.float64, device=DEV),
                                       sign * st["pos"][:, a].double() / step)[:, None]
                    lo, hi = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + pairs)
                    z = torch.complex(x[..., lo], x[..., hi]) * turn
                    y[..., lo], y[..., hi] = z.real, z.imag
                    j += 1
            out.append(y)
        return {"q": out[0], "k": out[1]}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    g = hq // hk
    like = {"dq": "q", "dk": "k", "dv": "v"} if op == "attn_bwd" else {"out": "q", "lse": "lse"}
    res = {n: torch.zeros(st[s].shape, dtype=torch.float64, device=DEV) for n, s in like.items()}
    for b, nk in enumerate(_ints(case["lens"])):
        kb = slice(st["ck"][b], st["ck"][b] + nk)
        n0, n1 = st["cq"][b], st["cq"][b + 1]
        j = torch.arange(nk, device=DEV)
        for i0 in range(n0, n1, 4096):
            i1 = min(n1, i0 + 4096)
            p = torch.arange(i0 - n0, i1 - n0, device=DEV) + nk - (n1 - n0)
            hidden = torch.zeros(i1 - i0, nk, dtype=torch.bool, device=DEV)
            if case["right"] >= 0:
                hidden |= j[None] - p[:, None] > case["right"]
            if case["left"] >= 0:
                hidden |= (p[:, None] - j[None] > case["left"]) & (j[None] >= case["sinks"])
            if st["keep"] is not None:
                hidden |= ~st["keep"][kb][None]
            for h in range(hq):
                q, k, v = (x.double() for x in (st["q"][i0:i1, h], st["k"][kb, h // g], st["v"][kb, h // g]))
                z = torch.einsum("id,jd->ij", q, k) / math.sqrt(d)
                z[hidden] = -math.inf
                if op != "attn_bwd":
                    lse = torch.logsumexp(z, 1)
                    w = torch.exp(z - lse[:, None])
                    w[torch.isinf(lse)] = 0.0
                    res["out"][i0:i1, h] = torch.einsum("ij,jd->id", w, v)
                    res["lse"][i0:i1, h] = lse
                    continue
                w = torch.exp(z - st["lse"][i0:i1, h].double()[:, None])
                do, o = st["dout"][i0:i1, h].double(), st["out"][i0:i1, h].double()
                dz = w * (torch.einsum("id,jd->ij", do, v) - torch.einsum("id,id->i", do, o)[:, None]) / math.sqrt(d)
                res["dq"][i0:i1, h] = torch.einsum("ij,jd->id", dz, k)
                res["dk"][kb, h // g] += torch.einsum("ij,id->jd", dz, q)
                res["dv"][kb, h // g] += torch.einsum("ij,id->jd", w, do)
    return res
