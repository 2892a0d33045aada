"""The context head as a run of its operators: logits and gradients against a plain 64-bit network, studies
of different lengths and missing windows, and the study loop that calls it."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import context_ref as ref
from rsna_knee_efficiency_b200 import infer
from rsna_knee_efficiency_b200.context import ContextHead
from test_gpu_study import IMG, SLICES, _packs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(m: ContextHead, p: dict, feats, lens, pos, keep):
    """The head's formulas in elementary 64-bit operations, study by study (p: its parameters by name)."""
    out, at = [], 0
    ln = lambda x, n: F.layer_norm(x, (x.shape[-1],), p[n + ".weight"], p[n + ".bias"], 1e-5)
    lin = lambda x, n: x @ p[n + ".weight"].T + p[n + ".bias"]
    G = m.heads // m.kv_heads

    def turn(x, ps):
        P, freq = m.d // 2, []
        for ax, n in enumerate(m.sections):
            freq += [ps[:, ax].double() * m.base ** (-i / n) for i in range(n)]
        ang = torch.stack(freq, 1)[:, None]
        a, b = x[..., :P], x[..., P:]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

    def attend(q, k, v, ok):
        s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(G, 1)) * m.d ** -0.5
        s = s.masked_fill(~ok, -torch.inf)
        w = torch.where(ok, s.softmax(-1), 0.0)
        return torch.einsum("hij,jhd->ihd", w, v.repeat_interleave(G, 1))
    for n in lens:
        x = lin(ln(feats[at:at + n].double(), "norm_in"), "embed")
        x = torch.cat([p["first"], x])
        ps = torch.cat([torch.zeros(m.first_tokens, 2, dtype=torch.int32, device=DEV), pos[at:at + n]])
        kp = torch.ones(len(x), dtype=torch.bool, device=DEV)
        if keep is not None:
            kp[m.first_tokens:] = keep[at:at + n]
        T = len(x)
        ok = ref.visible(torch.arange(T, device=DEV), T, T, m.window, m.window, m.first_tokens, kp, DEV)
        for i in range(len(m.layers)):
            q, k, v = lin(ln(x, f"layers.{i}.norm1"), f"layers.{i}.qkv").view(T, m.heads + 2 * m.kv_heads, m.d).split(
                (m.heads, m.kv_heads, m.kv_heads), 1)
            o = attend(turn(q, ps), turn(k, ps), v, ok)
            x = x + lin(o.flatten(1), f"layers.{i}.proj")
            x = x + lin(F.gelu(lin(ln(x, f"layers.{i}.norm2"), f"layers.{i}.up")), f"layers.{i}.down")
        k, v = lin(ln(x, "norm_out"), "kv").view(T, 2 * m.kv_heads, m.d).split((m.kv_heads, m.kv_heads), 1)
        o = attend(p["query"], k, v, kp[None].expand(m.n_out, T))
        out.append((o.reshape(m.n_out, -1) * p["out_weight"]).sum(1) + p["out_bias"])
        at += n
    return torch.stack(out)


def case(lens, seed, **kw):
    torch.manual_seed(seed)
    m = ContextHead(c=160, n_out=5, width=128, layers=2, dtype=torch.float16, **kw).to(DEV)
    for name, t in m.named_parameters():                 # every parameter takes part
        if "norm" in name or name.endswith("bias"):
            t.data += 0.2 * torch.randn_like(t)
    n = sum(lens)
    feats = torch.rand(n, 160, device=DEV) * 2
    pos = torch.stack([torch.randint(0, 2, (n,)), torch.randint(0, 24, (n,))], 1).int().to(DEV)
    return m, feats, pos


# Roundings to fp16 between features and logits: norm, linear and its weights at both ends and for the
# pooling (12), and per layer norm, linear and weights x 4, rotation, weights of the softmax, output, sums
# (16): 44 for two layers. Each is off by u of its tensor's size at most; norms and residual sums keep the
# size of what passes through, a gain of 2 is allowed. The backward pass has as many again.
ROUNDINGS, GAIN = 44, 2


@pytest.mark.parametrize("kw,lens,masked", [
    (dict(heads=4, first_tokens=4), [48, 48, 48], False), (dict(heads=8, kv_heads=2, first_tokens=2, window=5), [24, 1, 130, 7], True),
    (dict(heads=2, first_tokens=1, window=20), [300, 5], True), (dict(heads=4, first_tokens=0), [12, 0, 30], False)])
def test_logits_and_gradients_match_the_plain_network(kw, lens, masked):
    m, feats, pos = case(lens, len(lens), **kw)
    keep = torch.rand(len(feats), device=DEV) < 0.7 if masked else None
    logits = m(feats, lens, pos, keep)
    p = {k: v.detach().double().requires_grad_() for k, v in m.named_parameters()}
    want = plain(m, p, feats, lens, pos, keep)
    tol = ROUNDINGS * GAIN * ref.u(torch.float16)
    assert float((logits - want).detach().norm()) <= tol * float(want.detach().norm())
    g = torch.randn(want.shape, device=DEV)
    (logits * g).sum().backward()
    (want * g).sum().backward()
    for k, v in m.named_parameters():
        if v.numel():
            w = p[k].grad
            assert float((v.grad - w).norm()) <= 2 * tol * float(w.norm()), k
    with torch.no_grad():
        assert torch.equal(m(feats, m.layout(lens, DEV), pos, keep), logits)


def test_missing_windows_do_not_matter():
    m, feats, pos = case([20, 20], 3, heads=4)
    keep = torch.rand(40, device=DEV) < 0.5
    with torch.no_grad():
        a = m(feats, [20, 20], pos, keep)
        b = m(torch.where(keep[:, None], feats, feats.flip(0) + 3), [20, 20], pos, keep)
    assert torch.equal(a, b)


def test_refusals():
    m, feats, pos = case([8], 1, heads=4)
    for bad in (lambda: ContextHead(width=100, heads=8), lambda: ContextHead(window=-2), lambda: ContextHead(heads=4, kv_heads=3),
                lambda: m(feats, [9], pos), lambda: m(feats, [8], pos[:, :1]), lambda: m(feats, [8], pos, torch.ones(3)),
                lambda: m.layout([], DEV), lambda: m.layout([-1], DEV)):
        with pytest.raises(ValueError):
            bad()
    lay = m.layout([8], DEV)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m(feats, lay, pos)


def test_captured_inference_replays_on_new_features():
    m, feats, pos = case([30, 9], 2, heads=4, window=8)
    lay = m.layout([30, 9], DEV)
    with torch.no_grad():
        m(feats, lay, pos)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(feats, lay, pos)
        feats.copy_(torch.rand_like(feats))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m(feats, lay, pos))


@pytest.mark.parametrize("zoom", [None, (1.1, 0.0, 0.0)])
def test_study_loop_with_context_heads(zoom):
    """StudyRunner with a context head per seed: the head applied to each seed's features, study by study;
    a slot that a study lacks is not attended to."""
    studies = 2
    packs = [p for p, _, _ in _packs(studies * (SLICES - 2))]
    torch.manual_seed(0)
    heads = [ContextHead(n_out=12, window=6) for _ in packs]
    runner = infer.StudyRunner(packs, 0, studies, SLICES, context=heads, zoom=zoom)
    vols = torch.from_numpy(infer.make_volumes(studies, img=IMG, slices=SLICES, seed=5)).cuda()
    got = runner.run(vols).clone()
    assert got.shape == (studies, 12)
    want = torch.zeros_like(got)
    for k, h in enumerate(heads):
        w = torch.from_numpy(runner.windows[k]).int()
        pos = torch.stack([w // 24, w % 24], 1).cuda()
        for s in range(studies):
            with torch.no_grad():
                want[s] += h(runner.encoders[k].out[s * 24:(s + 1) * 24], [24], pos)[0] / len(heads)
    # one study alone or two together: the library's matrix products may add in another order
    torch.testing.assert_close(got, want, rtol=0, atol=ROUNDINGS * GAIN * 2.0 ** -8 * float(want.abs().max()))
    assert torch.equal(runner.run(vols), got)
    present = torch.tensor([[True, True], [True, False]], device=DEV)
    a = runner.run(vols, present).clone()
    vols[1, 1] = 255 - vols[1, 1]
    assert torch.equal(runner.run(vols, present), a)
    assert not torch.equal(a[1], got[1])
    with pytest.raises(ValueError, match="present"):
        runner.run(vols, present[:1])
    with pytest.raises(ValueError, match="channels"):
        infer.StudyRunner(packs, 0, studies, SLICES, context=[ContextHead(c=64)] * 2)
    shard = infer.run_shard(runner, vols.cpu().pin_memory())
    assert shard.shape == (2, 12)
