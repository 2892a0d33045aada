"""The network behind the encoder: a context transformer over a study's windows and an attention head per
finding, on the kernels of `ops` (layer norm, rotary positions, attention), for inference in the study
loop (`infer.StudyRunner(context=...)`) and for refitting it on the INT8 encoder's features.

The reference's network has the same parts behind its encoder (`KneeBaseline`,
src/knee/models/baseline.py:395-700: context transformer, then attention per finding over the windows
that a study has); this module's layout is its own:

    features [N, C] of the windows of B studies -> layer norm -> linear to `width`
    `first_tokens` learned tokens in front of every study's windows
    `layers` times: norm -> q, k, v -> rotary positions (slot, slice) -> attention (a window of slices to
        each side, the first tokens always visible, windows that a study lacks masked) -> linear -> sum;
        norm -> linear -> gelu -> linear -> sum
    norm -> k, v; one learned query per finding attends to the study's tokens -> logit [B, n_out]

Parameters are fp32; activations are `dtype` (bf16 or fp16), the sums and statistics inside the kernels
fp32. `layer_norm`, `rope` and `attention` below are the operators with their gradients for torch's
autograd. Their backward passes can be captured in a CUDA graph through `ops`; capturing through
autograd is refused, since torch ends the process when another graph of the same leaves is alive.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _native as nat
from . import ops


_NO_CAPTURE = "autograd through these operators cannot be captured: capture ops.*_backward, or use torch.no_grad()"


def _refuse_capture(*tensors) -> None:
    if torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing() and \
            any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(_NO_CAPTURE)


def _refuse_captured_backward() -> None:
    """(of a forward pass that was not captured)"""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(_NO_CAPTURE)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, dtype, res):
        out = torch.empty(x.shape, dtype=dtype, device=x.device)
        h = torch.empty_like(x, memory_format=torch.contiguous_format) if res is not None else None
        mean, rstd = (torch.empty(x.shape[0], dtype=torch.float32, device=x.device) for _ in range(2))
        ops.layer_norm(x, weight, bias, out, eps, res, h, mean, rstd)
        ctx.save_for_backward(x if h is None else h, weight, mean, rstd)
        ctx.has = (res is not None, None if bias is None else bias.dtype)
        if h is None:
            return out
        return out, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        _refuse_captured_backward()
        h, weight, mean, rstd = ctx.saved_tensors
        dx = torch.empty_like(h, memory_format=torch.contiguous_format)
        dw = None if weight is None else torch.empty_like(weight)
        has_res, bias_type = ctx.has
        db = None
        if bias_type is not None:                            # (of the weight's type, fp32 without one)
            db = torch.empty(h.shape[1], dtype=torch.float32 if weight is None else weight.dtype, device=h.device)
        ops.layer_norm_backward(dy.contiguous(), h, weight, mean, rstd, dx, dw, db,
                                None if dsum is None else dsum.contiguous())
        return dx, dw, None if db is None else db.to(bias_type), None, None, dx if has_res else None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float = 1e-5,
               dtype: torch.dtype | None = None, res: torch.Tensor | None = None):
    """`ops.layer_norm` of x [M, C] with a gradient; returns the output (of `dtype`, default x's), and with
    `res` (output, x + res)."""
    _refuse_capture(x, weight, bias, res)
    return _LayerNorm.apply(x, weight, bias, eps, dtype or x.dtype, res)


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, sections, base, per_axis):
        ctx.save_for_backward(pos)
        ctx.how = (sections, base, per_axis)
        out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
        ops.rope(q, k, pos, *out, sections, base, per_axis)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        _refuse_captured_backward()
        pos, = ctx.saved_tensors
        dq, dk = dq.contiguous(), dk.contiguous()
        out = [torch.empty_like(t) for t in (dq, dk)]
        ops.rope(dq, dk, pos, *out, *ctx.how, inverse=True)
        return *out, None, None, None, None


def rope(q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor, sections, base: float = 10000.0,
         per_axis: bool = False):
    """`ops.rope` of q [T, Hq, D] and k [T, Hk, D] with a gradient; returns both."""
    _refuse_capture(q, k)
    return _Rope.apply(q, k, pos, tuple(sections), base, per_axis)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, mask):
        # rows of no sequence are not written: they are zero here, and so are their gradients
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.full(q.shape[:2], -torch.inf, dtype=torch.float32, device=q.device)
        ops.attention(q, k, v, out, cu_q, cu_k, lse=lse, **mask)
        # (keep and len_k among the saved tensors: autograd notices when they change before the backward pass)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k, mask.get("keep"), mask.get("len_k"))
        ctx.mask = {n: x for n, x in mask.items() if n not in ("keep", "len_k")}
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _refuse_captured_backward()
        q, k, v, out, lse, cu_q, cu_k, keep, len_k = ctx.saved_tensors
        grads = [torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
        ops.attention_backward(dout.contiguous(), q, k, v, out, lse, *grads, cu_q, cu_k, keep=keep, len_k=len_k, **ctx.mask)
        return *grads, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor, **mask):
    """`ops.attention` with a gradient; `mask`: left, right, sinks, keep, len_k, scale, and `err`, the error word of
    both directions."""
    _refuse_capture(q, k, v)
    return _Attention.apply(q, k, v, cu_q, cu_k, mask)


class _Norm(nn.Module):
    def __init__(self, c: int) -> None:
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.ones(c)), nn.Parameter(torch.zeros(c))

    def forward(self, x, dtype=None, res=None):
        return layer_norm(x, self.weight, self.bias, 1e-5, dtype, res)


class _Layer(nn.Module):
    def __init__(self, width: int, heads: int, kv_heads: int, d: int, mlp: int) -> None:
        super().__init__()
        self.norm1, self.norm2 = _Norm(width), _Norm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * d)
        self.proj = nn.Linear(heads * d, width)
        self.up, self.down = nn.Linear(width, mlp * width), nn.Linear(mlp * width, width)


class ContextHead(nn.Module):
    """Study logits [B, n_out] from window features. `window`: how many neighbours to each side a window
    sees (-1: all); `kv_heads` key heads shared by `heads` query heads (default: as many)."""

    def __init__(self, c: int = 1664, n_out: int = 4, width: int = 256, heads: int = 4, kv_heads: int | None = None,
                 layers: int = 2, mlp: int = 2, first_tokens: int = 4, window: int = -1,
                 dtype: torch.dtype = torch.bfloat16, base: float = 100.0) -> None:
        super().__init__()
        kv_heads = kv_heads or heads
        d = width // heads
        if width % heads or heads % kv_heads or d % 8 or d > 128:
            raise ValueError(f"width {width}, {heads} heads, {kv_heads} key heads: the head size must be a multiple of 8 "
                             "up to 128 and the key heads divide the heads")
        if first_tokens < 0 or window < -1 or dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("first_tokens >= 0, window >= -1 and a 16-bit dtype expected")
        self.c, self.n_out, self.width, self.heads, self.kv_heads, self.d = c, n_out, width, heads, kv_heads, d
        self.first_tokens, self.window, self.dtype, self.base = first_tokens, window, dtype, base
        self.sections = (d // 8, d // 2 - d // 8)            # pairs that turn with the slot, with the slice
        self.norm_in, self.embed = _Norm(c), nn.Linear(c, width)
        self.first = nn.Parameter(0.02 * torch.randn(first_tokens, width))
        self.layers = nn.ModuleList(_Layer(width, heads, kv_heads, d, mlp) for _ in range(layers))
        self.norm_out, self.kv = _Norm(width), nn.Linear(width, 2 * kv_heads * d)
        self.query = nn.Parameter(torch.randn(n_out, heads, d))
        self.out_weight = nn.Parameter(torch.randn(n_out, heads * d) * (heads * d) ** -0.5)
        self.out_bias = nn.Parameter(torch.zeros(n_out))
        # The error word of the head's attention kernels, forward and backward (see check), made by the first call on
        # a device. No buffer: wrappers that share buffers between ranks would overwrite one rank's by another's.
        self.err: torch.Tensor | None = None

    def _error_word(self, dev: torch.device) -> torch.Tensor:
        if self.err is None or self.err.device != dev:
            with torch.inference_mode(False):                # (check clears it, in whatever mode)
                self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        return self.err

    def check(self) -> None:
        """Raises if a kernel of the head, forward or backward, gave up a bounded wait, or met offsets outside the
        tensors, since the last check (synchronises; its outputs hold zeros or rows that were never written then)."""
        if self.err is None:
            return
        torch.cuda.synchronize(self.err.device)
        code = int(self.err)
        if code:
            self.err.zero_()
            raise nat.Dn8Error(f"ContextHead: a kernel gave up a bounded wait or met offsets outside the tensors (code {code})")

    def _linear(self, x: torch.Tensor, m: nn.Linear) -> torch.Tensor:
        return F.linear(x, m.weight.to(self.dtype), m.bias.to(self.dtype))

    def layout(self, lens, device) -> dict:
        """Where the tokens of studies with lens[b] windows lie (kept by a caller whose studies do not
        change: `forward` makes it when it is given the lengths)."""
        lens = [int(m) for m in lens]
        if not lens or min(lens) < 0:
            raise ValueError(f"lengths {lens}: one or more studies of zero or more windows")
        cu, rows, firsts, f = [0], [], [], self.first_tokens
        for m in lens:
            firsts += range(cu[-1], cu[-1] + f)
            rows += range(cu[-1] + f, cu[-1] + f + m)
            cu.append(cu[-1] + f + m)
        def put(values, dtype):
            return torch.tensor(values, dtype=dtype).to(device)
        return dict(studies=len(lens), windows=len(rows), tokens=cu[-1], rows=put(rows, torch.long),
                    firsts=put(firsts, torch.long), cu_k=put(cu, torch.int32),
                    cu_q=put([self.n_out * i for i in range(len(lens) + 1)], torch.int32))

    def forward(self, feats: torch.Tensor, studies, pos: torch.Tensor, keep: torch.Tensor | None = None) -> torch.Tensor:
        """feats [N, C] fp32: the windows of all studies in order; `studies`: the number of windows of each
        study, or `layout` of them; pos int32 [N, 2] = (slot, slice) of each window; keep bool [N]: the
        windows that exist (default: all)."""
        lay = studies if isinstance(studies, dict) else self.layout(studies, feats.device)
        n, b, at, f, dev = lay["windows"], lay["studies"], lay["tokens"], self.first_tokens, feats.device
        if tuple(feats.shape) != (n, self.c):
            raise ValueError(f"features {tuple(feats.shape)}, expected {(n, self.c)}")
        if tuple(pos.shape) != (n, 2) or (keep is not None and tuple(keep.shape) != (n,)):
            raise ValueError(f"pos [{n}, 2] and keep [{n}] expected")
        rows, cu_k, cu_q, err = lay["rows"], lay["cu_k"], lay["cu_q"], self._error_word(dev)
        posn = torch.zeros(at, 2, dtype=torch.int32, device=dev).index_copy_(0, rows, pos)
        kept = None
        if keep is not None:
            kept = torch.ones(at, dtype=torch.bool, device=dev).index_copy_(0, rows, keep.bool())
        x = self._linear(self.norm_in(feats.float(), self.dtype), self.embed)
        tok = torch.zeros(at, self.width, dtype=self.dtype, device=dev).index_copy(0, rows, x)
        if f:
            tok = tok.index_copy(0, lay["firsts"], self.first.to(self.dtype).repeat(b, 1))
        H, K, d = self.heads, self.kv_heads, self.d
        branch = None                                        # the last sublayer's output, not yet added
        for la in self.layers:
            y, tok = (la.norm1(tok), tok) if branch is None else la.norm1(branch, None, tok)
            q, k, v = self._linear(y, la.qkv).view(at, H + 2 * K, d).split((H, K, K), 1)
            q, k = rope(q, k, posn, self.sections, self.base, True)
            o = attention(q, k, v, cu_k, cu_k, left=self.window, right=self.window, sinks=f, keep=kept, err=err)
            y, tok = la.norm2(self._linear(o.view(at, H * d), la.proj), None, tok)
            branch = self._linear(F.gelu(self._linear(y, la.up)), la.down)
        y = self.norm_out(tok) if branch is None else self.norm_out(branch, None, tok)[0]
        k, v = self._linear(y, self.kv).view(at, 2 * K, d).split((K, K), 1)
        q = self.query.to(self.dtype).repeat(b, 1, 1)
        o = attention(q, k, v, cu_q, cu_k, keep=kept, err=err)
        return (o.view(b, self.n_out, H * d).float() * self.out_weight).sum(2) + self.out_bias
