"""Kernel-level operators on torch CUDA tensors (the reference's per-kernel launches, through the
C ABI of include/dn8.h). Layouts:
  store  group-major in0 [G0, N, HW, 32] int8 and seg [L, N, HW, 32] int8, or (tile_groups = Gt > 0)
         the tile-major block store [ceil(N*HW/128), Gt, 128, 32] int8 holding every group;
  bottleneck u8 as 8 planes of 16 channels [8, N*HW, 16];
  conv2 output: the store slot [N, HW, 32] int8, or group `group` of a tile-major store.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _native as nat


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream(stream) -> int | None:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def conv1(in0: torch.Tensor, seg: torch.Tensor | None, w1: torch.Tensor, ab: torch.Tensor,
          gd: torch.Tensor, out: torch.Tensor, G0: int, G: int, N: int, HW: int,
          prologue_f16: bool, err: torch.Tensor | None = None, stream=None, tile_groups: int = 0) -> None:
    """tile_groups = 0: in0 / seg are group-major planes; > 0: in0 is a tile-major block store."""
    a = nat.Conv1Args(_ptr(in0), _ptr(seg), _ptr(w1), _ptr(ab), _ptr(gd), _ptr(out), _ptr(err),
                      G0, G, N, HW, int(bool(prologue_f16)), int(tile_groups))
    nat.check(nat.lib().dn8_conv1(a, _stream(stream)), "dn8_conv1")


def conv2(x: torch.Tensor, w2k: torch.Tensor, sc: torch.Tensor, out: torch.Tensor, N: int, H: int,
          W: int, err: torch.Tensor | None = None, stream=None, tile_groups: int = 0, group: int = 0) -> None:
    a = nat.Conv2Args(_ptr(x), _ptr(w2k), _ptr(sc), _ptr(out), _ptr(err), N, H, W, tile_groups, group)
    nat.check(nat.lib().dn8_conv2(a, _stream(stream)), "dn8_conv2")


def trans(in0: torch.Tensor, seg: torch.Tensor, tw: torch.Tensor, ab: torch.Tensor, gd: torch.Tensor,
          out: torch.Tensor, G0: int, G: int, N: int, H: int, W: int, prologue_f16: bool,
          err: torch.Tensor | None = None, stream=None, tile_groups: int = 0, out_tile_groups: int = 0) -> None:
    a = nat.TransArgs(_ptr(in0), _ptr(seg), _ptr(tw), _ptr(ab), _ptr(gd), _ptr(out), _ptr(err),
                      G0, G, N, H, W, int(bool(prologue_f16)), tile_groups, out_tile_groups)
    nat.check(nat.lib().dn8_trans(a, _stream(stream)), "dn8_trans")


def stem(x: torch.Tensor, w8u: torch.Tensor, kc: torch.Tensor, out: torch.Tensor, N: int, H: int,
         W: int, src: torch.Tensor | None = None, flags: torch.Tensor | None = None,
         err: torch.Tensor | None = None, stream=None, tile_groups: int = 0) -> None:
    """x: fp16 [N, 3, H, W] windows, or uint8 planes [P, H, W] with `src` int32 [N, 4]."""
    x_u8 = x.dtype == torch.uint8
    a = nat.StemArgs(_ptr(x), _ptr(src), _ptr(flags), _ptr(w8u), _ptr(kc), _ptr(out), _ptr(err),
                     N, H, W, int(x_u8), 0, tile_groups)
    nat.check(nat.lib().dn8_stem(a, _stream(stream)), "dn8_stem")


def head(in0: torch.Tensor, seg: torch.Tensor, fab: torch.Tensor, G0: int, G: int, N: int, HW: int,
         feat: torch.Tensor | None = None, hw: torch.Tensor | None = None, hb: torch.Tensor | None = None,
         logits: torch.Tensor | None = None, view_logits: torch.Tensor | None = None,
         tickets: torch.Tensor | None = None, per_view: int = 0, stream=None, tile_groups: int = 0) -> None:
    n_out = 0 if hw is None else hw.shape[0]
    a = nat.HeadArgs(_ptr(in0), _ptr(seg), _ptr(fab), _ptr(feat), _ptr(hw), _ptr(hb), _ptr(logits),
                     _ptr(view_logits), _ptr(tickets), G0, G, N, HW, n_out, per_view, 0, tile_groups)
    nat.check(nat.lib().dn8_head(a, _stream(stream)), "dn8_head")


def zoom(planes: torch.Tensor, src: torch.Tensor, out: torch.Tensor, N: int, H: int, W: int,
         scale: float, tx: float = 0.0, ty: float = 0.0, flags: torch.Tensor | None = None,
         err: torch.Tensor | None = None, stream=None) -> None:
    """Zoomed / shifted fp16 windows [N, 3, H, W] from uint8 planes [P, H, W] (src int32 [N, 4])."""
    a = nat.ZoomArgs(_ptr(planes), _ptr(src), _ptr(flags), _ptr(out), _ptr(err), N, H, W, scale, tx, ty)
    nat.check(nat.lib().dn8_zoom(a, _stream(stream)), "dn8_zoom")


def head_noalloc(in0: torch.Tensor, seg: torch.Tensor, fab: torch.Tensor, G0: int, G: int, N: int, HW: int,
                 feat: torch.Tensor | None = None, hw: torch.Tensor | None = None, hb: torch.Tensor | None = None,
                 logits: torch.Tensor | None = None, view_logits: torch.Tensor | None = None,
                 per_view: int = 0, stream=None) -> None:
    """`head` with the library's built-in per-view counters instead of a ticket array (no device
    allocation by the caller): at most DN8_HEAD_SCRATCH_VIEWS views per call, calls in order."""
    n_out = 0 if hw is None else hw.shape[0]
    a = nat.HeadArgs(_ptr(in0), _ptr(seg), _ptr(fab), _ptr(feat), _ptr(hw), _ptr(hb), _ptr(logits),
                     _ptr(view_logits), None, G0, G, N, HW, n_out, per_view, 0)
    nat.check(nat.lib().dn8_head_noalloc(a, _stream(stream)), "dn8_head_noalloc")


# --- the context transformer's operators -----------------------------------------------------
# Tensors of one call live on one GPU, which need not be the current one; the work goes to `stream`
# (default: that GPU's current stream), and so does a workspace that the call allocates.
_TYPES = {torch.float32: nat.DN8_F32, torch.float16: nat.DN8_F16, torch.bfloat16: nat.DN8_BF16}


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _on_gpu(call: str, stream, first: torch.Tensor, **tensors):
    """The device and the stream of a call whose tensors are `first` and `tensors` (None: absent)."""
    for name, t in tensors.items():
        if t is not None:
            _need(isinstance(t, torch.Tensor), f"{call}: {name} must be a tensor")
    _need(first.is_cuda, f"{call}: tensors on a GPU expected")
    for name, t in tensors.items():
        _need(t is None or t.device == first.device, f"{call}: {name} is not on {first.device}")
    s = stream if stream is not None else torch.cuda.current_stream(first.device)
    _need(s.device == first.device, f"{call}: the stream is not of {first.device}")
    return first.device, s


def _rows(call: str, name: str, t: torch.Tensor | None, shape, types) -> int:
    """Elements between the rows of a matrix with contiguous rows."""
    if t is None:
        return 0
    _need(tuple(t.shape) == tuple(shape), f"{call}: {name} {tuple(t.shape)}, expected {tuple(shape)}")
    _need(t.dtype in types, f"{call}: {name} is {t.dtype}")
    _need(t.shape[1] <= 1 or t.stride(1) == 1, f"{call}: the rows of {name} must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _flat(call: str, name: str, t: torch.Tensor | None, n, types) -> None:
    shape = n if isinstance(n, tuple) else (n,)
    _need(t is None or (tuple(t.shape) == shape and t.dtype in types and t.is_contiguous()),
          f"{call}: {name} must be contiguous {shape} of {', '.join(str(x) for x in types)}")


def _writable(call: str, **tensors) -> None:
    """Outputs whose elements share memory (an expanded tensor) cannot be written."""
    for name, t in tensors.items():
        _need(t is None or all(st > 0 or n <= 1 for st, n in zip(t.stride(), t.shape)),
              f"{call}: {name} has elements that share memory")


def _work(nbytes: int, device, stream) -> torch.Tensor:
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=device)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, out: torch.Tensor,
               eps: float = 1e-5, res: torch.Tensor | None = None, sum: torch.Tensor | None = None,
               mean: torch.Tensor | None = None, rstd: torch.Tensor | None = None, stream=None) -> None:
    """Layer norm of the rows of x [M, C] (fp32 / fp16 / bf16; rows contiguous, any row stride) into
    out (x's type, or 16 bits behind an fp32 x). With `res` the rows of x + res, rounded to x's
    type and stored in `sum`, are normalised. weight / bias [C]: fp32 or a 16-bit type, both of one
    type, or None. `mean` / `rstd` [M] fp32 keep the statistics for the backward pass. `out` and
    `sum` may be x or res themselves where types and strides agree."""
    c = "layer_norm"
    _need(x.dim() == 2 and x.dtype in _TYPES and x.shape[1] > 0, f"{c}: x [M, C] of fp32, fp16 or bf16 expected")
    dev, s = _on_gpu(c, stream, x, weight=weight, bias=bias, out=out, res=res, sum=sum, mean=mean, rstd=rstd)
    M, C = x.shape
    same = (x.dtype,)
    outs = tuple(_TYPES) if x.dtype == torch.float32 else same
    _need((res is None) == (sum is None), f"{c}: res and sum come together")
    strides = [_rows(c, "x", x, (M, C), same), _rows(c, "res", res, (M, C), same), _rows(c, "out", out, (M, C), outs),
               _rows(c, "sum", sum, (M, C), same)]
    wt = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
    for name, t in (("weight", weight), ("bias", bias)):
        _flat(c, name, t, C, (wt,) if wt in _TYPES else tuple(_TYPES))
    for name, t in (("mean", mean), ("rstd", rstd)):
        _flat(c, name, t, M, (torch.float32,))
    _writable(c, out=out, sum=sum)
    a = nat.LayerNormArgs(_ptr(x), _ptr(res), _ptr(weight), _ptr(bias), _ptr(out), _ptr(sum), _ptr(mean), _ptr(rstd),
                          M, *strides, C, _TYPES[x.dtype], _TYPES[out.dtype], _TYPES[wt], eps)
    with torch.cuda.device(dev):
        nat.check(nat.lib().dn8_layer_norm(a, s.cuda_stream), "dn8_layer_norm")


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                        rstd: torch.Tensor, dx: torch.Tensor, dweight: torch.Tensor | None = None,
                        dbias: torch.Tensor | None = None, dsum: torch.Tensor | None = None,
                        work: torch.Tensor | None = None, stream=None) -> None:
    """The gradient of `layer_norm`: x is what it normalised (`sum` where there was a residual), dy the
    gradient of its output (the output's type), dsum the gradient that reaches the sum past the
    norm. dx (x's type) is the gradient of x and of the residual alike; dweight / dbias [C] of the
    weight's type (fp32 without a weight) are sums over the rows, the same bits every call. dx may be
    dy, x or dsum itself. `work`: uint8 of `dn8_layer_norm_bwd_work(C)` bytes, allocated if not given."""
    c = "layer_norm_backward"
    _need(x.dim() == 2 and x.dtype in _TYPES and x.shape[1] > 0, f"{c}: x [M, C] of fp32, fp16 or bf16 expected")
    dev, s = _on_gpu(c, stream, x, dy=dy, weight=weight, mean=mean, rstd=rstd, dx=dx, dweight=dweight, dbias=dbias,
                     dsum=dsum, work=work)
    M, C = x.shape
    same = (x.dtype,)
    outs = tuple(_TYPES) if x.dtype == torch.float32 else same
    strides = [_rows(c, "dy", dy, (M, C), outs), _rows(c, "x", x, (M, C), same), _rows(c, "dsum", dsum, (M, C), same),
               _rows(c, "dx", dx, (M, C), same)]
    wt = weight.dtype if weight is not None else torch.float32
    for name, t in (("weight", weight), ("dweight", dweight), ("dbias", dbias)):
        _flat(c, name, t, C, (wt,) if wt in _TYPES else tuple(_TYPES))
    for name, t in (("mean", mean), ("rstd", rstd)):
        _need(t is not None, f"{c}: {name} is needed")
        _flat(c, name, t, M, (torch.float32,))
    _writable(c, dx=dx)
    with torch.cuda.device(dev):
        nbytes = nat.lib().dn8_layer_norm_bwd_work(C) if dweight is not None or dbias is not None else 0
        if work is None and nbytes:
            work = _work(nbytes, dev, s)
        _need(nbytes == 0 or (work.dtype == torch.uint8 and work.is_contiguous() and work.numel() >= nbytes
                              and work.data_ptr() % 16 == 0), f"{c}: work needs {nbytes} contiguous bytes (uint8)")
        a = nat.LayerNormBwdArgs(_ptr(dy), _ptr(x), _ptr(weight), _ptr(dsum), _ptr(mean), _ptr(rstd), _ptr(dx),
                                 _ptr(dweight), _ptr(dbias), _ptr(work), M, *strides, C, _TYPES[x.dtype],
                                 _TYPES[dy.dtype], _TYPES[wt])
        nat.check(nat.lib().dn8_layer_norm_bwd(a, s.cuda_stream), "dn8_layer_norm_bwd")


def _head_strides(call: str, name: str, t: torch.Tensor | None, shape, dtype) -> list:
    """Elements between tokens and between heads of a [T, H, D] tensor (0 where there is only one)."""
    if t is None:
        return [0, 0]
    _need(tuple(t.shape) == tuple(shape), f"{call}: {name} {tuple(t.shape)}, expected {tuple(shape)}")
    _need(t.dtype == dtype, f"{call}: {name} is {t.dtype}, expected {dtype}")
    _need(t.stride(2) == 1, f"{call}: the last dimension of {name} must be contiguous")
    return [t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0]


def rope(q: torch.Tensor, k: torch.Tensor | None, pos: torch.Tensor, q_out: torch.Tensor, k_out: torch.Tensor | None,
         sections, base: float = 10000.0, per_axis: bool = False, interleaved: bool = False, inverse: bool = False,
         stream=None) -> None:
    """Rotary positions with several axes on q [T, Hq, D] and k [T, Hk, D] (or None), any strides with a
    contiguous last dimension. pos int32 [T, axes] (1 to 4 axes: slot, slice, row, column, ...);
    sections[x] pairs of a head turn with axis x, the first 2 * sum(sections) elements of a head as
    pairs (j, j + P) or, interleaved, (2 j, 2 j + 1); the rest is copied. Frequencies base^(-j / P)
    over all pairs, or one ladder base^(-i / sections[x]) per axis. `inverse` turns back: the
    backward pass. q_out / k_out may be q / k themselves."""
    c = "rope"
    _need(q.dim() == 3 and q.dtype in _TYPES, f"{c}: q [T, H, D] of fp32, fp16 or bf16 expected")
    _need((k is None) == (k_out is None), f"{c}: k and k_out come together")
    dev, s = _on_gpu(c, stream, q, k=k, pos=pos, q_out=q_out, k_out=k_out)
    T, Hq, D = q.shape
    _need(k is None or k.dim() == 3, f"{c}: k [T, H, D] expected")
    Hk = 0 if k is None else k.shape[1]
    sections = [int(n) for n in sections]
    _need(1 <= len(sections) <= nat.DN8_ROPE_AXES, f"{c}: 1 to {nat.DN8_ROPE_AXES} axes")
    _flat(c, "pos", pos, (T, len(sections)), (torch.int32,))
    _writable(c, q_out=q_out, k_out=k_out)
    a = nat.RopeArgs(_ptr(q), _ptr(k), _ptr(pos), _ptr(q_out), _ptr(k_out), T,
                     *_head_strides(c, "q", q, (T, Hq, D), q.dtype), *_head_strides(c, "k", k, (T, Hk, D), q.dtype),
                     *_head_strides(c, "q_out", q_out, (T, Hq, D), q.dtype),
                     *_head_strides(c, "k_out", k_out, (T, Hk, D), q.dtype), Hq, Hk, D, _TYPES[q.dtype], len(sections),
                     (nat.I32 * nat.DN8_ROPE_AXES)(*sections), int(bool(per_axis)), int(bool(interleaved)),
                     int(bool(inverse)), base)
    with torch.cuda.device(dev):
        nat.check(nat.lib().dn8_rope(a, s.cuda_stream), "dn8_rope")


def _attention_common(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale):
    _need(q.dim() == 3 and k.dim() == 3 and q.dtype in (torch.float16, torch.bfloat16),
          f"{c}: q [Tq, Hq, D], k [Tk, Hk, D] of fp16 or bf16 expected")
    Tq, Hq, D = q.shape
    Tk, Hk, _ = k.shape
    _need(cu_q.dim() == 1 and cu_q.numel() >= 1, f"{c}: cu_q int32 [B + 1] expected")
    B = cu_q.numel() - 1
    for name, t, n in (("cu_q", cu_q, B + 1), ("cu_k", cu_k, B + 1), ("len_k", len_k, B)):
        _flat(c, name, t, n, (torch.int32,))
    _flat(c, "keep", keep, Tk, (torch.bool, torch.uint8))
    _flat(c, "lse", lse, (Tq, Hq), (torch.float32,))
    _flat(c, "err", err, 1, (torch.int32,))
    far = 1 << 29                                        # beyond every length: no limit
    mask = (B, Hq, Hk, D, _TYPES[q.dtype], min(int(left), far), min(int(right), far), min(int(sinks), far),
            D ** -0.5 if scale is None else float(scale))
    strides = [*_head_strides(c, "q", q, (Tq, Hq, D), q.dtype), *_head_strides(c, "k", k, (Tk, Hk, D), q.dtype),
               *_head_strides(c, "v", v, (Tk, Hk, D), q.dtype)]
    return Tq, Tk, strides, mask


def _attention_work(c: str, size, a, work, dev, s):
    nbytes = size(a)
    if nbytes < 0:
        nat.check(nat.DN8_EINVAL, c)
    if work is None and nbytes:
        work = _work(nbytes, dev, s)
    _need(nbytes == 0 or (work.dtype == torch.uint8 and work.is_contiguous() and work.numel() >= nbytes),
          f"{c}: work needs {nbytes} contiguous bytes (uint8)")
    a.work = _ptr(work)
    return work


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor,
              cu_k: torch.Tensor, left: int = -1, right: int = -1, sinks: int = 0, keep: torch.Tensor | None = None,
              len_k: torch.Tensor | None = None, lse: torch.Tensor | None = None, scale: float | None = None,
              err: torch.Tensor | None = None, work: torch.Tensor | None = None, stream=None) -> None:
    """Attention of packed sequences: q / out [Tq, Hq, D], k / v [Tk, Hk, D] (fp16 or bf16, Hq a multiple
    of Hk, D a multiple of 8 up to 128; token and head strides multiples of 8 elements). Sequence b:
    query rows cu_q[b] .. cu_q[b+1] - 1 and the keys from cu_k[b] on, len_k[b] of them (a cache slot) or
    up to cu_k[b+1]. Query i of nq with nk keys stands at p = i + nk - nq and sees key j iff keep[j]
    (bool or uint8 [Tk]), j <= p + right and (j >= p - left or j < sinks); -1: no limit. right = 0 is
    causal; a single new token per sequence over caches is nq = 1. out = softmax(scale q k) v; scale
    defaults to D^-1/2; lse [Tq, Hq] fp32 is kept for the backward pass. A query that sees nothing:
    0 and -inf. Masked keys may hold anything (NaN included), visible ones must be finite. Rows of no
    sequence are left as they are. Offsets are read on the device: a sequence outside the tensors
    counts as empty and sets `err` (int32 [1]). `work`: uint8 of `dn8_attention_work` bytes,
    allocated if needed and not given."""
    c = "attention"
    dev, s = _on_gpu(c, stream, q, k=k, v=v, out=out, cu_q=cu_q, cu_k=cu_k, keep=keep, len_k=len_k, lse=lse, err=err,
                     work=work)
    Tq, Tk, strides, mask = _attention_common(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale)
    strides += _head_strides(c, "out", out, q.shape, q.dtype)
    _writable(c, out=out, lse=lse)
    a = nat.AttentionArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(cu_q), _ptr(cu_k), _ptr(len_k),
                          _ptr(keep), _ptr(err), None, Tq, Tk, *strides, *mask)
    with torch.cuda.device(dev):
        work = _attention_work("dn8_attention", nat.lib().dn8_attention_work, a, work, dev, s)
        nat.check(nat.lib().dn8_attention(a, s.cuda_stream), "dn8_attention")


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, cu_q: torch.Tensor,
                       cu_k: torch.Tensor, left: int = -1, right: int = -1, sinks: int = 0,
                       keep: torch.Tensor | None = None, len_k: torch.Tensor | None = None, scale: float | None = None,
                       err: torch.Tensor | None = None, work: torch.Tensor | None = None, stream=None) -> None:
    """The gradient of `attention` from its inputs, its `out` and `lse` and the gradient `dout` of out:
    dq [Tq, Hq, D], dk and dv [Tk, Hk, D] (summed over the query heads that share a key head), all
    of the inputs' type and with strides of their own. The same bits every call (no atomics). Rows of
    no sequence are left as they are."""
    c = "attention_backward"
    dev, s = _on_gpu(c, stream, q, dout=dout, k=k, v=v, out=out, lse=lse, dq=dq, dk=dk, dv=dv, cu_q=cu_q, cu_k=cu_k,
                     keep=keep, len_k=len_k, err=err, work=work)
    _need(lse is not None, f"{c}: lse is needed")
    Tq, Tk, strides, mask = _attention_common(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale)
    strides = _head_strides(c, "dout", dout, q.shape, q.dtype) + strides
    for name, t, like in (("out", out, q), ("dq", dq, q), ("dk", dk, k), ("dv", dv, k)):
        strides += _head_strides(c, name, t, like.shape, q.dtype)
    _writable(c, dq=dq, dk=dk, dv=dv)
    a = nat.AttentionBwdArgs(_ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv),
                             _ptr(cu_q), _ptr(cu_k), _ptr(len_k), _ptr(keep), _ptr(err), None, Tq, Tk, *strides, *mask)
    with torch.cuda.device(dev):
        work = _attention_work("dn8_attention_bwd", nat.lib().dn8_attention_bwd_work, a, work, dev, s)
        nat.check(nat.lib().dn8_attention_bwd(a, s.cuda_stream), "dn8_attention_bwd")


# --- weight preparation (numpy in, numpy out) ----------------------------------------------
def prepare_stem_weights(w8: np.ndarray) -> np.ndarray:
    """`S_w8` [64, 176] int8 -> the stem operand table (14336 bytes)."""
    w8 = np.ascontiguousarray(w8, dtype=np.int8)
    out = np.empty(14336, np.uint8)
    nat.check(nat.lib().dn8_prepare_stem_weights(w8.ctypes.data, out.ctypes.data),
              "dn8_prepare_stem_weights")
    return out


def prepare_conv1_weights(w1: np.ndarray) -> np.ndarray:
    """`L*_w1` [G, 128, 32] int8 -> the UMMA-ready table (G * 4096 bytes)."""
    w1 = np.ascontiguousarray(w1, dtype=np.int8)
    out = np.empty(w1.shape[0] * 4096, np.uint8)
    nat.check(nat.lib().dn8_prepare_conv1_weights(w1.ctypes.data, w1.shape[0], out.ctypes.data),
              "dn8_prepare_conv1_weights")
    return out


def prepare_trans_weights(tw: np.ndarray) -> np.ndarray:
    """`T*_w` [G, c_out, 32] int8 -> the UMMA-ready table (G * c_out * 32 bytes)."""
    tw = np.ascontiguousarray(tw, dtype=np.int8)
    out = np.empty(tw.size, np.uint8)
    nat.check(nat.lib().dn8_prepare_trans_weights(tw.ctypes.data, tw.shape[0], tw.shape[1],
                                                  out.ctypes.data), "dn8_prepare_trans_weights")
    return out


def prepare_conv2_weights(w2k: np.ndarray) -> np.ndarray:
    """`L*_w2k` [4, 9, 32, 32] int8 -> the conv2 operand table (36864 bytes)."""
    w2k = np.ascontiguousarray(w2k, dtype=np.int8)
    out = np.empty(36864, np.uint8)
    nat.check(nat.lib().dn8_prepare_conv2_weights(w2k.ctypes.data, out.ctypes.data),
              "dn8_prepare_conv2_weights")
    return out
