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
# The checks below read each tensor property once and build no message unless they fail: a small call is
# over in 3 us on the GPU.
_TYPES = {torch.float32: nat.DN8_F32, torch.float16: nat.DN8_F16, torch.bfloat16: nat.DN8_BF16}
_ANY = tuple(_TYPES)
_HALF = (torch.float16, torch.bfloat16)
# Sizes that the C structures hold in 32 bits are refused beyond these (ctypes would drop the upper bits)
_MOST_C, _MOST_HEADS, _MOST_SEQUENCES = 1 << 29, 65535, 1 << 30
_F32, _I32, _FLAG = (torch.float32,), (torch.int32,), (torch.bool, torch.uint8)


def _refuse(call: str, name: str, t, shape, types, dev, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{call}: {name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{call}: {name} is not on a GPU")
    raise ValueError(f"{call}: {name} {tuple(t.shape)} {t.dtype} on {t.device}: expected {tuple(shape)} of "
                     f"{', '.join(str(x) for x in types)} on {dev}, {what}")


def _gpu(call: str, t, dims: int, types, what: str) -> torch.device:
    """The device of a call's first tensor."""
    if not isinstance(t, torch.Tensor) or t.dim() != dims or t.dtype not in types:
        raise ValueError(f"{call}: {what} expected")
    if not t.is_cuda:
        raise ValueError(f"{call}: tensors on a GPU expected")
    return t.device


def _rows(call: str, name: str, t, shape, types, dev, out: bool = False) -> int:
    """Elements between the rows of a matrix with contiguous rows."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype not in types or t.device != dev:
        _refuse(call, name, t, shape, types, dev, "rows contiguous")
    st, last = t.stride()
    if (last != 1 and shape[1] > 1) or (out and st == 0 and shape[0] > 1):
        _refuse(call, name, t, shape, types, dev, "rows contiguous, an output's of their own memory")
    return st if shape[0] > 1 else shape[1]


def _flat(call: str, name: str, t, shape, types, dev) -> None:
    if t is not None and (not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype not in types or t.device != dev
                          or not t.is_contiguous()):
        _refuse(call, name, t, shape, types, dev, "contiguous")


def _heads(call: str, name: str, t, shape, types, dev, out: bool = False) -> tuple:
    """Elements between tokens and between heads of a [T, H, D] tensor (0 where there is only one)."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype not in types or t.device != dev:
        _refuse(call, name, t, shape, types, dev, "last dimension contiguous")
    st, sh, last = t.stride()
    if shape[0] <= 1:
        st = 0
    elif out and st == 0:
        _refuse(call, name, t, shape, types, dev, "no two tokens the same memory")
    if shape[1] <= 1:
        sh = 0
    elif out and sh == 0:
        _refuse(call, name, t, shape, types, dev, "no two heads the same memory")
    if last != 1 and shape[2] > 1:
        _refuse(call, name, t, shape, types, dev, "last dimension contiguous")
    return st, sh


# the handle of a device's current stream, without a Stream object around it where torch offers that (2 us)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(what: str, fn, a, dev: torch.device, stream) -> None:
    """Calls `fn(a, stream)` with the tensors' device current."""
    if stream is None:
        s = _current_stream(dev.index)
    else:
        if stream.device != dev:
            raise ValueError(f"{what}: the stream is not of {dev}")
        s = stream.cuda_stream
    if torch.cuda.current_device() == dev.index:
        status = fn(a, s)
    else:
        with torch.cuda.device(dev):
            status = fn(a, s)
    if status:
        nat.check(status, what)


def _bytes_of(fn, a, dev: torch.device) -> int:
    """Workspace bytes of a call on `dev` (they depend on its SM count); -1: the call will be refused."""
    if torch.cuda.current_device() == dev.index:
        return fn(a)
    with torch.cuda.device(dev):
        return fn(a)


def _workspace(what: str, nbytes: int, work, dev, stream):
    """`work`, checked, or a new workspace that belongs to the call's stream."""
    if work is not None:
        if not (isinstance(work, torch.Tensor) and work.dtype == torch.uint8 and work.device == dev
                and work.is_contiguous() and work.numel() >= nbytes and work.data_ptr() % 16 == 0):
            raise ValueError(f"{what}: work needs {nbytes} contiguous bytes (uint8, 16-byte aligned) on {dev}")
        return work
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, out: torch.Tensor,
               eps: float = 1e-5, res: torch.Tensor | None = None, sum: torch.Tensor | None = None,
               mean: torch.Tensor | None = None, rstd: torch.Tensor | None = None, stream=None) -> None:
    """Layer norm of the rows of x [M, C] (fp32 / fp16 / bf16; rows contiguous, any row stride) into
    out (x's type, or 16 bits behind an fp32 x). With `res` the rows of x + res, rounded to x's
    type and stored in `sum`, are normalised. weight / bias [C]: fp32 or a 16-bit type, both of one
    type, or None. `mean` / `rstd` [M] fp32 keep the statistics for the backward pass. `out` and
    `sum` may be x or res themselves where types and strides agree."""
    c = "layer_norm"
    dev = _gpu(c, x, 2, _ANY, "x [M, C] of fp32, fp16 or bf16")
    shape = M, C = x.shape
    t = x.dtype
    same = (t,)
    if C >= _MOST_C:
        raise ValueError(f"{c}: rows of {C} elements (below 2^29)")
    if (res is None) != (sum is None):
        raise ValueError(f"{c}: res and sum come together")
    xs = _rows(c, "x", x, shape, same, dev)
    ys = _rows(c, "out", out, shape, _ANY if t is torch.float32 else same, dev, True)
    rs = ss = 0
    if res is not None:
        rs, ss = _rows(c, "res", res, shape, same, dev), _rows(c, "sum", sum, shape, same, dev, True)
    wt = (weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32)
    _flat(c, "weight", weight, (C,), _ANY, dev)
    _flat(c, "bias", bias, (C,), (wt,), dev)
    _flat(c, "mean", mean, (M,), _F32, dev)
    _flat(c, "rstd", rstd, (M,), _F32, dev)
    if wt not in _TYPES:
        _refuse(c, "bias", bias, (C,), _ANY, dev, "contiguous")
    a = nat.LayerNormArgs(x.data_ptr(), _ptr(res), _ptr(weight), _ptr(bias), out.data_ptr(), _ptr(sum), _ptr(mean),
                          _ptr(rstd), M, xs, rs, ys, ss, C, _TYPES[t], _TYPES[out.dtype], _TYPES[wt], eps)
    _launch("dn8_layer_norm", nat.lib().dn8_layer_norm, a, dev, stream)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                        rstd: torch.Tensor, dx: torch.Tensor, dweight: torch.Tensor | None = None,
                        dbias: torch.Tensor | None = None, dsum: torch.Tensor | None = None,
                        work: torch.Tensor | None = None, stream=None) -> None:
    """The gradient of `layer_norm`: x is what it normalised (`sum` where there was a residual), dy the
    gradient of its output (the output's type), dsum the gradient that reaches the sum past the
    norm. dx (x's type) is the gradient of x and of the residual alike; dweight / dbias [C] of the
    weight's type (fp32 without a weight) are sums over the rows, the same bits every call. dx may be
    dy, x or dsum itself where types and strides agree. `work`: uint8 of `dn8_layer_norm_bwd_work(C)`
    bytes, allocated if not given."""
    c = "layer_norm_backward"
    dev = _gpu(c, x, 2, _ANY, "x [M, C] of fp32, fp16 or bf16")
    shape = M, C = x.shape
    t = x.dtype
    same = (t,)
    if C >= _MOST_C:
        raise ValueError(f"{c}: rows of {C} elements (below 2^29)")
    xs, gs = _rows(c, "x", x, shape, same, dev), _rows(c, "dy", dy, shape, _ANY if t is torch.float32 else same, dev)
    ds = 0 if dsum is None else _rows(c, "dsum", dsum, shape, same, dev)
    os = _rows(c, "dx", dx, shape, same, dev, True)
    wt = torch.float32 if weight is None else weight.dtype
    _flat(c, "weight", weight, (C,), _ANY, dev)
    _flat(c, "dweight", dweight, (C,), (wt,), dev)
    _flat(c, "dbias", dbias, (C,), (wt,), dev)
    if mean is None or rstd is None:
        raise ValueError(f"{c}: mean and rstd are needed")
    _flat(c, "mean", mean, (M,), _F32, dev)
    _flat(c, "rstd", rstd, (M,), _F32, dev)
    lib = nat.lib()
    if dweight is not None or dbias is not None:
        work = _workspace(c, lib.dn8_layer_norm_bwd_work(C), work, dev, stream)
    a = nat.LayerNormBwdArgs(_ptr(dy), _ptr(x), _ptr(weight), _ptr(dsum), _ptr(mean), _ptr(rstd), _ptr(dx),
                             _ptr(dweight), _ptr(dbias), _ptr(work), M, gs, xs, ds, os, C, _TYPES[t],
                             _TYPES[dy.dtype], _TYPES[wt])
    _launch("dn8_layer_norm_bwd", lib.dn8_layer_norm_bwd, a, dev, stream)


_SECTIONS = nat.I32 * nat.DN8_ROPE_AXES


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
    dev = _gpu(c, q, 3, _ANY, "q [T, H, D] of fp32, fp16 or bf16")
    shape = T, Hq, D = q.shape
    t = (q.dtype,)
    axes = len(sections)
    if not 1 <= axes <= nat.DN8_ROPE_AXES:
        raise ValueError(f"{c}: 1 to {nat.DN8_ROPE_AXES} axes")
    if min(sections) < 0 or 2 * sum(sections) > D or Hq > _MOST_HEADS or D > _MOST_HEADS:
        raise ValueError(f"{c}: sections {tuple(sections)} of {Hq} heads of {D} elements")
    _flat(c, "pos", pos, (T, axes), _I32, dev)
    if pos is None or (k is None) != (k_out is None):
        raise ValueError(f"{c}: pos is needed, and k and k_out come together")
    qs, qo = _heads(c, "q", q, shape, t, dev), _heads(c, "q_out", q_out, shape, t, dev, True)
    Hk, ks, ko = 0, (0, 0), (0, 0)
    if k is not None:
        if not isinstance(k, torch.Tensor) or k.dim() != 3:
            raise ValueError(f"{c}: k [T, H, D] expected")
        Hk = k.shape[1]
        if Hk > _MOST_HEADS:
            raise ValueError(f"{c}: {Hk} heads")
        ks, ko = _heads(c, "k", k, (T, Hk, D), t, dev), _heads(c, "k_out", k_out, (T, Hk, D), t, dev, True)
    a = nat.RopeArgs(q.data_ptr(), _ptr(k), pos.data_ptr(), q_out.data_ptr(), _ptr(k_out), T, *qs, *ks, *qo, *ko, Hq, Hk,
                     D, _TYPES[t[0]], axes, _SECTIONS(*sections), per_axis, interleaved, inverse, base)
    _launch("dn8_rope", nat.lib().dn8_rope, a, dev, stream)


_FAR = 1 << 29                                               # beyond every length: no limit


def _packed(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale):
    """(device, shapes, head strides of q, k, v, mask fields) of an attention call."""
    dev = _gpu(c, q, 3, _HALF, "q [Tq, Hq, D], k [Tk, Hk, D] of fp16 or bf16")
    if not isinstance(k, torch.Tensor) or k.dim() != 3 or not isinstance(cu_q, torch.Tensor) or cu_q.dim() != 1:
        raise ValueError(f"{c}: k [Tk, Hk, D] and cu_q int32 [B + 1] expected")
    sq, sk = q.shape, k.shape
    t = (q.dtype,)
    n = cu_q.shape[0]
    if n < 1 or n > _MOST_SEQUENCES or cu_k is None or sk[2] != sq[2]:
        raise ValueError(f"{c}: cu_q and cu_k int32 [B + 1], q and k of one head size expected")
    if sq[1] > _MOST_HEADS or sk[1] > _MOST_HEADS or sq[2] > _MOST_HEADS or min(left, right, sinks) < -1:
        raise ValueError(f"{c}: q {tuple(sq)}, k {tuple(sk)}, left={left}, right={right}, sinks={sinks}")
    _flat(c, "cu_q", cu_q, (n,), _I32, dev)
    _flat(c, "cu_k", cu_k, (n,), _I32, dev)
    _flat(c, "len_k", len_k, (n - 1,), _I32, dev)
    _flat(c, "keep", keep, sk[:1], _FLAG, dev)
    _flat(c, "lse", lse, sq[:2], _F32, dev)
    _flat(c, "err", err, (1,), _I32, dev)
    strides = (*_heads(c, "q", q, sq, t, dev), *_heads(c, "k", k, sk, t, dev), *_heads(c, "v", v, sk, t, dev))
    mask = (n - 1, sq[1], sk[1], sq[2], _TYPES[q.dtype], min(left, _FAR), min(right, _FAR), min(sinks, _FAR),
            sq[2] ** -0.5 if scale is None else scale)
    return dev, sq, sk, t, strides, mask


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
    0 and -inf. Keys that no query of their sequence sees (by keep, len_k or the window) may hold anything
    (NaN included), the others must be finite. Rows of no sequence are left as they are. Offsets are read
    on the device: a sequence outside the tensors counts as empty and sets `err` (int32 [1]). `work`:
    uint8 of `dn8_attention_work` bytes, allocated if needed and not given."""
    c = "attention"
    dev, sq, sk, t, strides, mask = _packed(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale)
    os = _heads(c, "out", out, sq, t, dev, True)
    a = nat.AttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), cu_q.data_ptr(),
                          cu_k.data_ptr(), _ptr(len_k), _ptr(keep), _ptr(err), None, sq[0], sk[0], *strides, *os, *mask)
    lib = nat.lib()
    nbytes = _bytes_of(lib.dn8_attention_work, a, dev)
    if nbytes > 0:
        work = _workspace(c, nbytes, work, dev, stream)
        a.work = work.data_ptr()
    _launch("dn8_attention", lib.dn8_attention, a, dev, stream)


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, cu_q: torch.Tensor,
                       cu_k: torch.Tensor, left: int = -1, right: int = -1, sinks: int = 0,
                       keep: torch.Tensor | None = None, len_k: torch.Tensor | None = None, scale: float | None = None,
                       err: torch.Tensor | None = None, work: torch.Tensor | None = None, stream=None) -> None:
    """The gradient of `attention` from its inputs, its `out` and `lse` and the gradient `dout` of out:
    dq [Tq, Hq, D], dk and dv [Tk, Hk, D] (summed over the query heads that share a key head), all
    of the inputs' type and with strides of their own. The same bits every call (no atomics). Rows of
    no sequence are left as they are. `work`: uint8 of `dn8_attention_bwd_work` bytes, allocated if not
    given."""
    c = "attention_backward"
    if lse is None:
        raise ValueError(f"{c}: lse is needed")
    dev, sq, sk, t, strides, mask = _packed(c, q, k, v, cu_q, cu_k, len_k, keep, lse, err, left, right, sinks, scale)
    gs, os = _heads(c, "dout", dout, sq, t, dev), _heads(c, "out", out, sq, t, dev)
    outs = (*_heads(c, "dq", dq, sq, t, dev, True), *_heads(c, "dk", dk, sk, t, dev, True),
            *_heads(c, "dv", dv, sk, t, dev, True))
    a = nat.AttentionBwdArgs(_ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv),
                             _ptr(cu_q), _ptr(cu_k), _ptr(len_k), _ptr(keep), _ptr(err), None, sq[0], sk[0], *gs,
                             *strides, *os, *outs, *mask)
    lib = nat.lib()
    nbytes = _bytes_of(lib.dn8_attention_bwd_work, a, dev)
    if nbytes > 0:
        work = _workspace(c, nbytes, work, dev, stream)
        a.work = work.data_ptr()
    _launch("dn8_attention_bwd", lib.dn8_attention_bwd, a, dev, stream)


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
