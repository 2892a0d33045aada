"""The context transformer's operators without a GPU: the ctypes structures match include/dn8.h and bad
arguments are refused (DN8_EINVAL at the C entry, ValueError in Python) before any CUDA call."""
from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from rsna_knee_efficiency_b200 import _native as nat
from rsna_knee_efficiency_b200 import ops

ROOT = Path(__file__).resolve().parents[1]
STRUCTS = {"dn8_layer_norm_args": nat.LayerNormArgs, "dn8_layer_norm_bwd_args": nat.LayerNormBwdArgs,
           "dn8_rope_args": nat.RopeArgs, "dn8_attention_args": nat.AttentionArgs,
           "dn8_attention_bwd_args": nat.AttentionBwdArgs}


def test_struct_layouts_match_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dn8.h"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = ln.split()
        py = STRUCTS[s]
        assert int(v) == (ctypes.sizeof(py) if f == "size" else getattr(py, f).offset), (s, f)


def _attention(cls=nat.AttentionArgs, **kw):
    a = cls(B=1, Hq=4, Hk=2, D=64, type=nat.DN8_BF16, left=-1, right=-1, sinks=0, scale=0.1, Tq=4, Tk=8)
    for f, _ in cls._fields_:
        if f.endswith("stride_t"):
            setattr(a, f, 256)
        elif f.endswith("stride_h"):
            setattr(a, f, 64)
        elif f in ("q", "k", "v", "out", "cu_q", "cu_k", "dout", "dq", "dk", "dv", "lse", "work"):
            setattr(a, f, 4096)
    for f, v in kw.items():
        setattr(a, f, v)
    return a


@pytest.mark.parametrize("bad", [dict(D=0), dict(D=12), dict(D=136), dict(Hk=3), dict(Hk=0), dict(type=nat.DN8_F32), dict(B=-1),
                                 dict(Tq=-1), dict(Tk=1 << 28), dict(left=(1 << 29) + 1), dict(left=-2), dict(right=-2), dict(sinks=-1),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(q=4104), dict(k=None), dict(v=8),
                                 dict(q_stride_t=12), dict(scale=0.0), dict(scale=-1.0), dict(k_stride_h=0), dict(q_stride_t=0), dict(k_stride_h=-8), dict(cu_q=None)])
def test_attention_refusals(bad):
    lib = nat.lib()
    assert lib.dn8_attention(_attention(**bad), None) == nat.DN8_EINVAL
    assert lib.dn8_last_error().startswith(b"dn8_attention:")
    assert lib.dn8_attention_work(_attention(**bad)) == -1
    assert lib.dn8_attention_bwd(_attention(nat.AttentionBwdArgs, **bad), None) == nat.DN8_EINVAL
    assert lib.dn8_attention_bwd_work(_attention(nat.AttentionBwdArgs, **bad)) == -1


@pytest.mark.parametrize("bad", [dict(dk=None), dict(dv=8), dict(dq=None), dict(lse=None), dict(work=None),
                                 dict(dq_stride_t=4), dict(do_stride_h=1)])
def test_attention_bwd_refusals(bad):
    assert nat.lib().dn8_attention_bwd(_attention(nat.AttentionBwdArgs, **bad), None) == nat.DN8_EINVAL


def test_calls_with_nothing_to_do():
    lib = nat.lib()
    assert lib.dn8_attention(_attention(B=0), None) == nat.DN8_OK
    assert lib.dn8_attention(_attention(Tq=0), None) == nat.DN8_OK
    assert lib.dn8_attention_bwd(_attention(nat.AttentionBwdArgs, Tq=0, Tk=0), None) == nat.DN8_OK
    assert lib.dn8_layer_norm(nat.LayerNormArgs(rows=0, C=8), None) == nat.DN8_OK
    a = nat.RopeArgs(T=0, Hq=1, D=8, n_axes=1, base=10.0)
    a.sections[0] = 4
    assert lib.dn8_rope(a, None) == nat.DN8_OK


def test_layer_norm_refusals():
    lib = nat.lib()
    good = dict(x=4096, y=4096, rows=2, C=8, eps=1e-5)
    for bad in (dict(C=0), dict(rows=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None), dict(res=4096),
                dict(x_type=7), dict(w_type=-1), dict(x_type=nat.DN8_BF16, y_type=nat.DN8_F16), dict(x_type=1, y_type=0)):
        assert lib.dn8_layer_norm(nat.LayerNormArgs(**{**good, **bad}), None) == nat.DN8_EINVAL, bad
    good = dict(dy=4096, x=4096, mean=4096, rstd=4096, dx=4096, rows=2, C=8)
    for bad in (dict(C=0), dict(dy=None), dict(mean=None), dict(rstd=None), dict(dx=None), dict(dw=4096), dict(db=4096),
                dict(y_type=5)):
        assert lib.dn8_layer_norm_bwd(nat.LayerNormBwdArgs(**{**good, **bad}), None) == nat.DN8_EINVAL, bad
    assert lib.dn8_layer_norm_bwd_work(0) == -1


def test_rope_refusals():
    for bad in (dict(n_axes=0), dict(n_axes=5), dict(Hq=0), dict(D=7), dict(base=0.0), dict(base=float("nan")), dict(type=9),
                dict(q=None), dict(pos=None), dict(Hk=1), dict(T=-1), dict(sections=(4, -1)), dict(sections=(0, 0)),
                dict(sections=(200, 0), D=512)):
        sec = bad.pop("sections", (4, 0))
        a = nat.RopeArgs(**{**dict(q=4096, q_out=4096, pos=4096, T=2, Hq=1, D=8, n_axes=2, base=10.0), **bad})
        a.sections[0], a.sections[1] = sec
        assert nat.lib().dn8_rope(a, None) == nat.DN8_EINVAL, (bad, sec)


def test_python_refuses_host_tensors():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="GPU"):
        ops.layer_norm(x, None, None, x)
    with pytest.raises(ValueError, match="GPU"):
        ops.layer_norm_backward(x, x, None, x[:, 0], x[:, 0], x)
    q = torch.zeros(2, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.rope(q, None, torch.zeros(2, 1, dtype=torch.int32), q, None, (4,))
    cu = torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention(q, q, q, q, cu, cu)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_backward(q, q, q, q, q, q[..., 0].float(), q, q, q, cu, cu)
    with pytest.raises(ValueError, match=r"\[M, C\]"):
        ops.layer_norm(x.long(), None, None, x)
