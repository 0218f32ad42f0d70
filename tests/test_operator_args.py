"""CPU: the rotary and cross-attention entry points refuse bad arguments on the host, before any CUDA call (the
pointers below are placeholders that are never dereferenced)."""
import ctypes
import math

import pytest
import torch

from sa3_b200 import _lib

ARG, ALIGN, DTYPE, UNSUPPORTED = -1, -2, -3, -5
P = 0x100000


def rotary(**kw):
    a = dict(q=P, qo=P, k=None, ko=None, dtype=_lib.DT_BF16, rows=8, heads=2, kv=0, d=64, rot=32, ldq=128, ldqo=128, ldk=0,
             ldko=0, f=P, pos=None, per=0, off=0, il=0, inv=0, scale=1.0)
    a.update(kw)
    return _lib.load().sa3_rotary(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), ARG), (dict(qo=None), ARG), (dict(f=None), ARG), (dict(rows=-1), ARG), (dict(heads=0), ARG),
    (dict(d=0), ARG), (dict(rot=0), ARG), (dict(rot=33), ARG), (dict(rot=66), ARG), (dict(per=-1), ARG),
    (dict(ldq=127), ARG), (dict(ldqo=127), ARG), (dict(ko=P), ARG), (dict(kv=2), ARG),
    (dict(k=P, ko=P, kv=0, ldk=128, ldko=128), ARG), (dict(k=P, ko=None, kv=2, ldk=128, ldko=128), ARG),
    (dict(k=P, ko=P, kv=2, ldk=64, ldko=128), ARG), (dict(d=1024, rot=64, ldq=2048, ldqo=2048), UNSUPPORTED),
    (dict(dtype=_lib.DT_E4M3), DTYPE), (dict(dtype=7), DTYPE), (dict(q=P + 1), ALIGN), (dict(f=P + 4), ALIGN),
    (dict(pos=P + 2), ALIGN), (dict(dtype=_lib.DT_F32, qo=P + 2), ALIGN), (dict(rows=0), 0),
])
def test_rotary_refuses(kw, rc):
    assert rotary(**kw) == rc


def forward(**kw):
    a = dict(q=P, k=P, v=P, out=P, lse=None, cu_q=None, cu_k=None, lens=None, mask=None, batch=2, lq=4, lk=8, tq=8, tk=16,
             heads=4, kv=2, d=64, ldq=256, ldk=128, ldv=128, ldo=256, scale=0.125, dtype=_lib.DT_BF16, ws=None, nws=0)
    a.update(kw)
    return _lib.load().sa3_cross_attention(*a.values(), None)


def backward(**kw):
    a = dict(dout=P, q=P, k=P, v=P, out=P, lse=P, dq=P, dk=P, dv=P, cu_q=None, cu_k=None, lens=None, mask=None, batch=2,
             lq=4, lk=8, tq=8, tk=16, heads=4, kv=2, d=64, lddo=256, ldq=256, ldk=128, ldv=128, ldo=256, lddq=256, lddk=128,
             lddv=128, scale=0.125, dtype=_lib.DT_BF16, ws=P, nws=1 << 30)
    a.update(kw)
    return _lib.load().sa3_cross_attention_bwd(*a.values(), None)


SHARED = [
    (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(out=None), ARG), (dict(batch=-1), ARG),
    (dict(heads=0), ARG), (dict(kv=0), ARG), (dict(kv=3), ARG), (dict(tq=9), ARG), (dict(tk=15), ARG),
    (dict(lq=-1, tq=0), ARG), (dict(ldq=255), ARG), (dict(ldk=64), ARG), (dict(ldv=64), ARG), (dict(ldo=128), ARG),
    (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=math.nan), ARG), (dict(scale=math.inf), ARG),
    (dict(scale=3e38), ARG),
    (dict(d=96, ldq=384, ldk=192, ldv=192, ldo=384), UNSUPPORTED), (dict(dtype=_lib.DT_F32), DTYPE),
    (dict(q=P + 8), ALIGN), (dict(k=P + 2), ALIGN), (dict(out=P + 8), ALIGN), (dict(ldq=260), ALIGN),
    (dict(ldv=132), ALIGN), (dict(lens=P + 1), ALIGN), (dict(lse=P + 2), ALIGN), (dict(cu_q=P + 2), ALIGN),
    (dict(batch=70000, lq=1, tq=70000, lk=1, tk=70000), UNSUPPORTED),
    (dict(batch=1, lq=2 ** 31 - 1, tq=2 ** 31 - 1, heads=66, kv=2, ldq=4224, ldo=4224, lddo=4224, lddq=4224, lk=16),
     UNSUPPORTED),
]


@pytest.mark.parametrize("kw,rc", SHARED + [(dict(batch=0, tq=0, tk=0), 0), (dict(lq=0, tq=0, q=None, out=None), 0)])
def test_forward_refuses(kw, rc):
    kw = {k: v for k, v in kw.items() if k not in ("lddo", "lddq")}
    assert forward(**kw) == rc


@pytest.mark.parametrize("kw,rc", SHARED + [
    (dict(dout=None), ARG), (dict(dq=None), ARG), (dict(dk=None), ARG), (dict(dv=None), ARG), (dict(lse=None), ARG),
    (dict(lddo=128), ARG), (dict(lddq=128), ARG), (dict(lddk=64), ARG), (dict(lddv=64), ARG), (dict(lddk=129), ALIGN),
    (dict(dout=P + 8), ALIGN), (dict(dk=P + 4), ALIGN), (dict(ws=P + 8), ALIGN), (dict(batch=0, tq=0, tk=0), 0),
])
def test_backward_refuses(kw, rc):
    assert backward(**kw) == rc


A, B = 0x200000, 0x300000


@pytest.mark.parametrize("kw", [
    dict(qo=P, ldqo=256), dict(qo=A, k=P, ko=A, kv=2, ldk=128, ldko=128), dict(qo=A, k=A, ko=B, kv=2, ldk=128, ldko=128),
    dict(qo=A, k=B, ko=P, kv=2, ldk=128, ldko=128), dict(qo=A, k=B, ko=B, kv=2, ldk=128, ldko=256),
])
def test_rotary_refuses_overlaps(kw):
    assert rotary(**kw) == ARG


@pytest.mark.parametrize("kw", [dict(out=P), dict(out=A, k=A), dict(out=A, v=A)])
def test_forward_refuses_overlaps(kw):
    assert forward(**kw) == ARG


@pytest.mark.parametrize("which", [("dq", "dout"), ("dq", "q"), ("dq", "out"), ("dq", "k"), ("dk", "k"), ("dk", "dq"),
                                   ("dk", "dout"), ("dv", "v"), ("dv", "dk"), ("dv", "q")])
def test_backward_refuses_overlaps(which):
    own = {n: P + i * 0x100000 for i, n in enumerate(("dout", "q", "k", "v", "out", "dq", "dk", "dv"))}
    assert backward(**{**own, which[0]: own[which[1]]}) == ARG


def test_workspace_queries_refuse():
    lib = _lib.load()
    n = ctypes.c_longlong(0)
    assert lib.sa3_cross_attention_workspace(1, 1, 1, 1, 2, 1, 64, None) == ARG
    assert lib.sa3_cross_attention_workspace(1, 1, 1, 1, 3, 2, 64, ctypes.byref(n)) == ARG
    assert lib.sa3_cross_attention_workspace(1, 1, 1, 1, 2, 1, 32, ctypes.byref(n)) == UNSUPPORTED
    assert lib.sa3_cross_attention_bwd_workspace(1, 1, 1, 1, 1, 2, 1, 64, None) == ARG
    assert lib.sa3_cross_attention_bwd_workspace(-1, 1, 1, 1, 1, 2, 1, 64, ctypes.byref(n)) == ARG
    assert lib.sa3_cross_attention_bwd_workspace(1, 1, 1, 1, 1, 2, 1, 65, ctypes.byref(n)) == UNSUPPORTED


def test_cpu_tensors_are_refused():
    from sa3_b200 import autograd, ops

    x = torch.zeros(4, 128)
    f = torch.ones(16, dtype=torch.float64)
    o = torch.zeros(4, 128, dtype=torch.bfloat16)
    for mod in (ops, autograd):
        with pytest.raises(RuntimeError, match="CUDA"):
            mod.rotary(x, f, heads=2)
        with pytest.raises(RuntimeError, match="CUDA"):
            mod.cross_attention(o, o, o, heads=2, max_seqlen_q=4, max_seqlen_k=4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.cross_attention_backward(o, o, o, o, o, torch.zeros(2, 4), heads=2, max_seqlen_q=4, max_seqlen_k=4)


def test_frequencies_on_the_host():
    """The formulas of the scalings, and their refusals."""
    from sa3_b200 import ops

    f, s = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64), rtol=1e-15)
    lin, s = ops.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin, f / 4, rtol=1e-15) and s == 1.0
    b, s = ops.rotary_frequencies(8, base=100.0, scaling="base", factor=4.0, device="cpu")
    assert math.isclose(float(b[-1]), float(f[-1]) / 4, rel_tol=1e-12) and float(b[0]) == 1.0 and s == 1.0
    r, s = ops.rotary_frequencies(8, base=100.0, scaling="ramp", factor=4.0, original_length=64, low_turns=0.5,
                                  high_turns=8.0, device="cpu")
    keep = ((64 * f / (2 * math.pi) - 0.5) / 7.5).clamp(0, 1)
    assert torch.allclose(r, f * keep + f / 4 * (1 - keep), rtol=1e-15)
    assert math.isclose(s, 0.1 * math.log(4.0) + 1.0)
    for kw in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, factor=0.0), dict(rot_dim=8, base=-1.0),
               dict(rot_dim=2, scaling="base"), dict(rot_dim=8, scaling="ramp"),
               dict(rot_dim=8, scaling="ramp", original_length=8, low_turns=2.0, high_turns=2.0),
               dict(rot_dim=8, scaling="other")):
        with pytest.raises(RuntimeError):
            ops.rotary_frequencies(device="cpu", **kw)
