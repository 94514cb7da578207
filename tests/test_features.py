"""The feature operators' entry points without a GPU: structures, refusals, sizes (nothing is launched, no pointer is followed)."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ESHAPE, EWORKSPACE = -1, -2, -4
FAKE = 0x10000


def lib():
    from cuke_amd import _lib
    return _lib, _lib.lib()


def linear(rows=8, fin=16, fout=16, type=1, out_type=1, act=0, x=FAKE, xs=None, w=FAKE, ws=None, b=None, res=None, rs=0, p=0.0):
    from cuke_amd import _lib
    return _lib.Linear(type, out_type, act, 0, rows, fin, fout, x, fin if xs is None else xs, w, fin if ws is None else ws, b, res, rs, p, 0, 0, None)


def preference(B=4, N=8, type=0, kind=0, pos=FAKE, neg=FAKE, ns=None, rp=None, rn=None, rs=0, mask=None, ms=0, beta=1.0, sign=1.0, smoothing=0.0, heat=0.0):
    from cuke_amd import _lib
    return _lib.Preference(type, kind, B, N, pos, neg, N if ns is None else ns, rp, rn, rs, mask, ms, beta, sign, smoothing, heat)


def test_structures_are_laid_out_as_in_c(tmp_path):
    _lib, _ = lib()
    names = {"kge_linear": _lib.Linear, "kge_preference": _lib.Preference}
    fields = [(n, f[0]) for n, t in names.items() for f in t._fields_]
    prints = "".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in names)
    prints += "".join(f'printf("{n}.{f} %zu\\n", offsetof({n}, {f.rstrip("_")}));' for n, f in fields)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include "kge_mi355.h"\nint main(void) {{ {prints} return 0; }}\n')
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, t in names.items():
        assert int(got[n]) == C.sizeof(t)
    for n, f in fields:
        assert int(got[f"{n}.{f}"]) == getattr(names[n], f).offset, (n, f)


def test_constants_are_those_of_the_header():
    import re
    _lib, _ = lib()
    text = open(os.path.join(ROOT, "include", "kge_mi355.h")).read()
    value = {k: int(v) for k, v in re.findall(r"\b(KGE_[A-Z0-9_]+) = (\d+)", text)}
    assert _lib.TYPES == {"float32": value["KGE_F32"], "bfloat16": value["KGE_BF16"], "float16": value["KGE_F16"]}
    assert _lib.ACTS == {a: value["KGE_ACT_" + a.upper()] for a in ("none", "relu", "gelu", "silu")}
    assert _lib.PREFERENCES == {k: value["KGE_PREFER_" + k.upper()] for k in ("sigmoid", "hinge", "square")}


@pytest.mark.parametrize("bad,rc", [
    (dict(type=7), EINVAL), (dict(type=1, out_type=2), EINVAL), (dict(type=0, out_type=1), EINVAL), (dict(act=9), EINVAL), (dict(act=-1), EINVAL),
    (dict(p=-0.1), EINVAL), (dict(p=1.1), EINVAL), (dict(p=float("nan")), EINVAL), (dict(rows=-1), ESHAPE), (dict(fin=-1, xs=8, ws=8), ESHAPE),
    (dict(rows=1 << 31), ESHAPE), (dict(xs=15), ESHAPE), (dict(ws=8), ESHAPE), (dict(res=FAKE, rs=4), ESHAPE), (dict(x=None), EINVAL),
    (dict(w=None), EINVAL), (dict(rows=1 << 30, fout=1 << 30), ESHAPE)])
def test_linear_refusals(bad, rc):
    _, L = lib()
    d = linear(**bad)
    assert L.kge_linear_fwd(C.byref(d), FAKE, 1 << 31, 0, None, 0, FAKE, 1 << 40, None) == rc
    assert L.kge_linear_bwd(C.byref(d), FAKE, 1 << 31, FAKE, 1 << 40, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == rc
    assert L.kge_linear_saved_bytes(C.byref(d)) == 0 and L.kge_linear_bwd_workspace(C.byref(d)) == 0


def test_linear_outputs_and_workspaces_are_checked():
    _, L = lib()
    assert L.kge_linear_fwd(None, FAKE, 16, 0, None, 0, None, 0, None) == EINVAL
    assert L.kge_linear_bwd(None, FAKE, 16, None, 0, None, None, None, None, 0, None) == EINVAL
    d = linear(act=2)
    assert L.kge_linear_fwd(C.byref(d), None, 16, 0, None, 0, None, 0, None) == EINVAL
    assert L.kge_linear_fwd(C.byref(d), FAKE, 15, 0, None, 0, None, 0, None) == ESHAPE
    saved = L.kge_linear_saved_bytes(C.byref(d))
    assert saved >= 8 * 16 * 2
    assert L.kge_linear_fwd(C.byref(d), FAKE, 16, 1, None, 0, None, 0, None) == EWORKSPACE
    assert L.kge_linear_fwd(C.byref(d), FAKE, 16, 1, FAKE, saved - 1, None, 0, None) == EWORKSPACE
    assert L.kge_linear_fwd(C.byref(d), FAKE, 16, 1, FAKE + 8, saved, None, 0, None) == EWORKSPACE
    assert L.kge_linear_bwd(C.byref(d), FAKE, 15, FAKE, saved, FAKE, FAKE, None, FAKE, 1 << 30, None) == ESHAPE
    assert L.kge_linear_bwd(C.byref(d), None, 16, FAKE, saved, FAKE, FAKE, None, FAKE, 1 << 30, None) == EINVAL
    assert L.kge_linear_bwd(C.byref(d), FAKE, 16, None, 0, FAKE, FAKE, None, FAKE, 1 << 30, None) == EWORKSPACE
    assert L.kge_linear_bwd(C.byref(d), FAKE, 16, FAKE, saved, FAKE, FAKE, None, None, 0, None) == EWORKSPACE
    # nothing to write is no error
    for empty in (linear(rows=0, x=None), linear(fout=0, w=None)):
        assert L.kge_linear_fwd(C.byref(empty), None, 16, 0, None, 0, None, 0, None) == 0
    for empty in (linear(rows=0), linear(fin=0), linear(fout=0), linear(rows=0, fin=0, fout=0)):
        for act in (0, 2):
            empty.act = act
            assert L.kge_linear_saved_bytes(C.byref(empty)) <= 512 and L.kge_linear_bwd_workspace(C.byref(empty)) <= 1024
            assert L.kge_linear_fwd_workspace(C.byref(empty), 0) == 0


def test_linear_saves_no_more_than_it_needs():
    """Rows of whole 16-byte chunks are read where they lie, and so is fp32; odd 16-bit widths, strides and addresses take a packed copy."""
    _, L = lib()
    size = lambda **kw: L.kge_linear_saved_bytes(C.byref(linear(rows=64, fin=64, fout=32, **kw)))
    assert size() == 0
    assert size(act=1) == 64 * 32 * 2
    assert size(xs=68) == 64 * 64 * 2 and size(x=FAKE + 2) == 64 * 64 * 2 and size(xs=72) == 0
    assert size(w=FAKE + 8) == 32 * 64 * 2
    assert size(type=0, out_type=0) == 0 and size(type=0, out_type=0, x=FAKE + 4, xs=65) == 0
    assert size(type=0, out_type=0, act=3) == 4 * 64 * 32


@pytest.mark.parametrize("bad,rc", [
    (dict(type=3), EINVAL), (dict(kind=5), EINVAL), (dict(beta=0.0), EINVAL), (dict(beta=float("nan")), EINVAL), (dict(beta=float("inf")), EINVAL),
    (dict(sign=0.0), EINVAL), (dict(smoothing=1.5), EINVAL), (dict(smoothing=0.1, kind=1), EINVAL), (dict(heat=-1.0), EINVAL), (dict(heat=float("inf")), EINVAL),
    (dict(B=-1), ESHAPE), (dict(N=-1, ns=0), ESHAPE), (dict(ns=7), ESHAPE), (dict(rp=FAKE), EINVAL), (dict(rn=FAKE, rs=8), EINVAL),
    (dict(rp=FAKE, rn=FAKE, rs=7), ESHAPE), (dict(mask=FAKE, ms=7), ESHAPE), (dict(pos=None), EINVAL), (dict(neg=None), EINVAL)])
def test_preference_refusals(bad, rc):
    _, L = lib()
    d = preference(**bad)
    assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == rc
    assert L.kge_preference_workspace(C.byref(d)) == 0


def test_preference_workspace_and_outputs_are_checked():
    _, L = lib()
    d = preference()
    assert L.kge_preference_loss(None, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == EINVAL
    assert L.kge_preference_loss(C.byref(d), None, FAKE, FAKE, FAKE, 1 << 30, None) == EINVAL
    need = L.kge_preference_workspace(C.byref(d))
    assert need > 0
    assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, FAKE, need - 1, None) == EWORKSPACE
    assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, None, 0, None) == EWORKSPACE


@pytest.mark.parametrize("args,rc", [
    (dict(type=9), EINVAL), (dict(p=2.0), EINVAL), (dict(rows=-1), ESHAPE), (dict(cols=-1, xs=0, ys=0), ESHAPE), (dict(xs=3), ESHAPE), (dict(ys=3), ESHAPE),
    (dict(x=None), EINVAL), (dict(y=None), EINVAL), (dict(rows=0, x=None, y=None), 0), (dict(cols=0, x=None, y=None), 0)])
def test_dropout_refusals(args, rc):
    _, L = lib()
    a = dict(dict(type=0, x=FAKE, xs=4, y=FAKE, ys=4, rows=4, cols=4, p=0.5), **args)
    assert L.kge_dropout(a["type"], a["x"], a["xs"], a["y"], a["ys"], a["rows"], a["cols"], a["p"], 1, 0, None, None) == rc


def test_host_side_refuses_cpu_tensors():
    import torch
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    x = torch.zeros(4, 8)
    for call in (lambda: features.linear(x, x), lambda: features.dropout(x, 0.5, 1), lambda: features.preference_loss(x[:, 0], x)):
        with pytest.raises(KgeError):
            call()
