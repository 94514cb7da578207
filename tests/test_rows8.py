"""Rows in 8 bits and the norm without a GPU: structures, refusals, sizes (nothing is launched, no pointer is followed)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from eight import NUMBERS, pack64

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ESHAPE, EWORKSPACE = -1, -2, -4
FAKE = 0x10000


def lib():
    from cuke_amd import _lib
    return _lib, _lib.lib()


def rows8(q=FAKE, qs=64, scale=FAKE, ss=4):
    from cuke_amd import _lib
    return _lib.Rows8(q, qs, scale, ss)


def norm(rows=4, cols=40, type=1, out=1, x=FAKE, xs=40, res=None, rs=0, w=None, eps=1e-6):
    from cuke_amd import _lib
    return _lib.RmsNorm(type, out, rows, cols, x, xs, res, rs, w, eps)


def test_structures_are_laid_out_as_in_c(tmp_path):
    _lib, _ = lib()
    names = {"kge_rows8": _lib.Rows8, "kge_rms_norm": _lib.RmsNorm}
    fields = [(n, f[0]) for n, t in names.items() for f in t._fields_]
    prints = "".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in names) + 'printf("e4m3 %d\\n", KGE_E4M3);'
    prints += "".join(f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, f in fields)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "kge_mi355.h"\nint main(void) {{ {prints} return 0; }}\n')
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, t in names.items():
        assert int(got[n]) == C.sizeof(t)
    for n, f in fields:
        assert int(got[f"{n}.{f}"]) == getattr(names[n], f).offset, (n, f)
    assert int(got["e4m3"]) == _lib.E4M3


def test_the_reference_rounds_as_torch_does():
    """The list of numbers and their neighbours against torch's conversion on the CPU (which is not what the kernels are held to)."""
    v = np.concatenate([NUMBERS, (NUMBERS[1:] + NUMBERS[:-1]) / 2, np.random.default_rng(0).uniform(-448, 448, 4096)])
    v = np.concatenate([v, -v])
    x = np.zeros((len(v), 32))
    x[:, 0], x[:, 1] = v, 448.0       # (448 makes the unit 1)
    q, scale, values = pack64(x)
    assert (scale[:, 0] == 127).all()
    want = torch.from_numpy(v).to(torch.float32).to(torch.float8_e4m3fn)
    exact = torch.from_numpy(v).to(torch.float32).double().numpy() == v
    assert np.array_equal(values[exact, 0], want.double().numpy()[exact]) and np.array_equal(q[exact, 0], want.view(torch.uint8).numpy()[exact])


@pytest.mark.parametrize("bad,rc", [
    (dict(q=None), EINVAL), (dict(scale=None), EINVAL), (dict(q=FAKE + 8), EINVAL), (dict(scale=FAKE + 2), EINVAL), (dict(qs=32), ESHAPE),
    (dict(qs=72), ESHAPE), (dict(ss=0), ESHAPE), (dict(ss=6), ESHAPE)])
def test_rows_in_8_bits_are_checked(bad, rc):
    _, L = lib()
    r, n = rows8(**bad), norm(out=3)
    assert L.kge_pack8(0, FAKE, 40, 4, 40, C.byref(r), None) == rc
    assert L.kge_unpack8(C.byref(r), 4, 40, 0, FAKE, 40, None) == rc
    assert L.kge_rms_norm_fwd(C.byref(n), None, 0, C.byref(r), None, 0, None, None, None) == rc


@pytest.mark.parametrize("args,rc", [
    (dict(type=3), EINVAL), (dict(type=-1), EINVAL), (dict(rows=-1), ESHAPE), (dict(cols=-1), ESHAPE), (dict(rows=1 << 31), ESHAPE), (dict(xs=39), ESHAPE),
    (dict(x=None), EINVAL), (dict(rows=0, x=None), 0), (dict(cols=0, x=None), 0)])
def test_pack_refusals(args, rc):
    _, L = lib()
    a = dict(dict(type=0, x=FAKE, xs=40, rows=4, cols=40), **args)
    assert L.kge_pack8(a["type"], a["x"], a["xs"], a["rows"], a["cols"], C.byref(rows8()), None) == rc
    assert L.kge_unpack8(C.byref(rows8()), a["rows"], a["cols"], a["type"], a["x"], a["xs"], None) == rc
    assert L.kge_pack8(0, FAKE, 40, 4, 40, None, None) == EINVAL and L.kge_unpack8(None, 4, 40, 0, FAKE, 40, None) == EINVAL


@pytest.mark.parametrize("bad,rc", [
    (dict(type=3), EINVAL), (dict(out=4), EINVAL), (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL), (dict(eps=float("inf")), EINVAL),
    (dict(rows=-1), ESHAPE), (dict(cols=-1), ESHAPE), (dict(rows=1 << 31), ESHAPE), (dict(cols=1 << 31, xs=1 << 31), ESHAPE), (dict(xs=39), ESHAPE),
    (dict(res=FAKE, rs=39), ESHAPE), (dict(x=None), EINVAL)])
def test_norm_refusals(bad, rc):
    _, L = lib()
    d = norm(**bad)
    assert L.kge_rms_norm_fwd(C.byref(d), FAKE, 1 << 31, None, None, 0, None, None, None) == rc


def test_norm_outputs_and_workspaces_are_checked():
    _, L = lib()
    d = norm()
    fwd = lambda **k: L.kge_rms_norm_fwd(C.byref(k.get("d", d)), k.get("y", FAKE), k.get("ys", 40), None, k.get("h"), k.get("hs", 0), None, k.get("rest"), None)
    assert L.kge_rms_norm_fwd(None, FAKE, 40, None, None, 0, None, None, None) == EINVAL
    assert fwd(y=None) == EINVAL and fwd(rest=FAKE + 2) == EINVAL and fwd(ys=39) == ESHAPE and fwd(h=FAKE, hs=39) == ESHAPE
    assert L.kge_rms_norm_fwd(C.byref(norm(out=3)), FAKE, 40, None, None, 0, None, None, None) == EINVAL        # no y8
    assert fwd(d=norm(rows=0, x=None), y=None) == 0 and fwd(d=norm(cols=0, x=None), y=None) == 0
    need = L.kge_rms_norm_bwd_workspace(C.byref(d))
    assert need >= 40 * 4 and L.kge_rms_norm_bwd_workspace(None) == 0 and L.kge_rms_norm_bwd_workspace(C.byref(norm(type=9))) == 0
    ok = dict(h=FAKE, hs=40, rstd=FAKE, rest=None, t=1, dy=FAKE, dys=40, dh=None, dhs=0, dx=FAKE, dxs=40, dw=FAKE, ws=FAKE, n=need)

    def bwd(d=d, **k):
        a = dict(ok, **k)
        return L.kge_rms_norm_bwd(C.byref(d), a["h"], a["hs"], a["rstd"], a["rest"], a["t"], a["dy"], a["dys"], a["dh"], a["dhs"], a["dx"], a["dxs"], a["dw"],
                                  a["ws"], a["n"], None)
    assert bwd(t=3) == EINVAL and bwd(rest=FAKE + 1) == EINVAL and bwd(h=None) == EINVAL and bwd(rstd=None) == EINVAL and bwd(dy=None) == EINVAL
    assert bwd(hs=39) == ESHAPE and bwd(dys=39) == ESHAPE and bwd(dh=FAKE, dhs=39) == ESHAPE and bwd(dxs=39) == ESHAPE
    assert bwd(n=need - 1) == EWORKSPACE and bwd(ws=None) == EWORKSPACE and bwd(ws=FAKE + 8) == EWORKSPACE
    assert bwd(dx=None, dw=None, ws=None, n=0) == 0 and bwd(d=norm(cols=0), ws=None, n=0) == 0


def layer(type=1, out_type=None, rows=4, inn=40, out=24, weight=FAKE, ws=40, act=2, p=0.0):
    from cuke_amd import _lib
    return _lib.Linear(type, type if out_type is None else out_type, act, 0, rows, inn, out, None, 0, weight, ws, None, None, 0, p, 0, 0, None)


@pytest.mark.parametrize("bad,rc", [
    (dict(type=0), EINVAL), (dict(type=3), EINVAL), (dict(out_type=2), EINVAL), (dict(act=9), EINVAL), (dict(p=1.5), EINVAL), (dict(weight=None), EINVAL),
    (dict(rows=-1), ESHAPE), (dict(inn=-1), ESHAPE), (dict(ws=39), ESHAPE), (dict(rows=1 << 31), ESHAPE)])
def test_layers_of_rows_in_8_bits_refuse(bad, rc):
    _, L = lib()
    d, x = layer(**bad), rows8()
    assert L.kge_linear8_fwd(C.byref(d), C.byref(x), None, FAKE, 1 << 31, 0, None, 0, FAKE, 1 << 40, None) == rc
    assert L.kge_linear8_bwd(C.byref(d), C.byref(x), FAKE, 1 << 31, FAKE, 1 << 40, FAKE, FAKE, None, FAKE, 1 << 40, None) == rc
    assert L.kge_linear8_saved_bytes(C.byref(d)) == 0 and L.kge_linear8_fwd_workspace(C.byref(d), None, 0) == 0 and L.kge_linear8_bwd_workspace(C.byref(d)) == 0


@pytest.mark.parametrize("bad,rc", [
    (dict(q=None), EINVAL), (dict(scale=None), EINVAL), (dict(q=FAKE + 8), EINVAL), (dict(scale=FAKE + 2), EINVAL), (dict(qs=32), ESHAPE),
    (dict(qs=72), ESHAPE), (dict(ss=0), ESHAPE), (dict(ss=6), ESHAPE)])
def test_layers_check_their_rows_in_8_bits(bad, rc):
    _, L = lib()
    d, good, x = layer(), rows8(), rows8(**bad)
    fwd = lambda a, b: L.kge_linear8_fwd(C.byref(d), C.byref(a) if a else None, C.byref(b) if b else None, FAKE, 24, 0, None, 0, FAKE, 1 << 40, None)
    assert fwd(x, None) == rc and fwd(good, x) == rc and fwd(None, None) == EINVAL
    assert L.kge_linear8_bwd(C.byref(d), C.byref(x), FAKE, 24, FAKE, 1 << 40, FAKE, FAKE, None, FAKE, 1 << 40, None) == rc
    assert L.kge_linear8_bwd(C.byref(d), None, FAKE, 24, FAKE, 1 << 40, FAKE, FAKE, None, FAKE, 1 << 40, None) == EINVAL


def test_layers_check_outputs_blocks_and_workspaces():
    _, L = lib()
    d, x = layer(rows=300), rows8()
    saved, wide = L.kge_linear8_saved_bytes(C.byref(d)), L.kge_linear8_bwd_workspace(C.byref(d))
    assert saved >= 300 * 24 and wide >= 300 * 24 * 2
    for name in ("kge_linear8_saved_bytes", "kge_linear8_bwd_workspace"):
        assert getattr(L, name)(None) == 0
    assert L.kge_linear8_fwd_workspace(None, None, 0) == 0

    def fwd(d=d, y=FAKE, ys=24, keep=1, s=FAKE, sn=saved, w8=None):
        return L.kge_linear8_fwd(C.byref(d), C.byref(x), C.byref(w8) if w8 else None, y, ys, keep, s, sn, FAKE, 1 << 40, None)
    assert fwd(y=None) == EINVAL and fwd(ys=23) == ESHAPE and fwd(w8=rows8()) == EINVAL
    assert fwd(s=None) == EWORKSPACE and fwd(s=FAKE + 8) == EWORKSPACE and fwd(sn=saved - 1) == EWORKSPACE
    assert fwd(d=layer(rows=0), y=None) == 0 and fwd(d=layer(out=0), y=None, ys=0) == 0
    half = layer(type=2, rows=3000, out=1000, weight=None, ws=0)           # fp16 with the weight in 8 bits: widened into the workspace
    need = L.kge_linear8_fwd_workspace(C.byref(half), C.byref(rows8()), 0)
    assert need >= 1000 * 40 * 2
    for ws, n in ((None, need), (FAKE + 8, need), (FAKE, need - 1)):
        assert L.kge_linear8_fwd(C.byref(half), C.byref(x), C.byref(rows8()), FAKE, 1000, 0, None, 0, ws, n, None) == EWORKSPACE

    def bwd(d=d, x=x, dy=FAKE, dys=24, s=FAKE, sn=saved, ws=FAKE, n=wide):
        return L.kge_linear8_bwd(C.byref(d), C.byref(x), dy, dys, s, sn, FAKE, FAKE, None, ws, n, None)
    assert bwd(dy=None) == EINVAL and bwd(dys=23) == ESHAPE
    assert bwd(x=rows8(qs=1 << 26)) == ESHAPE and bwd(x=rows8(ss=1 << 26)) == ESHAPE           # (a stage's rows are addressed with 32 bits)
    assert bwd(s=None) == EWORKSPACE and bwd(sn=saved - 1) == EWORKSPACE and bwd(ws=None) == EWORKSPACE and bwd(n=wide - 1) == EWORKSPACE and bwd(ws=FAKE + 8) == EWORKSPACE


def test_rows8_says_what_it_takes():
    from cuke_amd import features
    q, s = torch.zeros((3, 64), dtype=torch.float8_e4m3fn), torch.zeros((3, 4), dtype=torch.uint8).view(torch.float8_e8m0fnu)
    assert features.Rows8(q, s, 40).shape == (3, 40) and features.Rows8(q, s, 64).shape == (3, 64)
    for bad in ((q, s, 32), (q, s, 65), (q, s, -1), (q[:2], s, 40), (q, s[:, :2], 40), (q[0], s[0], 40)):
        with pytest.raises(ValueError):
            features.Rows8(*bad)
    for bad in ((q.float(), s, 40), (q, s.view(torch.uint8), 40), (None, s, 40)):
        with pytest.raises(TypeError):
            features.Rows8(*bad)


def test_host_side_refuses_cpu_tensors():
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    x = torch.zeros(4, 8)
    r = features.Rows8(torch.zeros((4, 32), dtype=torch.float8_e4m3fn), torch.zeros((4, 4), dtype=torch.uint8).view(torch.float8_e8m0fnu), 8)
    for call in (lambda: features.pack8(x), lambda: features.unpack8(r), lambda: features.rms_norm(x)):
        with pytest.raises(KgeError):
            call()
    with pytest.raises(TypeError):
        features.unpack8(x)
