"""The root-mean-square norm where a formula loses its digits or a number its range: rows of one column, rows of the smallest numbers.

Tolerances as in test_gpu_rows8.py (u: half a step of a type, eps = 2^-24, r to 2 eps).  Of one column dx is eps_norm r^3 g, a product whose only error is that of
r: 6 eps, and its rounding.
"""
import ctypes as C
import dataclasses

import pytest
import torch

from test_gpu_rows8 import DEV, E4M3, EPS, TINY, TYPES, U, Norm, laid, within

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def one_column(c):
    """(dx, its tolerance) of a Norm of one column."""
    dx = c.eps * c.r ** 3 * c.dy.double() * c.w64
    tol = 8 * EPS * dx.abs()
    if c.dh is not None:
        dx, tol = dx + c.dh.double(), tol + 2 * EPS * c.dh.double().abs()
    return dx, tol + U[c.dtype] * (dx.abs() + tol) + TINY[c.dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dy", TYPES)
@pytest.mark.parametrize("weight", [False, True])
def test_gradients_of_one_column(dtype, dy, weight):
    """Two nearly equal terms leave some 1e-6 of themselves: of each row as exact as of longer ones."""
    from cuke_amd import features
    for rows in (1, 10, 257, 5000):
        for eps in (1e-6, 1e-2, 0.0, 7.0):
            for layout in ("plain", "apart"):
                c = Norm(rows, 1, dtype, residual=False, weight=weight, dy=dy, layout=layout, eps=eps)
                print("one column", dtype, dy, rows, eps, layout, flush=True)
                c.x.masked_fill_(c.x == 0, 1.0)
                c.h = c.x.double()
                c.r = (c.h.square() + eps).rsqrt()
                fw = c.forward()
                g = features.rms_norm_backward(fw, c.dy)
                within(g.x, *one_column(c), "dx")
                if weight:
                    n = c.dy.double() * c.h * c.r
                    tol = (rows + 8) * EPS * n.abs().sum(0)
                    within(g.weight, n.sum(0), tol + U[dtype] * (n.sum(0).abs() + tol) + TINY[dtype], "dweight")
                c.dh = (c.dy.double() * 1e-6).to(dtype)
                within(features.rms_norm_backward(fw, c.dy, c.dh, need_weight=False).x, *one_column(c), "dx with dh")


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_of_one_column_of_a_sum(dtype):
    from cuke_amd import features
    c = Norm(300, 1, dtype, eps=1e-4)
    fw = c.forward()
    assert fw.eps == 1e-4
    c.dh = None
    within(features.rms_norm_backward(fw, c.dy).x, *one_column(c), "dx")


def test_gradients_of_one_column_against_differences():
    from cuke_amd import features
    c = Norm(50, 1, torch.float32, residual=False, eps=0.5)
    g = features.rms_norm_backward(c.forward(), c.dy)
    value = lambda t: (c.dy.double() * c.w64 * (c.h + t) * ((c.h + t).square() + c.eps).rsqrt())
    t = 1e-4
    slope = (value(t) - value(-t)) / (2 * t)                                          # off by t^2 / 6 times a third derivative, |dy w| 30 at most
    within(g.x, slope, 5 * t * t * (c.dy.double() * c.w64).abs() + 8 * EPS * slope.abs() + 1e-12, "dx")


def test_one_column_that_is_not_a_number():
    from cuke_amd import features
    inf, nan = float("inf"), float("nan")
    for eps in (0.0, 1e-6):
        x = torch.tensor([[0.0], [inf], [-inf], [nan], [2.0]], device=DEV)
        fw = features.rms_norm_forward(x, eps=eps)
        dx = features.rms_norm_backward(fw, torch.ones_like(x)).x
        assert torch.isnan(dx[1:4]).all() and not torch.isnan(dx[4])
        assert torch.isnan(dx[0]) if eps == 0 else abs(dx[0].item() - 1e3) < 1e-3            # (0 / 0, as the formula says)
        dx = features.rms_norm_backward(fw, torch.tensor([[1.0], [1.0], [1.0], [1.0], [nan]], device=DEV)).x
        assert torch.isnan(dx[4])


def test_one_column_by_the_c_call():
    """In the place of dy and of dh, with nothing written beside the rows."""
    from cuke_amd import _lib, features
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for dtype in TYPES:
        c = Norm(300, 1, dtype, eps=1e-3)
        fw = c.forward()
        want = features.rms_norm_backward(fw, c.dy, c.dh)
        d = _lib.RmsNorm(CODE[dtype], CODE[dtype], 300, 1, None, 0, None, 0, c.w.data_ptr(), 1e-3)
        n = L.kge_rms_norm_bwd_workspace(C.byref(d))
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        for place in ("dy", "dh", "apart"):
            wide = {k: torch.full((303, 4), 7.0, dtype=dtype, device=DEV) for k in ("dy", "dh", "apart")}
            wide["dy"][:300, :1], wide["dh"][:300, :1] = c.dy, c.dh
            dw = torch.empty(1, dtype=dtype, device=DEV)
            rest = fw.rest.data_ptr() if fw.rest is not None else None
            assert L.kge_rms_norm_bwd(C.byref(d), fw.h.data_ptr(), 1, fw.rstd.data_ptr(), rest, CODE[dtype], wide["dy"].data_ptr(), 4, wide["dh"].data_ptr(), 4,
                                      wide[place].data_ptr(), 4, dw.data_ptr(), ws.data_ptr(), n, st) == 0
            assert torch.equal(wide[place][:300, :1], want.x) and torch.equal(dw, want.weight), (dtype, place)
            assert all(bool((t[300:] == 7).all()) and bool((t[:, 1:] == 7).all()) for t in wide.values())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 3, 4, 5, 6, 7])
def test_few_columns_and_many_rows(cols, dtype):
    """Ranges of rows that end inside a workgroup's turn, one and several turns a range; the same call gives the same bits."""
    from cuke_amd import features
    for i, rows in enumerate((255, 256, 257, 70001, 300000)):
        print("few columns", rows, cols, dtype, flush=True)
        c = Norm(rows, cols, dtype, residual=i % 2 == 0, weight=i != 1, layout=("plain", "apart")[i % 2])
        fw = c.forward()
        for dy in TYPES:
            c.dy = c.dy.to(dy)
            g = features.rms_norm_backward(fw, c.dy, c.dh)
            c.check_backward(fw, g, (rows, cols))
            again = features.rms_norm_backward(fw, c.dy, c.dh)
            assert torch.equal(g.x, again.x) and (g.weight is None or torch.equal(g.weight, again.weight))
            alone = features.rms_norm_backward(fw, c.dy, c.dh, need_weight=False)
            assert torch.equal(alone.x, g.x) and alone.weight is None
        if c.w is not None:
            assert torch.equal(features.rms_norm_backward(fw, c.dy, need_x=False).weight, g.weight)


def test_few_columns_by_the_c_call():
    """dx in the place of dy and of dh; nothing is written beside rows, behind the last one or behind the workspace."""
    from cuke_amd import _lib, features
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for dtype in TYPES:
        for cols in (2, 5, 7):
            c = Norm(777, cols, dtype)
            fw = c.forward()
            want = features.rms_norm_backward(fw, c.dy, c.dh)
            d = _lib.RmsNorm(CODE[dtype], CODE[dtype], 777, cols, None, 0, None, 0, c.w.data_ptr(), c.eps)
            n = L.kge_rms_norm_bwd_workspace(C.byref(d))
            for place in ("dy", "dh", "apart"):
                wide = {k: torch.full((780, cols + 3), 7.0, dtype=dtype, device=DEV) for k in ("dy", "dh", "apart")}
                wide["dy"][:777, :cols], wide["dh"][:777, :cols] = c.dy, c.dh
                dw, ws = torch.full((cols + 4,), 7.0, dtype=dtype, device=DEV), torch.full((n + 64,), 0x5A, dtype=torch.uint8, device=DEV)
                rest = fw.rest.data_ptr() if fw.rest is not None else None
                assert L.kge_rms_norm_bwd(C.byref(d), fw.h.data_ptr(), cols, fw.rstd.data_ptr(), rest, CODE[dtype], wide["dy"].data_ptr(), cols + 3, wide["dh"].data_ptr(),
                                          cols + 3, wide[place].data_ptr(), cols + 3, dw.data_ptr(), ws.data_ptr(), n, st) == 0
                assert torch.equal(wide[place][:777, :cols], want.x) and torch.equal(dw[:cols], want.weight), (dtype, cols, place)
                assert all(bool((t[777:] == 7).all()) and bool((t[:, cols:] == 7).all()) for t in wide.values())
                assert bool((dw[cols:] == 7).all()) and bool((ws[n:] == 0x5A).all())


def test_few_columns_in_a_graph():
    from cuke_amd import features
    c = Norm(3000, 3, torch.bfloat16)
    fw = c.forward()
    features.rms_norm_backward(fw, c.dy, c.dh)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = features.rms_norm_backward(fw, c.dy, c.dh)
    for _ in range(3):
        c.dy.mul_(0.7)
        eager = features.rms_norm_backward(fw, c.dy, c.dh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g.x, eager.x) and torch.equal(g.weight, eager.weight)
