"""The root-mean-square norm of rows so small that their r does not fit into fp32 (2^128 and more: a root mean square below 2^-128, which only an eps below
2^-256 leaves so).

Tolerances as in test_gpu_rows8.py: the numbers are multiplied by 2^64, which rounds nothing, and r by 2^-64.
"""
import dataclasses

import pytest
import torch

from test_gpu_rows8 import DEV, E4M3, EPS, TINY, U, Norm

pytestmark = pytest.mark.gpu

WIDE = [torch.float32, torch.bfloat16]      # (fp16 has no such numbers)


def small_rows(rows, cols, dtype, residual=False, out=None, eps=0.0, every=2):
    """A Norm whose every `every`-th row is of a few of the smallest numbers, with gradients that leave dx finite."""
    c = Norm(rows, cols, dtype, residual=residual, out=out, eps=eps)
    g = torch.Generator().manual_seed(rows + cols)
    few = lambda: (torch.randint(0, 8, (rows, cols), generator=g) * 2 - 7).to(DEV).double() * TINY[dtype]        # odd, so that none (and no sum below) is zero
    pick = (torch.arange(rows, device=DEV) % every == 0)[:, None]
    c.x = torch.where(pick, few(), c.x.double()).to(dtype)
    if residual:
        c.res = torch.where(pick, 2 * few(), c.res.double()).to(dtype)
        c.dh = torch.where(pick, c.dh.double() * 1e10, c.dh.double()).to(dtype)
    c.dy = torch.where(pick, c.dy.double() * 2.0 ** -40, c.dy.double()).to(dtype)
    c.h = c.x.double() + (c.res.double() if residual else 0.0)
    c.r = (c.h.square().mean(1, keepdim=True) + eps).rsqrt()
    c.y = c.h * c.r * c.w64 if c.w is not None else c.h * c.r
    c.small = pick[:, 0]
    assert bool((c.r[c.small] >= 2.0 ** 128).any())
    return c


def real(fw, c):
    """fw, its rstd as the numbers it stands for."""
    kept = fw.rstd.double()
    assert torch.equal(kept < 0, c.r[:, 0] >= 2.0 ** 128)
    return dataclasses.replace(fw, rstd=torch.where(kept < 0, -kept * 2.0 ** 64, kept))


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("cols", [2, 5, 8, 40, 300, 1000, 2048, 8192, 9000])
@pytest.mark.parametrize("residual", [False, True])
def test_the_smallest_rows(cols, residual, dtype):
    from cuke_amd import features
    for rows in (1, 6, 300):
        print("smallest", rows, cols, residual, dtype, flush=True)
        c = small_rows(rows, cols, dtype, residual)
        fw = c.forward()
        c.check_forward(real(fw, c), (rows, cols))
        g = features.rms_norm_backward(fw, c.dy, c.dh)
        assert bool(torch.isfinite(g.weight).all())
        c.check_backward(fw, g, (rows, cols))
        c = small_rows(rows, cols, dtype, residual, out=E4M3)
        c.check_forward(real(c.forward(), c), (rows, cols, "8 bits"))


@pytest.mark.parametrize("dtype", WIDE)
def test_the_smallest_rows_of_one_column(dtype):
    from cuke_amd import features
    c = small_rows(70, 1, dtype)
    fw = c.forward()
    c.check_forward(real(fw, c), "one column")
    assert bool((features.rms_norm_backward(fw, c.dy).x == 0).all())                            # eps = 0: y is a sign


def test_the_smallest_eps():
    """r between 2^128 and what the smallest numbers leave, by eps alone; a row of zeros is zeros."""
    from cuke_amd import features
    for eps in (1e-78, 1e-82, 1e-90, 1e-110):
        c = small_rows(40, 200, torch.float32, eps=eps)
        c.x[3] = 0
        c.h[3] = c.y[3] = 0
        c.r[3] = eps ** -0.5
        c.dy[3] *= 2.0 ** -100
        fw = c.forward()
        c.check_forward(real(fw, c), eps)
        c.check_backward(fw, features.rms_norm_backward(fw, c.dy), eps)
