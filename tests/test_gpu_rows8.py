"""Rows in 8 bits and the root-mean-square norm on the GPU against their definitions in 64 bits.

What is in 8 bits has to be equal: a power of two and the e4m3 number nearest to the 64-bit value are single answers.  Other tolerances, element by
element, from the roundings a result goes through (u: half a step of a type, eps = 2^-24):
  y      h = x + residual eps, r eps (from 64 bits), two products eps each: 4 eps |y|, doubled, and u |y|
  h      u |h| + eps |h|
  dx     a sum of K products in fp32 in any order: (K + 8) eps sum |g n|; its share of the row, and 8 eps of every other term; h of 16 bits with a residual is the
         sum to a 16th of a step; then u |dx|
  dweight  (M + 8) eps sum |dy n| and u |dweight|
"""
import ctypes as C
import dataclasses

import numpy as np
import pytest
import torch

from eight import NUMBERS, pack64

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # what lies below the normal numbers
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn
DEV = "cuda:0"


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for {want[i].item()} +- {tol.expand_as(want)[i].item()}")


def laid(x, layout):
    """x as it is, or as rows that start anywhere, some elements apart."""
    if layout == "plain":
        return x
    big = torch.full((x.shape[0], x.shape[1] + 5), float("nan"), dtype=x.dtype, device=x.device)
    big[:, 1:1 + x.shape[1]] = x
    return big[:, 1:1 + x.shape[1]]


def same_rows8(r, x64, what):
    """r holds what the definition says of x64, padding and all."""
    q, scale, _ = pack64(x64.cpu().numpy())
    got_q, got_s = r.q.view(torch.uint8).cpu().numpy(), r.scale.view(torch.uint8).cpu().numpy()
    assert np.array_equal(got_s, scale), f"{what}: {np.argwhere(got_s != scale)[:4].tolist()}"
    nan = (q & 0x7F) == 0x7F
    assert np.array_equal(nan, (got_q & 0x7F) == 0x7F), what
    zero = (q & 0x7F) == 0                                       # (the sign of a zero says nothing)
    diff = np.where(nan, False, np.where(zero, (got_q & 0x7F) != 0, got_q != q))
    assert not diff.any(), f"{what}: {int(diff.sum())} of {diff.size}, first at {np.argwhere(diff)[0].tolist()}"


# ---- to 8 bits and back ----------------------------------------------------------------------------
SIZES = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 100), (37, 300), (4, 127), (4, 128), (3, 129), (64, 512), (7, 1000), (2, 4096), (300, 8), (1, 70001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "apart"])
def test_pack_and_unpack(dtype, layout):
    from cuke_amd import features
    g = torch.Generator().manual_seed(1)
    for rows, cols in SIZES:
        x = torch.randn((rows, cols), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))
        x[:, ::17] *= 30
        x[rows // 2, :cols // 3] = 0
        x = laid(x.to(DEV).to(dtype), layout)
        r = features.pack8(x)
        assert r.shape == (rows, cols)
        same_rows8(r, x.double(), (rows, cols))
        values = torch.from_numpy(pack64(x.double().cpu().numpy())[2]).to(DEV)
        for t in TYPES:
            y = features.unpack8(r, t)
            assert y.dtype == t and torch.equal(y.double(), values.to(t).double()), (rows, cols, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_number(dtype):
    """All patterns, infinities and NaN among them: a block of one pattern each and one of 32 neighbours."""
    from cuke_amd import features
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype).to(DEV)
    for x in (every.view(2048, 32), every.view(65536, 1).contiguous(), every.view(32, 2048).t().contiguous()):
        r = features.pack8(x)
        same_rows8(r, x.double(), tuple(x.shape))
        back = features.unpack8(r, torch.float32).double()
        want = torch.from_numpy(pack64(x.double().cpu().numpy())[2]).to(DEV).float().double()       # (what rounds up to 2^128 is infinite in fp32)
        assert torch.equal(torch.nan_to_num(back, nan=7e77), torch.nan_to_num(want, nan=7e77))


def test_fp32_borders():
    """Numbers of e4m3 and the middles between them, each with its fp32 neighbours, in blocks of many powers; largest values around 448 2^k."""
    from cuke_amd import features
    mid = np.concatenate([NUMBERS, (NUMBERS[1:] + NUMBERS[:-1]) / 2]).astype(np.float32)
    v = np.concatenate([mid, np.nextafter(mid, np.float32(1e9)), np.nextafter(mid, np.float32(-1e9))])
    v = np.minimum(v, np.float32(448))
    for k in (-130, -127, -126, -100, -20, 0, 30, 100, 118):
        x = np.zeros((len(v), 32), np.float32)
        with np.errstate(under="ignore"):
            x[:, 5], x[:, 31] = np.ldexp(v, k), -np.ldexp(np.float32(448), k)
        same_rows8(features.pack8(torch.from_numpy(x).to(DEV)), torch.from_numpy(x).double(), k)
    top = np.array([np.ldexp(t, k) for k in (-140, -128, -60, 0, 60, 119) for t in np.float32([448, np.nextafter(np.float32(448), np.float32(500)), 447.99997, 256, 255.99998])],
                   np.float32)
    x = np.outer(top, np.linspace(-1, 1, 33)).astype(np.float32)
    same_rows8(features.pack8(torch.from_numpy(x).to(DEV)), torch.from_numpy(x).double(), "largest")
    huge = torch.tensor([[3.4028234e38, -3.4e38, 1.0, float("inf"), float("-inf"), float("nan")] + [1e30] * 30], device=DEV)
    same_rows8(features.pack8(huge), huge.double(), "huge")


def test_unpack_takes_every_byte():
    from cuke_amd import features
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1).to(DEV)
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 8).to(DEV)
    y = features.unpack8(features.Rows8(q.view(E4M3), scale.view(torch.float8_e8m0fnu), 256), torch.float32).cpu()
    want = q.cpu().view(E4M3).double() * scale.cpu()[:, :1].view(torch.float8_e8m0fnu).double()
    assert torch.equal(torch.nan_to_num(y, nan=7e30), torch.nan_to_num(want.float(), nan=7e30))


def test_rows8_made_elsewhere_and_empty_ones():
    from cuke_amd import features
    g = torch.Generator().manual_seed(2)
    x = torch.randn((9, 200), generator=g).to(DEV)
    r = features.pack8(x)
    want = features.unpack8(r, torch.float32)
    q = torch.zeros((9, 333), dtype=torch.uint8, device=DEV)
    s = torch.zeros((9, 13), dtype=torch.uint8, device=DEV)
    q[:, 3:227], s[:, 1:9] = r.q.view(torch.uint8), r.scale.view(torch.uint8)
    odd = features.Rows8(q[:, 3:227].view(E4M3), s[:, 1:9].view(torch.float8_e8m0fnu), 200)          # rows that start anywhere: copied
    assert torch.equal(features.unpack8(odd, torch.float32), want)
    assert torch.equal(features.unpack8(features.Rows8(r.q[2:5], r.scale[2:5], 200), torch.float32), want[2:5])
    for shape in ((0, 40), (3, 0), (0, 0)):
        e = features.pack8(torch.zeros(shape, device=DEV))
        assert e.shape == shape and features.unpack8(e).shape == shape


def test_more_elements_than_32_bits_count():
    from cuke_amd import features
    rows, cols = 70001, 65536 // 2 * 2                                       # 4.6e9 values
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.randn(cols, device=DEV)
    x[rows // 2, 7] = 3.25
    r = features.pack8(x)
    same_rows8(features.Rows8(r.q[-1:], r.scale[-1:], cols), x[-1:].double(), "last row")
    del x
    y = features.unpack8(r)
    assert y[rows // 2, 7] == 3.25 and int(torch.count_nonzero(y[:-1])) == 1
    assert torch.equal(y[-1:].float(), features.unpack8(features.Rows8(r.q[-1:], r.scale[-1:], cols), torch.float32))


# ---- norm ------------------------------------------------------------------------------------------
COLS = [1, 2, 7, 8, 31, 32, 33, 50, 96, 127, 128, 129, 256, 300, 400, 511, 512, 768, 1000, 1024, 1025, 1536, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 20000]


class Norm:
    def __init__(self, rows, cols, dtype, residual=True, weight=True, out=None, dy=None, layout="plain", seed=0, eps=1e-6):
        g = torch.Generator().manual_seed(seed + 31 * rows + cols)
        make = lambda *shape, scale=1.0, t=dtype: (torch.randn(shape, generator=g) * scale).to(DEV).to(t)
        self.eps, self.dtype, self.out = eps, dtype, out or dtype
        self.x = laid(make(rows, cols), layout)
        self.res = laid(make(rows, cols, scale=1.5), layout) if residual else None
        self.w = (1 + make(cols, scale=0.3, t=torch.float32)).to(dtype) if weight else None
        self.dy = laid(make(rows, cols, scale=0.1, t=dy or dtype), layout)
        self.dh = laid(make(rows, cols, scale=0.1), layout) if residual else None
        self.h = self.x.double() + (self.res.double() if residual else 0.0)
        self.r = (self.h.square().mean(1, keepdim=True) + eps).rsqrt()
        self.w64 = self.w.double() if weight else torch.ones(cols, dtype=torch.float64, device=DEV)
        self.y = self.h * self.r * self.w64

    def forward(self):
        from cuke_amd import features
        return features.rms_norm_forward(self.x, self.w, self.res, eps=self.eps, out_dtype=None if self.out == self.dtype else self.out)

    def check_forward(self, fw, what):
        if self.out == E4M3:
            same_rows8(fw.y, self.y, what)
        else:
            assert fw.y.dtype == self.out
            within(fw.y, self.y, (8 * EPS + U[self.out]) * self.y.abs() + TINY[self.out], (what, "y"))
        if self.res is not None:
            assert fw.h.dtype == self.dtype
            within(fw.h, self.h, (EPS + U[self.dtype]) * self.h.abs() + TINY[self.dtype], (what, "h"))
        within(fw.rstd[:, None], self.r, 2 * EPS * self.r, (what, "rstd"))

    def check_backward(self, fw, grads, what):
        M, K = self.h.shape
        n = self.h * self.r                              # (of the sum itself: what h's rounding dropped is kept to a 32nd of a step, a 16th where it is a half)
        dy = self.dy.double()
        g = dy * self.w64
        mean = (g * n).mean(1, keepdim=True)
        dx = self.r * (g - n * mean)
        # h's own error: of 16-bit sums a 16th of a step (2 u |h|, or 2 TINY where the type's numbers are evenly spaced), else its rounding to 32 bits
        off = EPS * n.abs() + ((2 * U[self.dtype] * n.abs() + 2 * TINY[self.dtype] * self.r) / 16 if self.res is not None and self.dtype != torch.float32 else 0.0)
        tol = self.r * (8 * EPS * (g.abs() + (n * mean).abs()) + n.abs() * (K + 8) * EPS * (g * n).abs().mean(1, keepdim=True))
        tol = tol + self.r * (off * mean.abs() + (n.abs() + off) * (g.abs() * off).mean(1, keepdim=True))
        if self.dh is not None:
            dx = dx + self.dh.double()
            tol = tol + 2 * EPS * self.dh.double().abs()
        within(grads.x, dx, tol + U[self.dtype] * (dx.abs() + tol) + TINY[self.dtype], (what, "dx"))
        if self.w is not None:
            dw, tol = (dy * n).sum(0), (M + 8) * EPS * (dy * n).abs().sum(0) + (dy.abs() * off).sum(0)
            within(grads.weight, dw, tol + U[self.dtype] * (dw.abs() + tol) + TINY[self.dtype], (what, "dweight"))
        else:
            assert grads.weight is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["same", "e4m3"])
def test_norm_of_every_width(dtype, kind):
    from cuke_amd import features
    for i, cols in enumerate(COLS):
        for rows in (1, 5, 67):
            c = Norm(rows, cols, dtype, residual=i % 2 == 0, weight=i % 3 != 2, out=E4M3 if kind == "e4m3" else None, layout=("plain", "apart")[i % 2])
            fw = c.forward()
            c.check_forward(fw, (rows, cols))
            c.check_backward(fw, features.rms_norm_backward(fw, c.dy, c.dh), (rows, cols))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES + [E4M3])
@pytest.mark.parametrize("dy", TYPES)
def test_norm_types(dtype, out, dy):
    from cuke_amd import features
    for rows, cols, residual, weight in ((70, 520, True, True), (9, 77, False, False), (3, 3000, True, True), (2, 9001, True, True)):
        c = Norm(rows, cols, dtype, residual, weight, out, dy)
        fw = c.forward()
        c.check_forward(fw, (rows, cols))
        c.check_backward(fw, features.rms_norm_backward(fw, c.dy, c.dh), (rows, cols))


def test_norm_of_many_rows():
    from cuke_amd import features
    for dtype, rows, cols, out in ((torch.bfloat16, 20011, 256, E4M3), (torch.float32, 5003, 48, None), (torch.float16, 1500, 2500, E4M3), (torch.bfloat16, 300, 10000, None)):
        c = Norm(rows, cols, dtype, out=out)
        fw = c.forward()
        c.check_forward(fw, (rows, cols))
        g = features.rms_norm_backward(fw, c.dy, c.dh)
        c.check_backward(fw, g, (rows, cols))
        again = features.rms_norm_backward(fw, c.dy, c.dh)
        assert torch.equal(g.x, again.x) and torch.equal(g.weight, again.weight)           # sums in a fixed order


def test_norm_gradients_against_differences():
    """d/dt of sum(dy y) along a direction, in 64 bits, by differences of the formula itself."""
    from cuke_amd import features
    c = Norm(6, 90, torch.float32)
    fw = c.forward()
    g = features.rms_norm_backward(fw, c.dy, c.dh)
    gen = torch.Generator().manual_seed(9)
    vx, vw = torch.randn(c.h.shape, generator=gen, dtype=torch.float64).to(DEV), torch.randn(90, generator=gen, dtype=torch.float64).to(DEV)

    def value(t):
        h, w = c.h + t * vx, c.w64 + t * vw
        return float((c.dy.double() * (h * (h.square().mean(1, keepdim=True) + c.eps).rsqrt() * w)).sum() + (c.dh.double() * h).sum())
    t = 1e-4
    slope = (value(t) - value(-t)) / (2 * t)                                       # off by t^2 times a third derivative: some 1e-7
    got = float((g.x.double() * vx).sum() + (g.weight.double() * vw).sum())
    scale = float((g.x.double() * vx).abs().sum() + (g.weight.double() * vw).abs().sum())
    assert abs(got - slope) <= 1e-6 * scale


def test_norm_of_unusual_rows():
    from cuke_amd import features
    inf, nan = float("inf"), float("nan")
    for cols in (40, 3000, 9000):
        x = torch.ones((6, cols), device=DEV)
        x[0] = 0                                 # y is 0: eps keeps r finite
        x[1, 3], x[2, 5] = inf, nan              # inf: r = 0, so that the others are 0 and it is NaN
        x[3] *= 3e38                             # squares overflow 32 bits
        x[4] *= 1e-38
        x[4, 0] = 1e-44
        y = features.rms_norm(x, eps=0.0 if cols == 40 else 1e-12)
        assert torch.isnan(y[1, 3]) and int(torch.isnan(y[1]).sum()) == 1 and bool((y[1][~torch.isnan(y[1])] == 0).all())
        assert bool(torch.isnan(y[2]).all())
        assert bool(((y[3] - 1).abs() < 1e-6).all()) and bool((y[5] == 1).all() if cols == 40 else ((y[5] - 1).abs() < 1e-6).all())
        if cols == 40:
            assert bool(torch.isnan(y[0]).all())                            # 0 / 0, as the formula says
        else:
            assert bool((y[0] == 0).all()) and bool((y[4].abs() < 1e-30).all())
        r = features.rms_norm(x, eps=1e-12, out_dtype=E4M3)
        q = r.q.float()[:, :cols]
        assert bool(torch.isnan(q[2]).all()) and int(torch.isnan(q[1]).sum()) == 1 and bool((q[0] == 0).all()) and bool((q[3] == 256).all())
        assert not torch.isnan(r.scale.float()).any()
    fw = features.rms_norm_forward(torch.zeros((0, 7), device=DEV), torch.ones(7, device=DEV))
    g = features.rms_norm_backward(fw, torch.zeros((0, 7), device=DEV))
    assert g.x.shape == (0, 7) and bool((g.weight == 0).all())
    assert features.rms_norm(torch.zeros((3, 0), device=DEV)).shape == (3, 0)


def test_norm_gradient_into_the_place_of_dy_or_dh():
    from cuke_amd import _lib, features
    L = _lib.lib()
    for cols in (64, 500, 5000, 9000):
        c = Norm(37, cols, torch.float32)
        fw = c.forward()
        want = features.rms_norm_backward(fw, c.dy, c.dh)
        d = _lib.RmsNorm(0, 0, 37, cols, None, 0, None, 0, c.w.data_ptr(), 0.0)
        n = L.kge_rms_norm_bwd_workspace(C.byref(d))
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        for place in ("dy", "dh"):
            t = {"dy": c.dy.clone(), "dh": c.dh.clone()}
            dw = torch.empty(cols, device=DEV)
            rc = L.kge_rms_norm_bwd(C.byref(d), fw.h.data_ptr(), cols, fw.rstd.data_ptr(), None, 0, t["dy"].data_ptr(), cols, t["dh"].data_ptr(), cols,
                                    t[place].data_ptr(), cols, dw.data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and torch.equal(t[place], want.x) and torch.equal(dw, want.weight), (cols, place)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_what_a_sum_loses_is_kept(dtype):
    """h and rest together are the sum to a 16th of a step, for all sizes of numbers; without rest the gradients are those of h."""
    from cuke_amd import _lib, features
    g = torch.Generator().manual_seed(4)
    for cols in (1, 5, 8, 100, 9001):
        size = torch.exp2(torch.randint(-30 if dtype == torch.float16 else -120, 12, (40, cols), generator=g).float())
        x, res = (torch.randn((40, cols), generator=g) * size).to(DEV).to(dtype), (torch.randn((40, cols), generator=g) * size * 1.7).to(DEV).to(dtype)
        fw = features.rms_norm_forward(x, None, res)
        assert fw.rest.shape == (40, -(-cols // 8))
        bits = (fw.rest.view(40, -1, 1) << torch.arange(28, -4, -4, device=DEV, dtype=torch.int32)) >> 28
        bits = bits.view(40, -1)[:, :cols].double()
        want = x.double() + res.double()
        step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -140)))) * 2 * U[dtype]
        if dtype == torch.float16:
            step = torch.exp2(torch.floor(torch.log2(fw.h.double().abs().clamp(min=2.0 ** -140)))) * 2 * U[dtype]
            step = step.clamp(min=2.0 ** -24)
            got = fw.h.double() + bits * step / 16
        else:
            got = (fw.h.float().view(torch.int32) + bits.int() * 4096).view(torch.float32).double()
        assert bool(((got - want).abs() <= step / 16 * 1.001 + EPS * want.abs() + 2.0 ** -130).all()), (dtype, cols)
    c = Norm(33, 70, dtype)
    fw = c.forward()
    fw.rest = None
    got = features.rms_norm_backward(fw, c.dy, c.dh)
    c.h, c.res = fw.h.double(), None                             # (r stays that of the sum)
    c.check_backward(fw, got, "rounded")


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_is_written_beside_rows(dtype):
    """Columns behind a row's end, rows behind the last one: left as they were, by every array of the C calls."""
    from cuke_amd import _lib, features
    L, st, code = _lib.lib(), torch.cuda.current_stream().cuda_stream, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    for rows, cols in ((5, 77), (3, 1027), (2, 9001), (4, 64)):
        c = Norm(rows, cols, dtype)
        want = features.rms_norm_forward(c.x, c.w, c.res)
        e = features.rms_norm(c.x, c.w, out_dtype=E4M3)
        canary = lambda r, n, t: torch.full((r, n), 0x5A, dtype=torch.uint8, device=DEV).view(t)
        size = c.x.element_size()
        y, h = canary(rows + 2, (cols + 9) * size, dtype), canary(rows + 2, (cols + 11) * size, dtype)
        rstd, rest = canary(1, 4 * (rows + 2), torch.float32), canary(rows + 2, 4 * (-(-cols // 8)), torch.int32)
        q, scale = canary(rows + 2, e.q.shape[1] + 32, torch.uint8), canary(rows + 2, e.scale.shape[1] + 8, torch.uint8)
        d = _lib.RmsNorm(code, code, rows, cols, c.x.data_ptr(), cols, c.res.data_ptr(), cols, c.w.data_ptr(), 1e-6)
        assert L.kge_rms_norm_fwd(C.byref(d), y.data_ptr(), cols + 9, None, h.data_ptr(), cols + 11, rstd.data_ptr(), rest.data_ptr(), st) == 0
        assert torch.equal(y[:rows, :cols], want.y) and torch.equal(h[:rows, :cols], want.h) and torch.equal(rstd[0, :rows], want.rstd)
        untouched = lambda t, keep: bool((t.view(torch.uint8)[keep(t.view(torch.uint8))] == 0x5A).all())

        def beside(width):
            def keep(t):
                m = torch.ones_like(t, dtype=torch.bool)
                m[:rows, :width] = False
                return m
            return keep
        assert untouched(y, beside(cols * size)) and untouched(h, beside(cols * size)) and bool((rstd[0, rows:].view(torch.uint8) == 0x5A).all())
        assert untouched(rest, beside(rest.shape[1] * 4 if dtype != torch.float32 else 0))
        r8 = _lib.Rows8(q.data_ptr(), q.shape[1], scale.data_ptr(), scale.shape[1])
        for call in ("norm", "pack"):
            q.fill_(0x5A), scale.fill_(0x5A)
            if call == "norm":
                d = _lib.RmsNorm(code, _lib.E4M3, rows, cols, c.x.data_ptr(), cols, None, 0, c.w.data_ptr(), 1e-6)
                assert L.kge_rms_norm_fwd(C.byref(d), None, 0, C.byref(r8), None, 0, None, None, st) == 0
                same = e
            else:
                assert L.kge_pack8(code, c.x.data_ptr(), cols, rows, cols, C.byref(r8), st) == 0
                same = features.pack8(c.x)
            assert torch.equal(q[:rows, :e.q.shape[1]], same.q.view(torch.uint8)) and torch.equal(scale[:rows, :e.scale.shape[1]], same.scale.view(torch.uint8))
            assert untouched(q, beside(e.q.shape[1])) and untouched(scale, beside(e.scale.shape[1]))
        assert L.kge_unpack8(C.byref(r8), rows, cols, code, y.fill_(7).data_ptr(), cols + 9, st) == 0
        assert torch.equal(y[:rows, :cols], features.unpack8(features.pack8(c.x), dtype)) and bool((y[rows:] == 7).all()) and bool((y[:, cols:] == 7).all())
        g = features.rms_norm_backward(want, c.dy, c.dh)
        d = _lib.RmsNorm(code, code, rows, cols, None, 0, None, 0, c.w.data_ptr(), 0.0)
        n = L.kge_rms_norm_bwd_workspace(C.byref(d))
        ws, dw = canary(1, n + 64, torch.uint8), canary(1, (cols + 5) * size, dtype)
        y.fill_(7)
        assert L.kge_rms_norm_bwd(C.byref(d), want.h.data_ptr(), cols, want.rstd.data_ptr(), want.rest.data_ptr() if want.rest is not None else None, code, c.dy.data_ptr(), cols,
                                  c.dh.data_ptr(), cols, y.data_ptr(), cols + 9, dw.data_ptr(), ws.data_ptr(), n, st) == 0
        assert torch.equal(y[:rows, :cols], g.x) and bool((y[rows:] == 7).all()) and bool((y[:, cols:] == 7).all())
        assert torch.equal(dw[0, :cols], g.weight) and bool((dw.view(torch.uint8)[0, cols * size:] == 0x5A).all()) and bool((ws[0, n:] == 0x5A).all())


def test_norm_refuses():
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    x, w = torch.zeros((4, 8), device=DEV), torch.ones(8, device=DEV)
    for call, error in ((lambda: features.rms_norm(x.double()), TypeError), (lambda: features.rms_norm(x, w.half()), TypeError),
                        (lambda: features.rms_norm(x, w[:7]), ValueError), (lambda: features.rms_norm(x, w, x.half()), TypeError),
                        (lambda: features.rms_norm(x, w, x[:3]), ValueError), (lambda: features.rms_norm(x, eps=-1.0), ValueError),
                        (lambda: features.rms_norm(x, eps=float("nan")), ValueError), (lambda: features.rms_norm(x, out_dtype=torch.int8), TypeError),
                        (lambda: features.rms_norm(x[0]), ValueError), (lambda: features.rms_norm(x.cpu()), KgeError), (lambda: features.rms_norm(None), TypeError),
                        (lambda: features.rms_norm_backward(x, x), TypeError), (lambda: features.pack8(x.int()), TypeError),
                        (lambda: features.unpack8(features.pack8(x), torch.int32), TypeError), (lambda: features.pack8([1.0]), TypeError)):
        with pytest.raises(error):
            call()
    fw = features.rms_norm_forward(x, w, x)
    for dy, dh, error in ((x[:3], None, ValueError), (x.int(), None, TypeError), (x, x.half(), TypeError), (x, x[:, :7], ValueError)):
        with pytest.raises(error):
            features.rms_norm_backward(fw, dy, dh)
    fw = features.rms_norm_forward(x.bfloat16(), w.bfloat16(), x.bfloat16())
    for name, bad, error in (("rest", fw.rest[:3], ValueError), ("rest", fw.rest.float(), TypeError), ("rstd", fw.rstd[:3], ValueError),
                             ("rstd", fw.rstd.double(), TypeError), ("rest", fw.rest.cpu(), KgeError), ("weight", fw.weight[:7], ValueError), ("h", fw.h[:, :7], ValueError)):
        with pytest.raises(error):
            features.rms_norm_backward(dataclasses.replace(fw, **{name: bad}), x)


def test_on_another_stream_and_in_a_graph():
    from cuke_amd import features
    c = Norm(130, 600, torch.bfloat16, out=E4M3)
    want = c.forward()
    want_g = features.rms_norm_backward(want, c.dy, c.dh)
    back = features.unpack8(want.y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fw = c.forward()
        g = features.rms_norm_backward(fw, c.dy, c.dh)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(fw.y.q.view(torch.uint8), want.y.q.view(torch.uint8)) and torch.equal(g.x, want_g.x) and torch.equal(g.weight, want_g.weight)
    x, res, dy = c.x.clone(), c.res.clone(), c.dy.clone()
    c.x, c.res, c.dy = x, res, dy
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fw = c.forward()
        g = features.rms_norm_backward(fw, c.dy, c.dh)
        y = features.unpack8(fw.y)
        again = features.pack8(y)
    for turn in range(3):
        x.copy_(c.dy * (turn + 1)), torch.cuda.synchronize()
        eager = c.forward()
        eager_g = features.rms_norm_backward(eager, c.dy, c.dh)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(fw.y.q.view(torch.uint8), eager.y.q.view(torch.uint8)) and torch.equal(fw.y.scale.view(torch.uint8), eager.y.scale.view(torch.uint8))
        assert torch.equal(g.x, eager_g.x) and torch.equal(g.weight, eager_g.weight)
        assert torch.equal(y, features.unpack8(eager.y)) and torch.equal(features.unpack8(again), y)
    assert not torch.equal(back, y)


def far(rows, cols, dtype, stride):
    """Rows `stride` elements apart, in memory that nobody has written."""
    base = torch.empty((rows - 1) * stride + cols, dtype=dtype, device=DEV)
    return base.as_strided((rows, cols), (stride, 1))


@pytest.mark.parametrize("cols", [40, 1027, 9000])
def test_rows_that_lie_more_than_32_bits_apart(cols):
    from cuke_amd import features
    c = Norm(5, cols, torch.bfloat16, out=E4M3)
    want = c.forward()
    want_g = features.rms_norm_backward(want, c.dy, c.dh)
    for name in ("x", "res", "dy", "dh"):
        t = far(5, cols, torch.bfloat16, 3 << 28)                # (the last row begins 6 GiB from the first)
        t.copy_(getattr(c, name))
        setattr(c, name, t)
    fw = c.forward()
    g = features.rms_norm_backward(fw, c.dy, c.dh)
    assert torch.equal(fw.y.q.view(torch.uint8), want.y.q.view(torch.uint8)) and torch.equal(fw.h, want.h)
    assert torch.equal(g.x, want_g.x) and torch.equal(g.weight, want_g.weight)
    q = far(5, want.y.q.shape[1], torch.uint8, 3 << 29)
    scale = far(5, want.y.scale.shape[1], torch.uint8, 3 << 28)
    q.copy_(want.y.q.view(torch.uint8)), scale.copy_(want.y.scale.view(torch.uint8))
    r = features.Rows8(q.view(E4M3), scale.view(torch.float8_e8m0fnu), cols)
    assert torch.equal(features.unpack8(r), features.unpack8(want.y))
