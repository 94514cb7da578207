"""Linear layers on rows in 8 bits on the GPU against plain formulas in 64 bits.

Tolerances, element by element, from the roundings a result goes through (u: half a step of a type, eps = 2^-24):
  a sum of K exact products in fp32, in any order   (K + 16) eps sum |a_k b_k|     (16: bias, activation, scale, residual, each a few eps)
  the last rounding                                 u |result|
  a derivative kept in 8 bits                       none where 64 bits say which of two steps it is; a step (0.005) where z's error reaches the border between them
  dz in the layer's type                            u |dz|, carried through the products by sum |w|
  a bf16 product of two sides in 8 bits             the matrix cores sum eight neighbouring terms at a time and drop of each what lies below 2^-13 of the largest one's
                                                    power of two: 8 times 2^-13 times the largest |a b| of the eight, which is at most max |a| max |b|
"""
import ctypes as C
import math

import pytest
import torch

from test_gpu_features import DEV, EPS, TINY, U, act64, draw, kept, within

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn


def values(r):
    """What rows in 8 bits stand for, in 64 bits."""
    n = -(-r.cols // 32)
    unit = torch.exp2(r.scale.view(torch.uint8)[:, :n].double() - 127.0)
    return (r.q.double() * unit.repeat_interleave(32, 1))[:, :r.cols]


class Layer8:
    def __init__(self, rows, fin, fout, dtype, act="none", drop=0.0, bias=True, residual=False, out=None, seed=0, layout="plain", eight=False, spread=1.0):
        from cuke_amd import features
        g = torch.Generator().manual_seed(1000 * seed + rows + 7 * fin + 13 * fout)
        grid = act == "relu"
        self.out = out or dtype
        x = draw(g, (rows, fin), torch.float32, 1.0, grid)
        if spread != 1.0:   # blocks of many sizes
            x = x * torch.exp(spread * torch.randn((rows, -(-fin // 32)), generator=g)).to(DEV).repeat_interleave(32, 1)[:, :fin]
        self.x = features.pack8(x)
        self.w = draw(g, (fout, fin + (3 if layout == "apart" else 0)), dtype, 1.0 if grid else fin ** -0.5, grid)[:, :fin]
        if eight:
            self.w = features.pack8(self.w.float() * (torch.exp(spread * torch.randn((fout, 1), generator=g)).to(DEV) if spread != 1.0 else 1.0))
        self.b = draw(g, (fout,), dtype, 0.3, grid) if bias else None
        self.res = draw(g, (rows, fout), self.out, 0.5, grid) if residual else None
        self.dy = draw(g, (rows, fout + (3 if layout == "apart" else 0)), self.out, 0.5, grid)[:, :fout]
        self.dtype, self.act, self.drop, self.seed, self.step = dtype, act, drop, 77 + seed, 5
        x, w, dy = values(self.x), values(self.w) if eight else self.w.double(), self.dy.double()
        z = x @ w.T + (self.b.double() if bias else 0.0)
        size = x.abs() @ w.abs().T + (self.b.double().abs() if bias else 0.0)
        k = kept(rows, fout, drop, self.seed, self.step) if drop else torch.ones_like(z)
        a, slope = act64(z, act)
        self.y = a * k + (self.res.double() if residual else 0.0)
        inner = (fin + 16) * EPS * (size + 1.0)
        if eight and self.out == torch.bfloat16:
            most = lambda v: torch.nn.functional.pad(v.abs(), (0, -fin % 8)).view(v.shape[0], -1, 8).amax(2)
            inner = inner + 8 * 2.0 ** -13 * (most(x) @ most(w).T)
        self.y_tol = U[self.out] * self.y.abs() + TINY[self.out] + 1.2 * k * inner + 16 * EPS * (self.y.abs() + (self.res.double().abs() if residual else 0.0))
        slope_tol = torch.zeros_like(z)
        if act != "none":
            at = 200 * slope + 27
            slope_tol = torch.where((at - at.floor() - 0.5).abs() <= 200 * (1.2 * inner + 16 * EPS), 0.005, 0.0) * (act != "relu") + 4 * EPS
            slope = (at.round() - 27) / 200
        dz = dy * k * slope
        exact_dz = act == "none" and not drop and self.out == dtype
        dz_tol = torch.zeros_like(dz) if exact_dz else dy.abs() * k * (slope_tol + 8 * EPS)
        db_tol = dz_tol
        if not exact_dz:
            dz_tol = dz_tol + U[dtype] * (dz.abs() + dz_tol) + TINY[dtype]
        self.dx, self.dw, self.db = dz @ w, dz.T.contiguous() @ x, dz.sum(0)
        self.dx_tol = dz_tol @ w.abs() + (fout + 16) * EPS * (dz.abs() @ w.abs()) + U[dtype] * self.dx.abs() + TINY[dtype]
        self.dw_tol = dz_tol.T.contiguous() @ x.abs() + (rows + 16) * EPS * (dz.abs().T.contiguous() @ x.abs()) + U[dtype] * self.dw.abs() + TINY[dtype]
        self.db_tol = db_tol.sum(0) + (rows + 16) * EPS * dz.abs().sum(0) + U[dtype] * self.db.abs() + TINY[dtype]

    def kw(self):
        return dict(act=self.act, drop=self.drop, seed=self.seed, step=self.step, residual=self.res, out_dtype=self.out)

    def check(self):
        from cuke_amd import features
        y = features.linear(self.x, self.w, self.b, dtype=self.dtype, **self.kw())
        assert y.dtype == self.out
        within(y, self.y, self.y_tol, "y without a backward pass")
        if isinstance(self.w, features.Rows8):
            return
        fw = features.linear_forward(self.x, self.w, self.b, **self.kw())
        within(fw.y, self.y, self.y_tol, "y")
        fw.y = None                                                      # not needed any more
        g = features.linear_backward(fw, self.dy)
        within(g.x, self.dx, self.dx_tol, "dx")
        within(g.weight, self.dw, self.dw_tol, "dw")
        if self.b is None:
            assert g.bias is None
        else:
            within(g.bias, self.db, self.db_tol, "db")
        again = features.linear_backward(fw, self.dy)
        assert torch.equal(again.x, g.x) and torch.equal(again.weight, g.weight), "the same call gives the same bits"


SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 33), (2, 7, 5), (3, 129, 257), (16, 8, 16), (17, 40, 24), (31, 96, 130), (33, 33, 31), (63, 300, 200),
          (64, 32, 96), (65, 31, 129), (100, 50, 400), (127, 128, 128), (129, 256, 136), (200, 2048, 72), (257, 264, 520), (300, 17, 3),
          (1000, 24, 8), (1025, 72, 264)]
TILED = [(1100, 72, 264, {}), (2100, 130, 264, {}), (2100, 132, 265, dict(act="silu", drop=0.2)), (1537, 64, 400, dict(act="relu", residual=True)),
         (4000, 33, 150, dict(act="gelu")), (8200, 520, 776, {}), (8200, 520, 776, dict(act="gelu", drop=0.1, residual=True)),
         (8200, 521, 777, dict(act="silu", residual=True)), (16640, 264, 1030, {}), (16640, 264, 1030, dict(act="gelu", drop=0.1)),
         (33000, 64, 130, dict(act="gelu", residual=True)), (16300, 520, 1000, {}), (16300, 1100, 1000, dict(act="silu", drop=0.1, residual=True)),
         (5000, 72, 40, dict(act="gelu", drop=0.1)), (2500, 520, 264, dict(act="gelu", drop=0.1)), (4096, 256, 512, dict(act="gelu"))]
name = lambda c: "%dx%dx%d%s" % (c[0], c[1], c[2], "".join("-" + str(v) for v in c[3].values()))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, eight, dtype):
    print("layer", shape, eight, dtype, flush=True)
    Layer8(*shape, dtype, act="gelu", eight=eight).check()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
@pytest.mark.parametrize("shape", [(5, 200, 40), (70, 520, 130), (300, 130, 90), (2100, 300, 270)])
def test_blocks_of_many_sizes(shape, eight, dtype):
    """Every block has a power of its own: sums come out right only if each meets its own numbers."""
    print("blocks", shape, eight, dtype, flush=True)
    Layer8(*shape, dtype, eight=eight, spread=1.5).check()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("drop,bias,residual", [(0.0, False, False), (0.0, True, True), (0.3, True, False), (0.1, False, True)])
def test_epilogues(dtype, eight, act, drop, bias, residual):
    print("epilogue", dtype, eight, act, drop, bias, residual, flush=True)
    for out in (dtype, torch.float32):
        Layer8(70, 88, 150, dtype, act=act, drop=drop, bias=bias, residual=residual, out=out, eight=eight).check()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
@pytest.mark.parametrize("case", TILED, ids=name)
def test_tiles(case, eight, dtype):
    print("tiles", case, eight, dtype, flush=True)
    Layer8(*case[:3], dtype, eight=eight, **case[3]).check()
    if case[3].get("residual"):
        Layer8(*case[:3], dtype, out=torch.float32, eight=eight, **case[3]).check()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(40, 64, 72), (150, 130, 66), (5, 33, 31), (2100, 136, 270)])
def test_weights_and_gradients_that_start_anywhere(shape, dtype):
    print("layout", shape, dtype, flush=True)
    Layer8(*shape, dtype, act="silu", drop=0.2, residual=True, layout="apart").check()


def test_a_weight_whose_rows_share_a_channel():
    Layer8(8200, 2048, 1030, torch.bfloat16, act="gelu").check()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", [3, 200, 2100])
@pytest.mark.parametrize("eight", [False, True], ids=["w16", "w8"])
def test_nans_and_ends_of_the_range(rows, eight, dtype):
    """NaN reaches the rows and columns whose sums hold it and no others; the smallest and largest powers multiply as they should."""
    from cuke_amd import features
    g = torch.Generator().manual_seed(3)
    x, w = draw(g, (rows, 136), torch.float32), draw(g, (264, 136), dtype, 0.1)
    x[0, 5], x[1, 7] = float("inf"), float("nan")
    r = features.pack8(x)
    r.scale.view(torch.uint8)[2, 1] = 255                    # a block that is NaN
    fresh = lambda: features.pack8(w) if eight else w
    y = features.linear(r, fresh(), out_dtype=torch.float32, dtype=dtype)
    assert bool(torch.isnan(y[:3]).all()) and not torch.isnan(y[3:]).any()
    if not eight:
        fw = features.linear_forward(r, w)
        got = features.linear_backward(fw, torch.ones_like(fw.y))
        assert not torch.isnan(got.x).any()
        nan = torch.zeros(136, dtype=torch.bool, device=DEV)
        nan[5] = nan[7] = True
        nan[32:64] = True
        assert torch.equal(torch.isnan(got.weight), nan.expand_as(got.weight))
    # one number a row: powers from 2^-127 to 2^119 times a weight that brings the product back
    if dtype == torch.bfloat16:
        k = torch.arange(-118, 119, device=DEV)
        x = torch.zeros((len(k), 40), device=DEV)
        x[:, 33] = torch.exp2(k.float()) * 1.5
        w = torch.zeros((3, 40), device=DEV)
        w[1, 33], w[2, 33] = 2.0 ** 8, -2.0 ** -8
        y = features.linear(features.pack8(x), features.pack8(w) if eight else w.to(dtype), out_dtype=torch.float32, dtype=dtype).double()
        want = x[:, 33].double()
        assert bool((y[:, 0] == 0).all()) and torch.equal(y[:, 1], want * 256) and torch.equal(y[:, 2], -want / 256)


def test_derivatives_reach_their_ends():
    from cuke_amd import features
    for dtype in HALF:
        z = torch.tensor([-60000.0, -40.0, -6.0, -1.0, -0.75, 0.0, 1.0, 1.4375, 6.0, 40.0, 60000.0], device=DEV)
        r = features.pack8(z[:, None])
        for act in ("relu", "gelu", "silu"):
            fw = features.linear_forward(r, torch.ones(1, 1, device=DEV, dtype=dtype), act=act)
            g = features.linear_backward(fw, torch.ones_like(fw.y))
            v = values(r)
            s = act64(v, act)[1]
            within(g.x, s, 0.0025 + 4 * EPS + 2 * U[dtype] * s.abs() + torch.zeros_like(s), f"{act}' {dtype}")
            assert g.x[0].item() == 0 and g.x[-1].item() == 1
            x = torch.tensor([[float("nan")], [1.0]], device=DEV)
            fw = features.linear_forward(features.pack8(x), torch.ones(1, 1, device=DEV, dtype=dtype), act=act)
            got = features.linear_backward(fw, torch.ones_like(fw.y)).x
            assert torch.isnan(got[0, 0]) and not torch.isnan(got[1, 0])


@pytest.mark.parametrize("dtype", HALF)
def test_layers_of_nothing(dtype):
    from cuke_amd import features
    for rows, fin, fout in [(0, 8, 8), (5, 0, 8), (5, 8, 0), (0, 0, 0), (0, 8, 0), (2000, 0, 1000), (9000, 0, 800)]:
        x, w = features.pack8(torch.randn(rows, fin, device=DEV)), torch.randn(fout, fin, device=DEV).to(dtype)
        b = torch.randn(fout, device=DEV).to(dtype)
        want = torch.nn.functional.silu(b.double()).expand(rows, fout)
        for weight in (w, features.pack8(w)):
            y = features.linear(x, weight, b, act="silu")
            assert y.shape == (rows, fout) and (fin > 0 or torch.allclose(y.double(), want, rtol=2 * U[dtype], atol=1e-6))
        fw = features.linear_forward(x, w, b, act="silu")
        g = features.linear_backward(fw, torch.ones_like(fw.y))
        assert g.x.shape == (rows, fin) and g.weight.shape == (fout, fin) and g.bias.shape == (fout,)
        if rows == 0:
            assert not g.bias.any() and not g.weight.any()


@pytest.mark.parametrize("dtype", HALF)
def test_gradients_against_differences(dtype):
    """The slope of sum(y dy) along random directions of the weight and bias, by central differences of the 64-bit formula; the kept derivative may be a
    half step (0.0025) off the formula's."""
    from cuke_amd import features
    L = Layer8(37, 45, 52, dtype, act="gelu", drop=0.25, residual=True, seed=3)
    g = features.linear_backward(features.linear_forward(L.x, L.w, L.b, **L.kw()), L.dy)
    k = kept(37, 52, L.drop, L.seed, L.step)
    gen = torch.Generator().manual_seed(9)
    at = [values(L.x), L.w.double(), L.b.double()]
    total = lambda x, w, b: ((act64(x @ w.T + b, "gelu")[0] * k + L.res.double()) * L.dy.double()).sum()
    half = 0.0025 * L.dy.double().abs() * k
    more = [half @ at[1].abs(), half.T.contiguous() @ at[0].abs(), half.sum(0)]
    for i, (grad, tol) in enumerate([(g.x, L.dx_tol), (g.weight, L.dw_tol), (g.bias, L.db_tol)]):
        v = torch.randn(at[i].shape, generator=gen, dtype=torch.float64).to(DEV)
        h = 1e-4
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - h * v, at[i] + h * v
        slope = (total(*hi) - total(*lo)) / (2 * h)
        assert abs((grad.double() * v).sum() - slope) <= ((tol + more[i]) * v.abs()).sum() + 2e3 * h * h


def test_rows_behind_the_last_are_left_alone():
    from cuke_amd import _lib, features
    L = Layer8(70, 100, 90, torch.bfloat16, act="gelu")
    lib = _lib.lib()
    d = _lib.Linear(1, 1, 2, 0, 70, 100, 90, None, 0, L.w.data_ptr(), 100, L.b.data_ptr(), None, 0, 0.0, 0, 0, None)
    x8 = features._rows8_c(L.x)
    big = torch.full((80, 100), 7.0, dtype=torch.bfloat16, device=DEV)
    n = lib.kge_linear8_fwd_workspace(C.byref(d), None, 0)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    assert lib.kge_linear8_fwd(C.byref(d), C.byref(x8), None, big.data_ptr(), 100, 0, None, 0, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
    within(big[:70, :90], L.y, L.y_tol, "y")
    assert bool((big[70:] == 7).all()) and bool((big[:70, 90:] == 7).all())


@pytest.mark.parametrize("shape", [(100, 1000, 24), (40, 520, 264), (3, 96, 50)])
def test_rows_that_lie_far_apart(shape):
    """x in 8 bits with the most bytes between its rows that the backward pass takes (the last of a hundred begins 6 GiB from the first)."""
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    c = Layer8(*shape, torch.bfloat16, "gelu", drop=0.1)
    fw = features.linear_forward(c.x, c.w, c.b, **c.kw())
    g = features.linear_backward(fw, c.dy)

    def moved(stride):
        def one(t, unit):
            base = torch.empty((shape[0] - 1) * (stride - unit) + t.shape[1], dtype=torch.uint8, device=DEV)
            v = base.as_strided(t.shape, (stride - unit, 1))
            v.copy_(t.view(torch.uint8))
            return v.view(t.dtype)
        return features.Rows8(one(c.x.q, 16), one(c.x.scale, 4), c.x.cols)
    x = moved(1 << 26)
    again = features.linear_forward(x, c.w, c.b, **c.kw())
    got = features.linear_backward(again, c.dy)
    assert torch.equal(again.y, fw.y) and torch.equal(got.x, g.x) and torch.equal(got.weight, g.weight) and torch.equal(got.bias, g.bias)
    again = features.linear_forward(moved((1 << 26) + 16), c.w, c.b, **c.kw())
    assert torch.equal(again.y, fw.y)
    with pytest.raises(KgeError):
        features.linear_backward(again, c.dy)


@pytest.mark.parametrize("side", ["x", "w"])
def test_both_sides_in_8_bits_far_apart(side):
    """More bytes between rows than the largest tiles address with 32 bits."""
    from cuke_amd import features
    c = Layer8(8200 if side == "w" else 900, 520, 776 if side == "w" else 8200, torch.bfloat16, "gelu", eight=True)
    old = getattr(c, side)
    base = torch.empty((old.q.shape[0] - 1) * (1 << 24) + old.q.shape[1], dtype=torch.uint8, device=DEV)
    q = base.as_strided(old.q.shape, (1 << 24, 1))
    q.copy_(old.q.view(torch.uint8))
    setattr(c, side, features.Rows8(q.view(E4M3), old.scale, old.cols))
    within(features.linear(c.x, c.w, c.b, dtype=c.dtype, **c.kw()), c.y, c.y_tol, side)


def test_on_another_stream_and_in_two_graphs():
    from cuke_amd import features
    small, large = Layer8(300, 200, 136, torch.float16, "silu", drop=0.2, residual=True), Layer8(2100, 520, 264, torch.bfloat16, "gelu", drop=0.1, residual=True)

    def run(c):
        fw = features.linear_forward(c.x, c.w, c.b, **c.kw())
        g = features.linear_backward(fw, c.dy)
        return [fw.y, g.x, g.weight, g.bias, features.linear(c.x, features.pack8(c.w), c.b, dtype=c.dtype, **c.kw())]
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    want = [run(small), run(large)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, c in zip(streams, (small, large)):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(c))
    torch.cuda.synchronize()
    assert same(got[0], want[0]) and same(got[1], want[1])
    graphs, got = [], []
    for c in (small, large):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(c))
    for turn in range(3):
        for c in (small, large):
            c.dy.mul_(0.5)
        eager = [run(small), run(large)]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert same(got[0], eager[0]) and same(got[1], eager[1])


def test_refusals():
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    x, w, b = torch.randn(6, 40, device=DEV), torch.randn(8, 40, device=DEV).bfloat16(), torch.zeros(8, device=DEV).bfloat16()
    r, w8 = features.pack8(x), features.pack8(w)
    for call, error in ((lambda: features.linear(r, w.float()), TypeError), (lambda: features.linear(r, w[:, :39]), ValueError), (lambda: features.linear(r, w, b.half()), TypeError),
                        (lambda: features.linear(r, w, b[:7]), ValueError), (lambda: features.linear(r, w, out_dtype=torch.float16), TypeError),
                        (lambda: features.linear(r, w, dtype=torch.float16), TypeError), (lambda: features.linear(r, w8, dtype=torch.float32), TypeError),
                        (lambda: features.linear(r, w8, b, dtype=torch.float16), TypeError), (lambda: features.linear(x.bfloat16(), w8), TypeError),
                        (lambda: features.linear(x.bfloat16(), w, dtype=torch.float16), TypeError), (lambda: features.linear_forward(r, w8), TypeError),
                        (lambda: features.linear_forward(x.bfloat16(), w8), TypeError), (lambda: features.linear(r, w, act="tanh"), ValueError),
                        (lambda: features.linear(r, w, drop=1.5), ValueError), (lambda: features.linear(r, w, residual=x), ValueError),
                        (lambda: features.linear(r, w.cpu()), KgeError), (lambda: features.linear(features.Rows8(r.q.cpu(), r.scale.cpu(), 40), w), KgeError)):
        with pytest.raises(error):
            call()
    fw = features.linear_forward(r, w, b)
    for dy, error in ((torch.zeros(6, 7, device=DEV).bfloat16(), ValueError), (torch.zeros(6, 8, device=DEV), TypeError), (None, TypeError)):
        with pytest.raises(error):
            features.linear_backward(fw, dy)


# ---- all of them together --------------------------------------------------------------------------
def encoder(dtype, width=96, inner=200, dim=50, features_=60, blocks=3, drop=0.1, seed=0):
    from cuke_amd import features
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(DEV).to(dtype)
    one = lambda n: (1 + 0.2 * torch.randn(n, generator=g)).to(DEV).to(dtype)
    bl = [features.Block(one(width), mk(inner, width, scale=width ** -0.5), mk(inner, scale=0.1), mk(width, inner, scale=inner ** -0.5), mk(width, scale=0.1))
          for _ in range(blocks)]
    return features.ResidualEncoder(mk(width, features_, scale=features_ ** -0.5), mk(width, scale=0.1), bl, one(width), mk(dim, width, scale=width ** -0.5),
                                    mk(dim, scale=0.1), act="gelu", drop=drop, seed=seed)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("given8", [False, True])
def test_encoder_against_its_own_operators(dtype, given8):
    """The encoder's rows and gradients are those of its operators called one after another by hand."""
    from cuke_amd import features as f
    enc = encoder(dtype)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(301, 60, generator=g).to(DEV).to(dtype)
    x = f.pack8(x) if given8 else x
    base, drows = torch.randn(301, 50, generator=g).to(DEV), torch.randn(301, 50, generator=g).to(DEV)
    fw = enc.forward(x, base, step=4)
    h, more, kept_ = f.linear(x, enc.w_in, enc.b_in), None, []
    for i, b in enumerate(enc.blocks):
        n = f.rms_norm_forward(h, b.norm, out_dtype=E4M3) if more is None else f.rms_norm_forward(more, b.norm, h, out_dtype=E4M3)
        a = f.linear_forward(n.y, b.w1, b.b1, act="gelu", drop=0.1, seed=i, step=4)
        o = f.linear_forward(f.pack8(a.y), b.w2, b.b2)
        h, more = n.h, o.y
        kept_.append((n, a, o))
    n = f.rms_norm_forward(more, enc.norm, h, out_dtype=E4M3)
    last = f.linear_forward(n.y, enc.w_out, enc.b_out, residual=base, out_dtype=torch.float32)
    assert torch.equal(fw.rows, last.y) and fw.rows.dtype == torch.float32
    back = enc.backward(fw, drows, need_x=True)
    gl = f.linear_backward(last, drows)
    gn = f.rms_norm_backward(n, gl.x)
    assert torch.equal(back.last.weight, gl.weight) and torch.equal(back.norm, gn.weight) and back.base is drows
    d = gn.x
    for i in (2, 1, 0):
        n, a, o = kept_[i]
        go = f.linear_backward(o, d)
        ga = f.linear_backward(a, go.x)
        gn = f.rms_norm_backward(n, ga.x, d)
        b = back.blocks[i]
        assert torch.equal(b.norm, gn.weight) and torch.equal(b.w1, ga.weight) and torch.equal(b.b1, ga.bias) and torch.equal(b.w2, go.weight) and torch.equal(b.b2, go.bias)
        d = gn.x
    assert back.first.x.shape == (301, 60) and back.first.weight.shape == enc.w_in.shape


def test_encoder_without_blocks():
    from cuke_amd import features as f
    enc = encoder(torch.bfloat16)
    enc = f.ResidualEncoder(enc.w_in, enc.b_in, [], enc.norm, enc.w_out, enc.b_out)
    g = torch.Generator().manual_seed(6)
    x, drows = torch.randn(301, 60, generator=g).to(DEV).bfloat16(), torch.randn(301, 50, generator=g).to(DEV)
    fw = enc.forward(x)
    assert torch.equal(enc.encode(x), fw.rows)
    n = f.rms_norm_forward(f.linear(x, enc.w_in, enc.b_in), enc.norm, out_dtype=E4M3)
    last = f.linear_forward(n.y, enc.w_out, enc.b_out, out_dtype=torch.float32)
    back, gl = enc.backward(fw, drows), f.linear_backward(last, drows)
    assert torch.equal(last.y, fw.rows) and back.blocks == [] and torch.equal(back.last.weight, gl.weight)
    assert torch.equal(back.norm, f.rms_norm_backward(n, gl.x).weight) and enc.packed().encode(x).shape == (301, 50)


def test_encoder_against_64_bits():
    """Rows and gradients against the formula without any rounding: every layer's input is off by up to 2^-4 of itself, at random, so that what comes out is off by
    some hundredths in the root mean square: 2^-4 / sqrt(12) * 1.5 = 0.027 of a layer's output from each of its two 8-bit inputs' roundings, five layers deep and in
    quadrature 0.027 sqrt(5) = 0.06; gradients go through the forward rows' errors and 16-bit roundings: twice that."""
    enc = encoder(torch.bfloat16, drop=0.0, blocks=2)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(400, 60, generator=g).to(DEV).bfloat16()
    drows = torch.randn(400, 50, generator=g).to(DEV)
    leaves = []

    def leaf(t):
        leaves.append(t.double().clone().requires_grad_(True))
        return leaves[-1]
    norm = lambda h, w: h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * w
    h = x.double() @ leaf(enc.w_in).T + leaf(enc.b_in)
    for b in enc.blocks:
        u = torch.nn.functional.gelu(norm(h, leaf(b.norm)) @ leaf(b.w1).T + leaf(b.b1))
        h = h + u @ leaf(b.w2).T + leaf(b.b2)
    rows = norm(h, leaf(enc.norm)) @ leaf(enc.w_out).T + leaf(enc.b_out)
    want = torch.autograd.grad(rows, leaves, drows.double())
    fw = enc.forward(x)
    back = enc.backward(fw, drows)
    off = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert off(fw.rows, rows.detach()) < 0.06 and off(enc.encode(x), rows.detach()) < 0.06
    assert off(enc.packed().encode(x), rows.detach()) < 0.12                       # the weights are rounded too
    got = [back.first.weight, back.first.bias]
    for b in back.blocks:
        got += [b.norm, b.w1, b.b1, b.w2, b.b2]
    got += [back.norm, back.last.weight, back.last.bias]
    for i, (a, b) in enumerate(zip(got, want)):
        assert off(a, b) < 0.12, (i, off(a, b))


def test_encoder_answers_as_it_trains():
    enc = encoder(torch.float16, drop=0.0)
    g = torch.Generator().manual_seed(7)
    x, base = torch.randn(130, 60, generator=g).to(DEV).half(), torch.randn(130, 50, generator=g).to(DEV)
    assert torch.equal(enc.encode(x, base), enc.forward(x, base).rows)
    one = enc.encode(x[17:18], base[17:18])
    assert float((one - enc.encode(x, base)[17:18]).abs().max()) < 0.02            # (a few rows go another way through the sums)
    empty = encoder(torch.float16, blocks=0)
    assert empty.encode(x).shape == (130, 50) and empty.backward(empty.forward(x), base).blocks == []


def test_encoder_in_a_graph():
    enc = encoder(torch.bfloat16)
    g = torch.Generator().manual_seed(8)
    x, drows = torch.randn(200, 60, generator=g).to(DEV).bfloat16(), torch.randn(200, 50, generator=g).to(DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        enc.backward(enc.forward(x, step=step), drows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fw = enc.forward(x, step=step)
        back = enc.backward(fw, drows)
    seen = []
    for turn in range(3):
        x.copy_(torch.randn(200, 60, generator=g).to(DEV).bfloat16())
        step.fill_(turn + 3)
        torch.cuda.synchronize()
        eager = enc.forward(x, step=step)
        eager_back = enc.backward(eager, drows)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(fw.rows, eager.rows)
        for a, b in zip(back.blocks, eager_back.blocks):
            assert torch.equal(a.w1, b.w1) and torch.equal(a.w2, b.w2) and torch.equal(a.norm, b.norm)
        assert torch.equal(back.first.weight, eager_back.first.weight)
        seen.append(fw.rows.clone())
    assert not torch.equal(seen[0], seen[1])
