"""Linear layers, dropout and the preference loss where values, sizes or memory are at the edge of what they take.

Tolerances as in test_gpu_features.py, element by element (EPS = 2^-24), from the roundings a result goes through; infinities and NaN have to stand
where the formulas in 64 bits have them.  There a pair without a share adds nothing, also where its own loss is infinite.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, LEAST = 2.0 ** -24, 2.0 ** -126         # (LEAST: what is smaller may become zero)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda:0"


def draw(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(DEV).to(dtype)


def like(got, want, tol, what):
    """The same infinities and NaN, and finite values within tol."""
    got = got.double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[torch.isinf(got)], want[torch.isinf(want)]) and torch.equal(torch.isinf(got), torch.isinf(want)), what
    off = torch.isfinite(want) & ~((got - want).abs() <= tol.expand_as(want))
    if off.any():
        i = tuple(torch.nonzero(off)[0].tolist())
        raise AssertionError(f"{what}: {int(off.sum())} of {off.numel()} off, first at {i}: {got[i].item()} for {want[i].item()} +- {tol.expand_as(want)[i].item()}")


# ---- preference loss -------------------------------------------------------------------------------
def prefer64(pos, neg, rpos=None, rneg=None, *, beta=1.0, kind="sigmoid", smoothing=0.0, temperature=0.0, sign=1.0, mask=None):
    """(loss, dpos, dneg) and their tolerances."""
    pos, neg = pos.double(), neg.double()
    on = torch.ones_like(neg, dtype=torch.bool) if mask is None else mask.bool()
    zero = torch.zeros_like(neg)
    n = torch.where(on, neg, zero)
    rp = torch.zeros_like(pos) if rpos is None else rpos.double()
    rn = zero if rneg is None else torch.where(on, rneg.double(), zero)
    d = sign * ((pos - rp)[:, None] - (n - rn))
    z = beta * d
    # sizes of what is rounded; scores at the end of the range saturate, and what they come to is exact
    small = lambda v: torch.where(v.abs() < 1e4, v.abs(), torch.zeros_like(v))
    d_tol = 2 * EPS * (small(pos)[:, None] + small(n) + small(rp)[:, None] + small(rn))
    z_tol = beta * d_tol
    if kind == "sigmoid":
        part = lambda c, v: c * torch.where(v > 0, v + torch.log1p(torch.exp(-v)), torch.log1p(torch.exp(v))) if c else zero
        f = part(1 - smoothing, -z) + part(smoothing, z) + 0.0 * torch.where(torch.isnan(z), z, zero)
        s = beta * (smoothing - torch.sigmoid(-z))
        f_tol, s_tol = z_tol + 16 * EPS * (1 + small(z)), beta * (z_tol / 4 + 16 * EPS * (1 + small(z)))
    elif kind == "hinge":
        f, s = torch.clamp(1 - z, min=0), torch.where(z >= 1, zero, torch.where(z < 1, zero - beta, z))
        f_tol = z_tol + 8 * EPS * (1 + small(z))
        s_tol = torch.where((1 - z).abs() <= f_tol, beta, 2 * EPS * beta).to(z)
    else:
        f, s = (d - 0.5 / beta) ** 2, 2 * (d - 0.5 / beta)
        s_tol = 2 * d_tol + 8 * EPS * (small(d) + 0.5 / beta)
        f_tol = s_tol * small(s) + s_tol ** 2
    B, N = n.shape
    if temperature:
        u = torch.where(on, sign * n, zero - math.inf)
        top = u.amax(1, keepdim=True)
        t = temperature * (u - torch.where(top == -math.inf, torch.zeros_like(top), top))
        e = torch.where(on, torch.exp(t), zero)
    else:
        t, e = zero, on.double()
    total = e.sum(1, keepdim=True)
    a = torch.where(total == 0, zero, e / total)
    # a weight: the difference, its product and the exponential; the sum of N of them
    a_tol = a * (8 * EPS * (1 + torch.where(torch.isfinite(t), t.abs(), zero)) + (N + 16) * EPS) + LEAST * (a > 0)

    def times(w, v):
        return torch.where((w == 0) & torch.isinf(v) | ~on, zero, w * v)
    loss = times(a, f).sum() / B
    loss_tol = (times(a_tol, f.abs()) + a * f_tol + (N + 16) * EPS * times(a, f.abs())).nan_to_num(0, 0, 0).sum() / B + 2 * EPS * loss.abs()
    g = sign * times(a, s) / B
    g_tol = (times(a_tol, s.abs()) + a * s_tol) / B + 8 * EPS * g.abs() + LEAST * (a > 0)
    return loss.view(1), g.sum(1), -g, loss_tol.view(1), g_tol.sum(1) + (N + 16) * EPS * g.abs().sum(1), g_tol


def check_prefer(pos, neg, rpos=None, rneg=None, **kw):
    from cuke_amd import features
    loss, dpos, dneg = features.preference_loss(pos, neg, rpos, rneg, **kw)
    want = prefer64(pos, neg, rpos, rneg, **kw)
    like(loss, want[0], want[3], "loss")
    like(dpos, want[1], want[4], "dpos")
    like(dneg, want[2], want[5], "dneg")
    return loss, dpos, dneg


# one lane to a row and more, all quads a lane holds, and segments with and without a pass for the weights' sums
WIDTHS = [1, 7, 300, 700, 2051]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sigmoid_of_infinite_scores(n, sign, dtype):
    """-log sigma(infinity) is 0, whatever the factor of a term that is not there: filters leave infinite scores where there is no mask."""
    g = torch.Generator().manual_seed(n)
    pos, neg = draw(g, (6,), dtype, 2.0), draw(g, (6, n), dtype, 2.0)
    neg[1, n // 2] = neg[2, 0] = -sign * math.inf       # the better the lower they are: no loss, no gradient
    pos[4] = sign * math.inf
    for kw in (dict(sign=sign), dict(sign=sign, mask=torch.ones(6, n, device=DEV, dtype=torch.bool))):
        loss, dpos, dneg = check_prefer(pos, neg, beta=0.5, **kw)
        assert bool(torch.isfinite(loss)) and dneg[1, n // 2] == 0 and not dneg[4].any() and dpos[4] == 0
        # the other side: all weight on the flipped labels
        check_prefer(-pos, -neg, beta=0.5, smoothing=1.0, **kw)
        # labels that are not certain make the loss infinite, the gradient stays what sigma's limit makes it
        loss, _, dneg = check_prefer(pos, neg, beta=0.5, smoothing=0.25, **kw)
        assert loss.item() == math.inf and bool(torch.isfinite(dneg).all())
        # and a score on the wrong side
        loss, _, dneg = check_prefer(-pos, -neg, beta=0.5, **kw)
        assert loss.item() == math.inf and bool(torch.isfinite(dneg).all())


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "square"])
@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("where", ["pos", "neg", "ref_pos", "ref_neg"])
def test_preference_of_nan(n, where, kind):
    """A NaN that no mask excludes makes NaN of the loss, of its pair's (or row's) gradients and of no other's."""
    g = torch.Generator().manual_seed(n + 1)
    pos, neg, rpos, rneg = draw(g, (5,), torch.float32), draw(g, (5, n), torch.float32), draw(g, (5,), torch.float32), draw(g, (5, n), torch.float32)
    bad = {"pos": pos, "neg": neg, "ref_pos": rpos, "ref_neg": rneg}[where]
    row = where.endswith("pos")
    bad[3 if row else (3, n // 2)] = math.nan
    mask = torch.ones(5, n, device=DEV, dtype=torch.bool)
    mask[1, 0] = False
    for kw in (dict(), dict(mask=mask), dict(mask=mask, temperature=0.5)):
        loss, dpos, dneg = check_prefer(pos, neg, rpos, rneg, beta=0.7, kind=kind, **kw)
        assert bool(torch.isnan(loss)) and torch.isnan(dpos).nonzero().flatten().tolist() == [3]
        whole = row or (where == "neg" and "temperature" in kw)          # (its weight is part of every other's)
        assert int(torch.isnan(dneg).sum()) == (n if whole else 1) and bool(torch.isnan(dneg[3, n // 2]))


def lowest(dtype, infinite):
    return -math.inf if infinite else torch.finfo(dtype).min


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("infinite", [False, True])
@pytest.mark.parametrize("n,first,end", [(2, 1, 2), (7, 4, 7), (700, 256, 512), (2049, 2048, 2049), (4099, 2048, 4096), (4099, 4096, 4099), (6200, 0, 2048)])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge"])
def test_scores_that_take_no_share(n, first, end, infinite, dtype, kind):
    """A stretch of scores of the type's lowest value, or infinitely low, beside others: it takes no share of the softmax."""
    g = torch.Generator().manual_seed(n + first)
    for sign in (1.0, -1.0):
        pos, neg = draw(g, (4,), dtype, 2.0), draw(g, (4, n), dtype, 2.0)
        neg[:3, first:end] = sign * lowest(dtype, infinite)
        mask = torch.rand(4, n, generator=g).to(DEV) >= 0.2
        mask[:, 0 if first else end] = True                    # (something is left)
        mask[1, first:end - 1] = False                         # in a row of its own, the last of them alone
        for temperature in (0.5, 1.0, 30.0):
            for m in (None, mask):
                loss, dpos, dneg = check_prefer(pos, neg, beta=0.3, kind=kind, temperature=temperature, sign=sign, mask=m)
                assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dpos).all()) and not dneg[:3, first:end].any()
                assert bool(dpos.any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 6, 700, 4099])
def test_rows_of_nothing_but_lowest_scores(n, dtype):
    """Infinitely low: the row adds nothing, as one without a pair.  Of the lowest value: equal scores, that share evenly."""
    g = torch.Generator().manual_seed(n)
    pos, neg = draw(g, (4,), dtype, 2.0), draw(g, (4, n), dtype, 2.0)
    neg[1], neg[2] = -math.inf, torch.finfo(dtype).min
    for kind in ("sigmoid", "hinge"):
        loss, dpos, dneg = check_prefer(pos, neg, beta=0.3, kind=kind, temperature=1.0)
        assert bool(torch.isfinite(loss)) and not dneg[1:3].any() and not dpos[1:3].any()


@pytest.mark.parametrize("n", [16, 300, 2048 + 16])
def test_softmax_of_scores_far_from_zero(n):
    """The weights are those of the scores' differences, which fp32 holds exactly beside a common offset of a thousand."""
    g = torch.Generator().manual_seed(n)
    neg = (1000.0 + draw(g, (64, n), torch.float64, 2.0)).float()
    mask = torch.zeros(64, n, device=DEV, dtype=torch.bool)
    mask[:, -16:] = True                                        # few enough that sums of them add little
    pos = (1000.0 + draw(g, (64,), torch.float64, 2.0)).float()
    from cuke_amd import features
    _, _, dneg = features.preference_loss(pos, neg, temperature=1.0, mask=mask)
    p, v = pos.double(), neg[:, -16:].double()
    a = torch.softmax(v, 1)
    want = a * torch.sigmoid(v - p[:, None]) / 64
    top = v.amax(1, keepdim=True)
    # 16 + 16 roundings of the sum and around it; the exponents' own, and the sigmoid's: both differences are exact
    tol = want * (8 * EPS * (1 + (top - v)) + 32 * EPS + 16 * EPS * (1 + (v - p[:, None]).abs()))
    like(dneg[:, -16:], want, tol, "dneg")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 7, 700, 2051])
def test_pairs_without_a_share_add_nothing(n, dtype):
    """A pair whose weight is zero adds neither loss nor gradient, also where its own loss is infinite or passes fp32's range."""
    g = torch.Generator().manual_seed(n)
    pos, neg = draw(g, (4,), dtype, 2.0), draw(g, (4, n), dtype, 2.0)
    neg[1, n - 1], neg[2, n - 1] = torch.finfo(dtype).min, -math.inf
    for kw in (dict(kind="square", beta=0.5), dict(smoothing=0.1, beta=4.0), dict(smoothing=0.1, beta=0.5)):
        loss, dpos, dneg = check_prefer(pos, neg, temperature=1.0, **kw)
        assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dpos).all()) and not dneg[1:3, n - 1].any()
    if n > 2:                                               # a NaN there is none the less one
        rneg = torch.zeros_like(neg)
        rneg[1, n - 1] = math.nan
        loss, dpos, _ = check_prefer(pos, neg, torch.zeros_like(pos), rneg, temperature=1.0)
        assert bool(torch.isnan(loss)) and bool(torch.isnan(dpos[1]))


def test_rows_of_no_pairs_are_not_read():
    """With n_neg = 0 nothing is looked at: pos and neg may be NULL, and so may one of the references."""
    import ctypes as C
    from cuke_amd import _lib
    L = _lib.lib()
    for kind in range(3):
        loss, dpos = torch.full((1,), -7.0, device=DEV), torch.full((3000,), -7.0, device=DEV)
        d = _lib.Preference(0, kind, 3000, 0, None, None, 0, None, None, 0, None, 0, 1.0, 1.0, 0.0, 0.5)
        need = L.kge_preference_workspace(C.byref(d))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        assert L.kge_preference_loss(C.byref(d), loss.data_ptr(), dpos.data_ptr(), None, ws.data_ptr(), need,
                                     torch.cuda.current_stream().cuda_stream) == 0
        assert loss.item() == 0 and not dpos.any()


def test_a_step_on_another_device_is_refused(monkeypatch):
    """The kernels read the word of the step: it has to be on the device that they run on."""
    from cuke_amd import features
    from cuke_amd.kge import KgeError
    word = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert features._random(1, word)[2] is word
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(KgeError):
        features._random(1, word)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_into_the_other_columns_of_an_array(dtype):
    """Two column ranges of one array share no element: one may be dropped into the other."""
    from cuke_amd import features
    g = torch.Generator().manual_seed(6)
    for rows, cols, at in [(9, 8, 8), (64, 30, 37), (1, 5, 5), (300, 1, 2)]:
        both = draw(g, (rows, cols + at + 3), dtype)
        was = both.clone()
        for x, out, rest in [(both[:, :cols], both[:, at:at + cols], [slice(0, at), slice(at + cols, None)]),
                             (both[:, at:at + cols], both[:, :cols], [slice(cols, None)])]:
            both.copy_(was)
            want = features.dropout(x.clone(), 0.4, 3, 1)
            assert features.dropout(x, 0.4, 3, 1, out=out) is out and torch.equal(out, want)
            assert all(torch.equal(both[:, s], was[:, s]) for s in rest)
    rows = torch.zeros(12, 16, device=DEV, dtype=dtype)
    flat, nine = rows.view(-1), rows[:9]
    for x, out in [(nine[:, :8], nine[:, 7:15]), (nine[:, 7:15], nine[:, :8]), (rows[:8, 8:], flat[20:148].view(8, 16)[:, :8]),
                   (flat[:96].view(6, 16)[:, :9], flat[24:120].view(6, 16)[:, :9]), (nine[:, 4:12], flat[:72].view(9, 8))]:
        with pytest.raises(ValueError):
            features.dropout(x, 0.5, 1, out=out)


# ---- fp32 products as products of bf16 parts ---------------------------------------------------------
# (rows, in, out): large enough that forward pass and gradients are made in tiles, on both sides of the rules that choose them
PRODUCTS = [(2100, 72, 264), (2100, 136, 265), (2500, 520, 264), (851, 1968, 1016), (4090, 1021, 509), (8200, 520, 776)]


def operand(gen, shape, values):
    t = torch.randn(shape, generator=gen, dtype=torch.float64)
    if values == "one sign":
        t = t.abs() + 0.1
    if values == "spread":
        t = t * torch.exp2(torch.randint(-20, 21, shape, generator=gen).double())
    return t.float().to(DEV)


@pytest.mark.parametrize("values", ["normal", "one sign", "spread"])
@pytest.mark.parametrize("shape", PRODUCTS, ids=lambda s: "%dx%dx%d" % s)
def test_fp32_products_are_no_worse_than_fp32(shape, values):
    """The error's 2-norm over the result's, of y, dx and dW, against that of fp32 sums of K products.

    A chain of K fp32 additions leaves each partial sum off by a rounding of 2^-24 / sqrt(3) (root mean square) of it: of partial sums that grow as
    sqrt(k) that comes to 2^-24 sqrt(K / 6), of those of one sign to less.  The result's own rounding is 2^-24 / sqrt(3).  Three of the six products of
    parts, instead of all, leave 4e-6."""
    from cuke_amd import features
    rows, fin, fout = shape
    g = torch.Generator().manual_seed(fin)
    x, w, dy = operand(g, (rows, fin), values), operand(g, (fout, fin), values), operand(g, (rows, fout), values)
    fw = features.linear_forward(x, w)
    got = features.linear_backward(fw, dy)
    for have, want, k, what in [(fw.y, x.double() @ w.double().T, fin, "y"), (got.x, dy.double() @ w.double(), fout, "dx"),
                                (got.weight, dy.double().T.contiguous() @ x.double(), rows, "dw")]:
        error = ((have.double() - want).norm() / want.norm()).item()
        print(f"{what} {shape} {values}: {error:.2e} of {EPS * math.sqrt(k / 6 + 1 / 3):.2e}", flush=True)
        assert error <= EPS * math.sqrt(k / 6 + 1 / 3), (what, error)


def test_fp32_tiles_at_the_edge_of_the_range():
    """Values whose leading bf16 part rounds to infinity, sums near the largest number, and very small ones, in sizes whose sums are made in tiles."""
    from cuke_amd import features
    rows, fin, fout = 2100, 136, 264
    x = torch.full((rows, fin), 3.4e38, device=DEV)
    w = torch.zeros(fout, fin, device=DEV)
    w[:, 3], w[1, 4], w[2, 3], w[200, 135], w[263, 3] = 1.0, -1.0, 2.0, -0.5, -2.0
    fw = features.linear_forward(x, w)
    assert torch.equal(fw.y, (x.double() @ w.double().T).float())
    dy = torch.zeros(rows, fout, device=DEV)
    dy[7, 5], dy[8, 2], dy[2099, 263], dy[2099, 200] = 3.4e38, 3.4e38, -0.25, 3.3e38
    dy[7, 6] = 1e36                                              # (of x, dy[7, 5] 3.4e38 passes the range, of w it does not)
    got = features.linear_backward(fw, dy)
    assert torch.equal(got.x, (dy.double() @ w.double()).float())
    assert torch.equal(got.weight, (dy.double().T.contiguous() @ x.double()).float())
    small, tiny = torch.full((rows, fin), 1e-30, device=DEV), torch.full((fout, fin), 1e-3, device=DEV)
    y = features.linear(small, tiny)
    want = small.double() @ tiny.double().T
    assert bool(((y.double() - want).abs() <= (fin + 16) * EPS * want).all())
