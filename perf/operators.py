"""The operators of feature-encoded entity rows, as cases that can be timed and compared.

Three operators, named by a case's ``op``:

  linear      y = dropout(act(x W^T + b)) + residual: rows of features to rows of an entity table; ``train`` adds its gradients
  dropout     rows dropped by a counter-based generator, and the gradient through the same mask
  preference  a paired loss of positive and negative scores against a frozen reference's, with its gradients

``own`` picks the framework's kernels; without it the same values come from elementary torch operations in 32 bits.
Features are N(0, 1), weights N(0, 1 / in), scores N(0, 2) beside a reference that is near them; everything is drawn on the
GPU from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _linear(name, rows, fin, fout, dtype, act, drop=0.0, bias=True, residual=False, out="same", train=False):
    c = dict(op="linear", rows=rows, fin=fin, fout=fout, dtype=dtype, act=act, drop=drop, bias=bias, residual=residual, out=out,
             train=train)
    return dict(c, name=name) if name else c


def _dropout(name, rows, cols, dtype, p):
    c = dict(op="dropout", rows=rows, cols=cols, dtype=dtype, p=p)
    return dict(c, name=name) if name else c


def _preference(name, rows, n_neg, dtype, kind="sigmoid", beta=0.5, ref=True, masked=False, temperature=0.0, smoothing=0.0,
                sign=1.0):
    c = dict(op="preference", rows=rows, n_neg=n_neg, dtype=dtype, kind=kind, beta=beta, ref=ref, masked=masked,
             temperature=temperature, smoothing=smoothing, sign=sign)
    return dict(c, name=name) if name else c


def listed():
    return [
        # A query names one entity that has features and no row yet: latency.
        _linear("linear_1x1024x512_bf16", 1, 1024, 512, "bf16", "gelu"),
        # A handful of new entities between two evaluations, in the tables' own type; their free rows are added.
        _linear("linear_37x300x200_f32", 37, 300, 200, "f32", "relu", residual=True),
        # The distinct entities of a small batch, trained in half precision.
        _linear("linear_train_512x768x400_f16", 512, 768, 400, "f16", "silu", drop=0.1, train=True),
        # The usual batch: its entities' text embeddings into hidden rows.
        _linear("linear_train_4096x1024x512_bf16", 4096, 1024, 512, "bf16", "gelu", drop=0.1, train=True),
        # Every entity of a benchmark graph (14951), word vectors of 300 into rows of 200, everything in fp32.
        _linear("linear_train_14951x300x200_f32", 14951, 300, 200, "f32", "silu", drop=0.2, residual=True, train=True),
        # Re-encoding a table after training: hidden rows in bf16 onto fp32 rows of the benchmark's width 400.
        _linear("linear_65536x512x400_bf16_f32", 65536, 512, 400, "bf16", "none", residual=True, out="f32"),
        # The largest: wide features, wide rows, a large batch.
        _linear("linear_train_32768x2048x2048_bf16", 32768, 2048, 2048, "bf16", "gelu", drop=0.1, train=True),
        # A first experiment's rows (500 triples, width 50).
        _dropout("dropout_500x50_f32", 500, 50, "f32", 0.1),
        # The rows of a large batch and its negatives.
        _dropout("dropout_65536x1000_bf16", 65536, 1000, "bf16", 0.2),
        # Plain pairs: one rejected answer for every chosen one.
        _preference("preference_8192x1_f32", 8192, 1, "f32", beta=0.1),
        # The benchmark's largest batch of shared negatives: known positives masked, hard negatives weighted up.
        _preference("preference_16384x1024_f32", 16384, 1024, "f32", masked=True, temperature=1.0),
        # A few queries against every entity of a benchmark graph.
        _preference("preference_64x40943_bf16", 64, 40943, "bf16", masked=True, smoothing=0.1),
    ]


# ---- drawn cases -----------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    d = _log(rng, lo, hi)
    return max(lo, d // 8 * 8) if rng.random() < 0.6 else d


def draw(rng):
    op = rng.choice(["linear", "linear", "dropout", "preference"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "linear":
        while True:
            train = rng.random() < 0.6
            c = _linear(None, _log(rng, 16 if train else 1, 65536), _width(rng, 32, 2048), _width(rng, 32, 2048), dtype,
                        # (relu's derivative jumps: in fp32 the last bit of one sum would decide over a whole row's gradient)
                        rng.choice(["none", "gelu", "silu"] + ([] if train and dtype == "f32" else ["relu"])), drop=rng.choice([0.0, 0.1, 0.3]) if train else 0.0,
                        bias=rng.random() < 0.8, residual=rng.random() < 0.5,
                        out="f32" if dtype != "f32" and rng.random() < 0.3 else "same", train=train)
            most = 2.0 * 32768 * 2048 * 2048 * (0.25 if dtype == "f32" else 1.0)
            if 2.0 * c["rows"] * c["fin"] * c["fout"] <= most:
                return c
    if op == "dropout":
        while True:
            c = _dropout(None, _log(rng, 1, 65536), _log(rng, 1, 4096), dtype, rng.choice([0.05, 0.1, 0.2, 0.5]))
            if c["rows"] * c["cols"] <= 65536 * 1000:
                return c
    while True:
        kind = rng.choice(["sigmoid", "sigmoid", "hinge", "square"])
        c = _preference(None, _log(rng, 1, 262144), _log(rng, 1, 65536), dtype, kind, beta=rng.choice([0.1, 0.5, 1.0]),
                        ref=rng.random() < 0.7, masked=rng.random() < 0.5, temperature=rng.choice([0.0, 0.0, 0.5, 1.0]),
                        smoothing=rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0, sign=rng.choice([1.0, -1.0]))
        if c["rows"] * c["n_neg"] <= 16384 * 1024:
            return c


# ---- inputs ----------------------------------------------------------------------------------------
def _dev():
    return torch.device("cuda:0")


class _State:
    pass


def prepare(case, seed):
    g = torch.Generator(device=_dev())
    g.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(shape, generator=g, device=_dev(), dtype=torch.float32).mul_(scale).to(dtype)

    s = _State()
    s.case = case
    s.seed, s.step = int(seed) * 7919 + 17, int(seed) % 1000 + 3
    if case["op"] == "linear":
        M, K, N = case["rows"], case["fin"], case["fout"]
        s.x, s.w = normal(M, K), normal(N, K, scale=K ** -0.5)
        s.b = normal(N, scale=0.1) if case["bias"] else None
        s.out = torch.float32 if case["out"] == "f32" else dt
        s.res = normal(M, N, scale=0.5, dtype=s.out) if case["residual"] else None
        s.dy = normal(M, N, scale=0.1, dtype=s.out) if case["train"] else None
    elif case["op"] == "dropout":
        s.x, s.dy = normal(case["rows"], case["cols"]), normal(case["rows"], case["cols"], scale=0.1)
    else:
        B, N = case["rows"], case["n_neg"]
        pos, neg = normal(B, scale=2.0, dtype=torch.float32), normal(B, N, scale=2.0, dtype=torch.float32)
        s.ref_pos = s.ref_neg = s.mask = None
        if case["ref"]:
            s.ref_pos = (pos + normal(B, dtype=torch.float32)).to(dt)
            s.ref_neg = (neg + normal(B, N, dtype=torch.float32)).to(dt)
        s.pos, s.neg = pos.to(dt), neg.to(dt)
        if case["masked"]:
            # a tenth of the pairs are known to be true; some rows have no negative left.  A filter leaves its mark there.
            s.mask = torch.rand((B, N), generator=g, device=_dev()) >= 0.1
            s.mask[96::97] = False
            s.neg[~s.mask] = torch.finfo(dt).min if int(seed) % 2 else float("-inf")
    return s


# ---- the plain forms -------------------------------------------------------------------------------
GOLDEN, MASK64 = 0x9E3779B97F4A7C15, (1 << 64) - 1


def _signed(v):
    return v - (1 << 64) if v >> 63 else v


def _mix(z):
    """splitmix64 of a Python integer."""
    z = (z + GOLDEN) & MASK64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK64
    return z ^ (z >> 31)


def _mix_all(z):
    """The same of 64-bit integers in a tensor, whose products wrap as unsigned ones do."""
    z = z + _signed(GOLDEN)
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * _signed(0x94D049BB133111EB)
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _drop(v, p, seed, step):
    """v with its dropped elements zero and the others scaled up: four elements of a row share 64 random bits."""
    t = round(p * 65536)
    if t == 0:
        return v
    rows, cols = v.shape
    base = _mix(_mix((seed & MASK64) ^ 0xD1B54A32D192ED03) ^ (step & MASK64))
    quads = (cols + 3) // 4
    q = torch.arange(rows * quads, device=v.device, dtype=torch.int64)
    z = _mix_all((q * _signed(GOLDEN)) ^ _signed(base)).view(rows, quads, 1)
    bits = (z >> torch.tensor([0, 16, 32, 48], device=v.device)) & 0xFFFF
    keep = bits.view(rows, quads * 4)[:, :cols] >= t
    return torch.where(keep, v * (65536.0 / (65536 - t) if t < 65536 else 0.0), torch.zeros_like(v))


def _act(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        on = z > 0
        return torch.where(on, z, torch.zeros_like(z)), on.to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    return z, torch.ones_like(z)


def _plain_linear(s):
    c = s.case
    x, w = s.x.float(), s.w.float()
    z = x @ w.t()
    if s.b is not None:
        z = z + s.b.float()
    a, slope = _act(z, c["act"])
    y = _drop(a, c["drop"], s.seed, s.step)
    if s.res is not None:
        y = y + s.res.float()
    out = {"y": y.to(s.out)}
    if c["train"]:
        dz = _drop(s.dy.float(), c["drop"], s.seed, s.step) * slope
        out["dx"], out["dw"] = (dz @ w).to(s.x.dtype), (dz.t() @ x).to(s.x.dtype)
        if s.b is not None:
            out["db"] = dz.sum(0).to(s.x.dtype)
    return out


def _plain_preference(s):
    c = s.case
    neg = s.neg.float()
    on = torch.ones_like(neg, dtype=torch.bool) if s.mask is None else s.mask
    zero = torch.zeros_like(neg)
    neg = torch.where(on, neg, zero)
    B = neg.shape[0]
    p, n = s.pos.float(), neg
    if s.ref_pos is not None:
        p, n = p - s.ref_pos.float(), torch.where(on, n - s.ref_neg.float(), zero)
    d = c["sign"] * (p[:, None] - n)
    if c["kind"] == "sigmoid":
        z = c["beta"] * d
        e = torch.exp(-z.abs())
        soft = torch.log1p(e)              # softplus(-|z|)
        sig = torch.where(z > 0, e, torch.ones_like(e)) / (1.0 + e)       # sigma(-z)
        f = (1.0 - c["smoothing"]) * (soft + (-z).clamp(min=0)) + c["smoothing"] * (soft + z.clamp(min=0))
        df = c["beta"] * (c["smoothing"] - sig)
    elif c["kind"] == "hinge":
        z = c["beta"] * d
        f = (1.0 - z).clamp(min=0)
        df = torch.where(z < 1.0, torch.full_like(z, -c["beta"]), zero)
    else:
        f = (d - 0.5 / c["beta"]) ** 2
        df = 2.0 * (d - 0.5 / c["beta"])
    t = torch.where(on, c["temperature"] * c["sign"] * neg, torch.full_like(neg, -math.inf))
    top = t.max(1, keepdim=True).values
    e = torch.where(on, torch.exp(t - torch.where(top == -math.inf, torch.zeros_like(top), top)), zero)
    a = e / e.sum(1, keepdim=True).clamp(min=1e-30)
    loss = torch.where(on, a * f, zero).sum(1).sum() / B
    slope = torch.where(on, a * df, zero) * (c["sign"] / B)
    return {"loss": loss.view(1), "dpos": slope.sum(1), "dneg": -slope}


# ---- one pass --------------------------------------------------------------------------------------
def run(s):
    c = s.case
    if c["op"] == "linear":
        if not own:
            return _plain_linear(s)
        from cuke_amd import features
        if not c["train"]:
            return {"y": features.linear(s.x, s.w, s.b, act=c["act"], residual=s.res, out_dtype=s.out)}
        fw = features.linear_forward(s.x, s.w, s.b, act=c["act"], drop=c["drop"], seed=s.seed, step=s.step, residual=s.res,
                                     out_dtype=s.out)
        g = features.linear_backward(fw, s.dy)
        out = {"y": fw.y, "dx": g.x, "dw": g.weight}
        if s.b is not None:
            out["db"] = g.bias
        return out
    if c["op"] == "dropout":
        if not own:
            return {"y": _drop(s.x.float(), c["p"], s.seed, s.step).to(s.x.dtype),
                    "dx": _drop(s.dy.float(), c["p"], s.seed, s.step).to(s.x.dtype)}
        from cuke_amd import features
        return {"y": features.dropout(s.x, c["p"], s.seed, s.step), "dx": features.dropout_backward(s.dy, c["p"], s.seed, s.step)}
    if not own:
        return _plain_preference(s)
    from cuke_amd import features
    loss, dpos, dneg = features.preference_loss(s.pos, s.neg, s.ref_pos, s.ref_neg, beta=c["beta"], kind=c["kind"], mask=s.mask,
                                                temperature=c["temperature"], smoothing=c["smoothing"], sign=c["sign"])
    return {"loss": loss, "dpos": dpos, "dneg": dneg}


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "linear":
        M, K, N = case["rows"], case["fin"], case["fout"]
        out = 4 if case["out"] == "f32" else size
        b = size * (M * K + N * K + (N if case["bias"] else 0)) + out * M * N * (2 if case["residual"] else 1)
        if case["train"]:
            b += out * M * N + size * (M * K + N * K + (N if case["bias"] else 0))
        return {"bytes": float(b), "flops": (6.0 if case["train"] else 2.0) * M * N * K}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4.0 * size * n, "flops": 2.0 * n}
    n = float(case["rows"]) * case["n_neg"]
    side = 2 if case["ref"] else 1
    per_row = side * size + 4
    return {"bytes": n * (side * size + 4 + (1 if case["masked"] else 0)) + case["rows"] * per_row, "flops": n * (12 + (4 if case["temperature"] else 0))}


# ---- 64 bits ---------------------------------------------------------------------------------------
def _kept64(rows, cols, p, seed, step):
    """What every element is multiplied by, from the generator's definition in unsigned 64-bit arithmetic on the host."""
    cut = int(round(p * 65536))
    if cut == 0:
        return None

    def scramble(v):
        v = v + np.uint64(0x9E3779B97F4A7C15)
        v = (v ^ (v >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        v = (v ^ (v >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return v ^ (v >> np.uint64(31))

    with np.errstate(over="ignore"):
        start = scramble(np.array([seed % (1 << 64)], dtype=np.uint64) ^ np.uint64(0xD1B54A32D192ED03))
        start = scramble(start ^ np.uint64(step))
        per_row = -(-cols // 4)
        words = scramble(start ^ (np.arange(rows * per_row, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)))
    lots = words.view("<u2").reshape(rows, 4 * per_row)[:, :cols]      # 16 bits each, the lowest first
    return torch.from_numpy((lots >= cut).astype(np.float64) * (65536.0 / (65536 - cut))).to(_dev())


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "dropout":
        k = _kept64(case["rows"], case["cols"], case["p"], s.seed, s.step)
        return {"y": s.x.to(f64) * k, "dx": s.dy.to(f64) * k}
    if case["op"] == "linear":
        k = _kept64(case["rows"], case["fout"], case["drop"], s.seed, s.step)
        x, w = s.x.to(f64), s.w.to(f64)
        z = torch.matmul(x, w.T)
        if s.b is not None:
            z += s.b.to(f64)
        if case["act"] == "relu":
            y, slope = z.clamp(min=0.0), (z > 0).to(f64)
        elif case["act"] == "gelu":
            half = torch.special.ndtr(z)
            y, slope = z * half, half + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        elif case["act"] == "silu":
            sg = torch.special.expit(z)
            y, slope = z * sg, sg + z * sg * torch.special.expit(-z)
        else:
            y, slope = z, None
        if k is not None:
            y = y * k
        if s.res is not None:
            y = y + s.res.to(f64)
        out = {"y": y}
        if case["train"]:
            dz = s.dy.to(f64)
            if k is not None:
                dz = dz * k
            if slope is not None:
                dz = dz * slope
            out["dx"], out["dw"] = torch.matmul(dz, w), torch.matmul(dz.T.contiguous(), x)
            if s.b is not None:
                out["db"] = torch.sum(dz, dim=0)
        return out
    B, sg, beta, eps = case["rows"], case["sign"], case["beta"], case["smoothing"]
    pos, neg = s.pos.to(f64), s.neg.to(f64)
    gone = torch.zeros(neg.shape, dtype=torch.bool, device=neg.device) if s.mask is None else ~s.mask
    neg = neg.masked_fill(gone, 0.0)
    gap = sg * (pos.unsqueeze(1) - neg)
    if s.ref_pos is not None:
        gap = gap - sg * (s.ref_pos.to(f64).unsqueeze(1) - s.ref_neg.to(f64).masked_fill(gone, 0.0))
    if case["kind"] == "sigmoid":
        value = -(1 - eps) * torch.nn.functional.logsigmoid(beta * gap) - eps * torch.nn.functional.logsigmoid(-beta * gap)
        rise = beta * (eps - torch.sigmoid(-beta * gap))
    elif case["kind"] == "hinge":
        value = torch.relu(1 - beta * gap)
        rise = -beta * (beta * gap < 1).to(f64)
    else:
        value = (gap - 1 / (2 * beta)).square()
        rise = 2 * gap - 1 / beta
    share = torch.softmax((case["temperature"] * sg * neg).masked_fill(gone, -math.inf), dim=1).nan_to_num(0.0).masked_fill(gone, 0.0)
    back = sg * share * rise / B
    return {"loss": (share * value).sum().reshape(1) / B, "dpos": back.sum(1), "dneg": -back}
