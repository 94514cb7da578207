"""The operators of deeper encoders, as cases that can be timed and compared.

Four operators, named by a case's ``op``:

  norm    rows plus a residual through a root-mean-square norm, to rows of a type or of 8 bits; ``train`` adds the gradients
  rows8   rows packed to 8 bits (e4m3, a power of two for each 32 columns), and back
  layer   a training pass of a linear layer that keeps its input in 8 bits, and the derivative of its activation too
  answer  a linear layer whose rows and weight are both in 8 bits

``own`` picks the framework's kernels; without it the same values come from elementary torch operations in 32 bits (in 64 where a value is rounded
to 8 bits next to a border).  Features and rows are N(0, 1), weights N(0, 1 / in); everything is drawn on the GPU from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6


def _norm(name, rows, cols, dtype, out="same", residual=True, weight=True, train=False):
    c = dict(op="norm", rows=rows, cols=cols, dtype=dtype, out=out, residual=residual, weight=weight, train=train)
    return dict(c, name=name) if name else c


def _rows8(name, rows, cols, dtype):
    c = dict(op="rows8", rows=rows, cols=cols, dtype=dtype)
    return dict(c, name=name) if name else c


def _layer(name, rows, fin, fout, dtype, act, drop=0.0, bias=True, residual=False, out="same", given="rows"):
    c = dict(op="layer", rows=rows, fin=fin, fout=fout, dtype=dtype, act=act, drop=drop, bias=bias, residual=residual, out=out, given=given)
    return dict(c, name=name) if name else c


def _answer(name, rows, fin, fout, dtype, act, bias=True, residual=False, out="same"):
    c = dict(op="answer", rows=rows, fin=fin, fout=fout, dtype=dtype, act=act, bias=bias, residual=residual, out=out)
    return dict(c, name=name) if name else c


def listed():
    return [
        # A query names one entity: its row on the way into an 8-bit layer.  Latency.
        _norm("norm_1x1024_bf16_e4m3", 1, 1024, "bf16", out="e4m3"),
        # A small batch of fp32 rows of the benchmark's width, normed for a layer in bf16.
        _norm("norm_train_512x400_f32_bf16", 512, 400, "f32", out="bf16", residual=False, train=True),
        # The usual batch: the residual added, the layer's input made in 8 bits and kept like that.
        _norm("norm_train_4096x1024_bf16_e4m3", 4096, 1024, "bf16", out="e4m3", train=True),
        # A large batch and its negatives, wide rows, everything in bf16.
        _norm("norm_train_65536x2048_bf16", 65536, 2048, "bf16", train=True),
        # A few rows of word vectors: odd sizes, fp32.
        _rows8("rows8_37x300_f32", 37, 300, "f32"),
        # The activations of a large batch, kept for the backward pass and brought back.
        _rows8("rows8_65536x1000_bf16", 65536, 1000, "bf16"),
        # The distinct entities of a small batch, trained in half precision.
        _layer("layer_512x768x400_f16", 512, 768, 400, "f16", "silu", drop=0.1),
        # The usual batch behind a norm that has made 8-bit rows already.
        _layer("layer_4096x1024x512_bf16_given8", 4096, 1024, 512, "bf16", "gelu", drop=0.1, given="rows8"),
        # The largest: wide features, wide rows, a large batch.
        _layer("layer_32768x2048x2048_bf16", 32768, 2048, 2048, "bf16", "gelu", drop=0.1),
        # One new entity is encoded for a query: latency.
        _answer("answer_1x1024x512_bf16", 1, 1024, 512, "bf16", "gelu"),
        # Re-encoding a table after training: onto fp32 rows of the benchmark's width 400.
        _answer("answer_65536x512x400_f32", 65536, 512, 400, "bf16", "none", residual=True, out="f32"),
        # The same of wide rows.
        _answer("answer_32768x2048x2048_bf16", 32768, 2048, 2048, "bf16", "gelu"),
    ]


# ---- drawn cases -----------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    d = _log(rng, lo, hi)
    return max(lo, d // 8 * 8) if rng.random() < 0.6 else d


def draw(rng):
    op = rng.choice(["norm", "norm", "rows8", "layer", "layer", "answer"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        while True:
            c = _norm(None, _log(rng, 1, 65536), _width(rng, 1, 8192), dtype, out=rng.choice(["same", "e4m3"] + (["bf16"] if dtype == "f32" else [])),
                      residual=rng.random() < 0.6, weight=rng.random() < 0.8, train=rng.random() < 0.6)
            if c["rows"] * c["cols"] <= 65536 * 2048 // (2 if dtype == "f32" else 1):
                return c
    if op == "rows8":
        while True:
            c = _rows8(None, _log(rng, 1, 65536), _log(rng, 1, 4096), dtype)
            if c["rows"] * c["cols"] <= 65536 * 1000:
                return c
    dtype = rng.choice(["bf16", "f16"])
    while True:
        act = rng.choice(["none", "gelu", "silu", "relu"])
        more = dict(bias=rng.random() < 0.8, residual=rng.random() < 0.5, out="f32" if rng.random() < 0.3 else "same")
        if op == "layer":
            c = _layer(None, _log(rng, 16, 65536), _width(rng, 32, 2048), _width(rng, 32, 2048), dtype, act, drop=rng.choice([0.0, 0.1, 0.3]),
                       given=rng.choice(["rows", "rows8"]), **more)
        else:
            c = _answer(None, _log(rng, 1, 65536), _width(rng, 32, 4096), _width(rng, 32, 2048), dtype, act, **more)
        if c["rows"] * c["fin"] * c["fout"] <= 32768 * 2048 * 2048:
            return c


# ---- 8 bits ----------------------------------------------------------------------------------------
def _blocks(x):
    """Rows as blocks of 32 columns, zeros behind the last one."""
    rows, cols = x.shape
    n = (cols + 31) // 32
    return torch.nn.functional.pad(x, (0, 32 * n - cols)).view(rows, n, 32)


def _exponents(blocks):
    """The least k with amax <= 448 2^k of every block (-127 of one that is all zero)."""
    top = blocks.abs().amax(2)
    m, e = torch.frexp(top)
    k = (e - 9 + (m > 0.875).int()).clamp(min=-127)
    return torch.where(top == 0, torch.full_like(k, -127), k)


def _power(k, dtype):
    """2^k from the bits of the number (pow is a bit off for some k, and bf16 values lie on borders of e4m3 often)."""
    k = k.long()
    return ((k + 127) << 23).int().view(torch.float32) if dtype == torch.float32 else ((k + 1023) << 52).view(torch.float64)


def _pack(x):
    """(q, scale) of rows of 32 or 64 bits: e4m3 [rows, 32 n] and e8m0 [rows, 4 ceil(n / 4)]."""
    blocks = _blocks(x)
    k = _exponents(blocks)
    v = blocks * _power(-k, x.dtype).unsqueeze(2)
    if x.dtype == torch.float64:  # (to e4m3 in one rounding: the conversion goes through 32 bits)
        step = torch.frexp(v)[1].clamp(min=-5) - 4
        v = torch.round(v * _power(-step, x.dtype)) * _power(step, x.dtype)
    rows, n = k.shape
    scale = torch.nn.functional.pad((k + 127).to(torch.uint8), (0, -n % 4))
    return v.float().to(E4M3).view(rows, 32 * n), scale.view(E8M0)


def _unpack(q, scale, cols):
    rows, n = q.shape[0], q.shape[1] // 32
    return (q.float().view(rows, n, 32) * scale[:, :n].float().unsqueeze(2)).view(rows, 32 * n)[:, :cols]


def _shown(q, scale, cols):
    """What rows in 8 bits hold, without what is behind their end: tensors of types whose elements stand for their values."""
    return {"q": q[:, :cols], "scale": scale[:, :(cols + 31) // 32]}


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
    if case["op"] == "norm":
        M, N = case["rows"], case["cols"]
        s.x = normal(M, N)
        s.res = normal(M, N, scale=1.5) if case["residual"] else None
        s.w = (1.0 + normal(N, scale=0.2, dtype=torch.float32)).to(dt) if case["weight"] else None
        if case["train"]:
            s.dy = normal(M, N, scale=0.1, dtype=dt if case["out"] in ("same", "e4m3") else DTYPES[case["out"]])
            s.dh = normal(M, N, scale=0.1) if case["residual"] else None
        return s
    if case["op"] == "rows8":
        s.x = normal(case["rows"], case["cols"])
        # rows of another size each, as gradients and activations of different entities have, and a feature in 64 that stands out
        s.x *= torch.exp(2.0 * torch.randn((case["rows"], 1), generator=g, device=_dev())).to(dt)
        s.x[:, 17::64] *= 12.0
        return s
    M, K, N = case["rows"], case["fin"], case["fout"]
    s.x, s.w = normal(M, K), normal(N, K, scale=K ** -0.5)
    s.b = normal(N, scale=0.1) if case["bias"] else None
    s.out = torch.float32 if case["out"] == "f32" else dt
    s.res = normal(M, N, scale=0.5, dtype=s.out) if case["residual"] else None
    if case["op"] == "layer":
        s.dy = normal(M, N, scale=0.1, dtype=s.out)
        if case["given"] == "rows8":
            s.x = _pack(s.x.float())
    else:
        s.x, s.w = _pack(s.x.float()), _pack(s.w.float())
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


def _plain_norm(s):
    c = s.case
    t = torch.float64 if c["out"] == "e4m3" else torch.float32
    h = s.x.to(t)
    if s.res is not None:
        h = h + s.res.to(t)
    r = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * r
    if s.w is not None:
        y = y * s.w.to(t)
    dt = s.x.dtype
    out = _shown(*_pack(y), c["cols"]) if c["out"] == "e4m3" else {"y": y.to(dt if c["out"] == "same" else DTYPES[c["out"]])}
    if s.res is not None:
        out["h"] = h.to(dt)
    if c["train"]:
        h, r, dy = h.float(), r.float(), s.dy.float()
        g = dy if s.w is None else dy * s.w.float()
        dx = r * (g - h * (r * r) * (g * h).mean(1, keepdim=True))
        if s.dh is not None:
            dx = dx + s.dh.float()
        out["dx"] = dx.to(dt)
        if s.w is not None:
            out["dw"] = (dy * h * r).sum(0).to(dt)
    return out


def _plain_layer(s):
    c = s.case
    q, scale = s.x if c["given"] == "rows8" else _pack(s.x.float())
    x, w = _unpack(q, scale, c["fin"]), s.w.float()
    z = x @ w.t()
    if s.b is not None:
        z = z + s.b.float()
    a, slope = _act(z, c["act"])
    y = _drop(a, c["drop"], s.seed, s.step)
    if s.res is not None:
        y = y + s.res.float()
    if c["act"] != "none":  # the derivative as it is kept: 8 bits of fixed point
        slope = (torch.round(slope * 200.0 + 27.0) - 27.0) / 200.0
    dz = _drop(s.dy.float(), c["drop"], s.seed, s.step) * slope
    dt = s.w.dtype
    out = {"y": y.to(s.out), "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(dt)}
    if s.b is not None:
        out["db"] = dz.sum(0).to(dt)
    return out


def _plain_answer(s):
    c = s.case
    z = _unpack(*s.x, c["fin"]) @ _unpack(*s.w, c["fin"]).t()
    if s.b is not None:
        z = z + s.b.float()
    y = _act(z, c["act"])[0]
    if s.res is not None:
        y = y + s.res.float()
    return {"y": y.to(s.out)}


# ---- one pass --------------------------------------------------------------------------------------
def run(s):
    c = s.case
    if c["op"] == "norm":
        if not own:
            return _plain_norm(s)
        from cuke_amd import features
        dt = {"same": None, "e4m3": E4M3}.get(c["out"], DTYPES.get(c["out"]))
        if not c["train"]:
            y = features.rms_norm(s.x, s.w, s.res, eps=EPS, out_dtype=dt)
            y, h = y if s.res is not None else (y, None)
        else:
            fw = features.rms_norm_forward(s.x, s.w, s.res, eps=EPS, out_dtype=dt)
            g = features.rms_norm_backward(fw, s.dy, s.dh)
            y, h = fw.y, fw.h
        out = _shown(y.q, y.scale, c["cols"]) if c["out"] == "e4m3" else {"y": y}
        if s.res is not None:
            out["h"] = h
        if c["train"]:
            out["dx"] = g.x
            if s.w is not None:
                out["dw"] = g.weight
        return out
    if c["op"] == "rows8":
        if not own:
            q, scale = _pack(s.x.float())
            return {**_shown(q, scale, c["cols"]), "y": _unpack(q, scale, c["cols"]).to(s.x.dtype)}
        from cuke_amd import features
        r = features.pack8(s.x)
        return {**_shown(r.q, r.scale, c["cols"]), "y": features.unpack8(r, s.x.dtype)}
    if c["op"] == "layer":
        if not own:
            return _plain_layer(s)
        from cuke_amd import features
        r = features.Rows8(*s.x, c["fin"]) if c["given"] == "rows8" else features.pack8(s.x)
        fw = features.linear_forward(r, s.w, s.b, act=c["act"], drop=c["drop"], seed=s.seed, step=s.step, residual=s.res, out_dtype=s.out)
        g = features.linear_backward(fw, s.dy)
        out = {"y": fw.y, "dx": g.x, "dw": g.weight}
        if s.b is not None:
            out["db"] = g.bias
        return out
    if not own:
        return _plain_answer(s)
    from cuke_amd import features
    x, w = features.Rows8(*s.x, c["fin"]), features.Rows8(*s.w, c["fin"])
    return {"y": features.linear(x, w, s.b, act=c["act"], residual=s.res, out_dtype=s.out, dtype=DTYPES[c["dtype"]])}


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    eighth = 1.0 + 1.0 / 32  # bytes of a value in 8 bits
    if case["op"] == "norm":
        n = float(case["rows"]) * case["cols"]
        out = {"same": size, "e4m3": eighth, "bf16": 2}[case["out"]]
        b = n * (size * (3 if case["residual"] else 1) + out)
        if case["train"]:
            # (without a residual x is read once for both passes)
            b += n * ((size if case["out"] in ("same", "e4m3") else out) + size + (size if case["residual"] else 0))
        return {"bytes": b + (2 * size if case["train"] else size) * case["cols"] * case["weight"], "flops": n * (18 if case["train"] else 6)}
    if case["op"] == "rows8":
        n = float(case["rows"]) * case["cols"]
        return {"bytes": n * (2 * size + eighth), "flops": 3.0 * n}
    M, K, N = case["rows"], case["fin"], case["fout"]
    out = 4 if case["out"] == "f32" else size
    ends = out * M * N * (2 if case["residual"] else 1) + (size * N if case["bias"] else 0)
    if case["op"] == "answer":
        return {"bytes": ends + eighth * K * (M + N), "flops": 2.0 * M * N * K}
    b = ends + (size if case["given"] == "rows" else eighth) * M * K + size * N * K
    b += out * M * N + size * (M * K + N * K + (N if case["bias"] else 0))
    return {"bytes": float(b), "flops": 6.0 * M * N * K}


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


def _eight64(x):
    """The values (in units of the scale), the scales and the values that rows of 64 bits stand for in 8 bits, from the list of all e4m3 numbers."""
    M, K = x.shape
    n = -(-K // 32)
    full = torch.zeros((M, 32 * n), dtype=torch.float64, device=x.device)
    full[:, :K] = x
    cells = full.reshape(M * n, 32)
    top = cells.abs().max(dim=1, keepdim=True).values
    unit = torch.full_like(top, 2.0 ** -127)
    powers = torch.tensor([2.0 ** k for k in range(-127, 128)], dtype=torch.float64, device=x.device)
    at = torch.searchsorted(448.0 * powers, top.flatten())     # the first unit that is large enough
    unit = powers[at].reshape(-1, 1)
    numbers = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    numbers = torch.tensor(numbers, dtype=torch.float64, device=x.device)
    middle = (numbers[1:] + numbers[:-1]) / 2
    size = cells.abs() / unit
    low, high = torch.bucketize(size, middle), torch.bucketize(size, middle, right=True)   # they differ at a tie: the even one of the two
    pick = torch.where(low == high, low, torch.where(low % 2 == 0, low, high))
    q = numbers[pick] * torch.sign(cells)
    return q.reshape(M, -1)[:, :K], unit.reshape(M, n), (q * unit).reshape(M, -1)[:, :K]


def _given64(pair, cols):
    """Rows in 8 bits as they were given, in 64 bits."""
    q, scale = pair
    unit = torch.exp2(scale.view(torch.uint8).to(torch.float64) - 127.0)
    return (q.to(torch.float64) * unit.repeat_interleave(32, dim=1)[:, :q.shape[1]])[:, :cols]


def _act64(z, act):
    if act == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if act == "gelu":
        half = torch.special.ndtr(z)
        return z * half, half + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        sg = torch.special.expit(z)
        return z * sg, sg + z * sg * torch.special.expit(-z)
    return z, None


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "rows8":
        q, scale, y = _eight64(s.x.to(f64))
        return {"q": q, "scale": scale, "y": y}
    if case["op"] == "norm":
        h = s.x.to(f64)
        if s.res is not None:
            h = torch.add(h, s.res.to(f64))
        w = torch.ones(case["cols"], dtype=f64, device=h.device) if s.w is None else s.w.to(f64)
        size = torch.sqrt(torch.linalg.vector_norm(h, dim=1).square() / case["cols"] + EPS).unsqueeze(1)
        unit = h / size
        y = unit * w
        out = {}
        if case["out"] == "e4m3":
            out["q"], out["scale"], _ = _eight64(y)
        else:
            out["y"] = y
        if s.res is not None:
            out["h"] = h
        if case["train"]:
            dy = s.dy.to(f64)
            g = dy * w
            dx = (g - unit * (g * unit).mean(dim=1, keepdim=True)) / size
            out["dx"] = dx if s.dh is None else dx + s.dh.to(f64)
            if s.w is not None:
                out["dw"] = torch.sum(dy * unit, dim=0)
        return out
    if case["op"] == "answer":
        z = torch.matmul(_given64(s.x, case["fin"]), _given64(s.w, case["fin"]).T)
        if s.b is not None:
            z += s.b.to(f64)
        y = _act64(z, case["act"])[0]
        return {"y": y if s.res is None else y + s.res.to(f64)}
    k = _kept64(case["rows"], case["fout"], case["drop"], s.seed, s.step)
    x = _given64(s.x, case["fin"]) if case["given"] == "rows8" else _eight64(s.x.to(f64))[2]
    w = s.w.to(f64)
    z = torch.matmul(x, w.T)
    if s.b is not None:
        z += s.b.to(f64)
    y, slope = _act64(z, case["act"])
    if k is not None:
        y = y * k
    if s.res is not None:
        y = y + s.res.to(f64)
    dz = s.dy.to(f64)
    if k is not None:
        dz = dz * k
    if slope is not None:
        dz = dz * ((200 * slope + 27).round() - 27) / 200
    out = {"y": y, "dx": torch.matmul(dz, w), "dw": torch.matmul(dz.T.contiguous(), x)}
    if s.b is not None:
        out["db"] = torch.sum(dz, dim=0)
    return out
