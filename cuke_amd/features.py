"""Entity rows made from features, and a loss against a frozen model.

The score functions of :mod:`cuke_amd.kge` look rows up.  The operators here stand in front of that lookup and behind the scores:

  linear / linear_forward / linear_backward   ``drop(act(x W^T + b)) + residual`` and its gradients
  dropout / dropout_backward                  rows dropped by a counter-based generator; no mask is kept
  preference_loss                             positive against negative scores, relative to a frozen reference's
  Rows8, pack8, unpack8                       rows in 8 bits, with a power of two for each 32 columns: what deeper encoders keep
  rms_norm / rms_norm_forward / rms_norm_backward   a residual's addition and the norm of the sum, to rows of a type or of 8 bits
  FeatureEncoder                              two linear layers that turn feature rows into entity rows
  ResidualEncoder                             blocks of a norm and two layers on a residual stream, whose inputs are all kept in 8 bits

Like the rest of the package they work on the current stream, allocate their outputs, give every gradient by an explicit call,
and raise where an argument is not what the kernels take: there is no fallback.  The ordinary call goes through csrc/host.cpp, what that does
not take through the code here, which converts or raises.  16-bit and fp32 tensors are taken as they are; one whose rows
are not contiguous is copied.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import KgeError

__all__ = ["linear", "linear_forward", "linear_backward", "LinearForward", "LinearGrads", "dropout", "dropout_backward",
           "preference_loss", "Rows8", "pack8", "unpack8", "rms_norm", "rms_norm_forward", "rms_norm_backward", "NormForward", "NormGrads",
           "FeatureEncoder", "EncoderForward", "EncoderGrads", "Block", "ResidualEncoder", "ResidualForward", "ResidualGrads"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # kge_type_t
_U64 = (1 << 64) - 1


def _stream() -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _tensor(x, name: str, ndim: int) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor (got {type(x).__name__})")
    if not x.is_cuda:
        raise KgeError(f"{name} must live on the GPU (got {x.device}); there is no CPU path")
    if x.device.index != torch.cuda.current_device():
        raise KgeError(f"{name} must live on the current device (got {x.device}, current is cuda:{torch.cuda.current_device()})")
    if x.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions (got {x.dim()})")
    return x


def _rows(x, name: str, dtype=None, ndim: int = 2, shape=None) -> torch.Tensor:
    """x with contiguous rows, whatever the stride between them."""
    x = _tensor(x, name, ndim)
    if dtype is None and x.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16 (got {x.dtype})")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {x.dtype})")
    if shape is not None and tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)} (got {tuple(x.shape)})")
    if ndim == 1:
        return x.contiguous()
    inner, outer = x.stride(1), x.stride(0)
    return x if (inner == 1 or x.shape[1] <= 1) and (outer >= x.shape[1] or x.shape[0] <= 1) else x.contiguous()


def _apart(x, out) -> bool:
    """Whether two blocks of equal rows are the very same one or do not overlap: as ranges of memory, or, with rows equally far apart, as ranges
    of columns."""
    if x.data_ptr() == out.data_ptr() and (x.stride() == out.stride() or x.shape[0] <= 1):
        return True
    ends = [(t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * _row_stride(t) + t.shape[1]) * t.element_size()) for t in (x, out)]
    if x.numel() == 0 or ends[0][1] <= ends[1][0] or ends[1][1] <= ends[0][0]:
        return True
    width, pitch = x.shape[1] * x.element_size(), _row_stride(x) * x.element_size()
    return _row_stride(out) == _row_stride(x) and width <= (out.data_ptr() - x.data_ptr()) % pitch <= pitch - width


def _row_stride(x: torch.Tensor) -> int:
    """Elements between rows (of a single row: its length, whatever torch says)."""
    return x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1])


def _random(seed, step):
    """(seed, step, device word or None) as the library takes them."""
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or not step.is_cuda or step.numel() != 1:
            raise TypeError("step must be an integer or one int64 on the GPU")
        if step.device.index != torch.cuda.current_device():
            raise KgeError(f"step must live on the current device (got {step.device}, current is cuda:{torch.cuda.current_device()})")
        return int(seed) & _U64, 0, step
    return int(seed) & _U64, int(step) & _U64, None


def _probability(p) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"the probability of a drop must lie in [0, 1] (got {p})")
    return p


def _p(t):
    return None if t is None else t.data_ptr()


def _bytes(n: int, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


# ---- linear layers ---------------------------------------------------------------------------------
@dataclass
class LinearForward:
    """A layer's output, and what its backward pass needs (x and weight have to stay as they are until then).  A layer on :class:`Rows8` does not need y: it may
    be set to None."""
    y: torch.Tensor
    desc: bytes     # a kge_linear
    saved: torch.Tensor | None
    tensors: tuple  # what desc points to: x, weight, bias, residual, step


@dataclass
class LinearGrads:
    """Gradients in the layer's type; that of the residual is the gradient of y itself."""
    x: torch.Tensor | None
    weight: torch.Tensor | None
    bias: torch.Tensor | None


def _describe(x, weight, bias, act, drop, seed, step, residual, out_dtype):
    x = _rows(x, "x")
    weight = _rows(weight, "weight", x.dtype)
    if weight.shape[1] != x.shape[1]:
        raise ValueError(f"weight must have as many columns as x (got {tuple(weight.shape)} for x {tuple(x.shape)})")
    rows, out = x.shape[0], weight.shape[0]
    if bias is not None:
        bias = _rows(bias, "bias", x.dtype, ndim=1, shape=(out,))
    if out_dtype is None:
        out_dtype = x.dtype if residual is None else residual.dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {x.dtype} or float32 (got {out_dtype})")
    if residual is not None:
        residual = _rows(residual, "residual", out_dtype, shape=(rows, out))
    seed, step, word = _random(seed, step)
    desc = _lib.Linear(_TYPES[x.dtype], _TYPES[out_dtype], _act(act), 0, rows, x.shape[1], out, _p(x), _row_stride(x),
                       _p(weight), _row_stride(weight), _p(bias), _p(residual), _row_stride(residual) if residual is not None else 0,
                       _probability(drop), seed, step, _p(word))
    return desc, (x, weight, bias, residual, word), out_dtype


def _linear_call(desc, tensors, out_dtype, for_backward):
    L, x = _lib.lib(), tensors[0]
    y = torch.empty((desc.rows, desc.out), dtype=out_dtype, device=x.device)
    saved_bytes = int(L.kge_linear_saved_bytes(C.byref(desc))) if for_backward else 0
    ws_bytes = int(L.kge_linear_fwd_workspace(C.byref(desc), int(for_backward)))
    saved, ws = _bytes(saved_bytes, x.device), _bytes(ws_bytes, x.device)
    _lib.check(L.kge_linear_fwd(C.byref(desc), _p(y), max(desc.out, 1), int(for_backward), _p(saved), saved_bytes, _p(ws), ws_bytes,
                                _stream()), "kge_linear_fwd")
    return y, saved


def _act(act) -> int:
    code = _lib.ACTS.get(act or "none")
    if code is None:
        raise ValueError(f"act must be one of {sorted(_lib.ACTS)} (got {act!r})")
    return code


def _describe8(x, weight, bias, act, drop, seed, step, residual, out_dtype, dtype):
    x, weight8 = _rows8(x, "x"), None
    if isinstance(weight, Rows8):
        weight = weight8 = _rows8(weight, "weight")
        if dtype is None:
            dtype = bias.dtype if isinstance(bias, torch.Tensor) else (out_dtype if out_dtype in (torch.bfloat16, torch.float16) else torch.bfloat16)
    else:
        weight = _rows(weight, "weight")
        if dtype not in (None, weight.dtype):
            raise TypeError(f"dtype must be that of weight, {weight.dtype} (got {dtype})")
        dtype = weight.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"layers on rows in 8 bits are bfloat16 or float16 (got {dtype})")
    if weight.shape[1] != x.cols:
        raise ValueError(f"weight must have as many columns as x (got {tuple(weight.shape)} for x {tuple(x.shape)})")
    rows, out = x.shape[0], weight.shape[0]
    if bias is not None:
        bias = _rows(bias, "bias", dtype, ndim=1, shape=(out,))
    if out_dtype is None:
        out_dtype = dtype if residual is None else residual.dtype
    if out_dtype not in (dtype, torch.float32):
        raise TypeError(f"out_dtype must be {dtype} or float32 (got {out_dtype})")
    if residual is not None:
        residual = _rows(residual, "residual", out_dtype, shape=(rows, out))
    seed, step, word = _random(seed, step)
    desc = _lib.Linear(_TYPES[dtype], _TYPES[out_dtype], _act(act), 0, rows, x.cols, out, None, 0, None if weight8 else _p(weight),
                       0 if weight8 else _row_stride(weight), _p(bias), _p(residual), _row_stride(residual) if residual is not None else 0,
                       _probability(drop), seed, step, _p(word))
    return desc, (x, weight, bias, residual, word), out_dtype, weight8


def _linear8_call(desc, tensors, out_dtype, weight8, for_backward):
    L, x = _lib.lib(), tensors[0]
    if weight8 and for_backward:
        raise TypeError("weight must be a tensor where there are gradients: a weight in 8 bits is for answering")
    y = torch.empty((desc.rows, desc.out), dtype=out_dtype, device=x.q.device)
    w8 = C.byref(_rows8_c(weight8)) if weight8 else None
    saved_bytes = int(L.kge_linear8_saved_bytes(C.byref(desc))) if for_backward else 0
    ws_bytes = int(L.kge_linear8_fwd_workspace(C.byref(desc), w8, int(for_backward)))
    saved, ws = _bytes(saved_bytes, y.device), _bytes(ws_bytes, y.device)
    _lib.check(L.kge_linear8_fwd(C.byref(desc), C.byref(_rows8_c(x)), w8, _p(y), max(desc.out, 1), int(for_backward), _p(saved), saved_bytes, _p(ws),
                                 ws_bytes, _stream()), "kge_linear8_fwd")
    return y, saved


def _host8(x, weight, bias, act, residual, out_dtype, dtype, drop, seed, step, keep):
    """The native call, or None."""
    if isinstance(weight, Rows8):
        if weight.cols != x.cols:
            return None
        w, scale = weight.q, weight.scale
    else:
        w, scale = weight, None
    return _lib.host().linear8(x.q, x.scale, x.cols, w, scale, bias, _act(act), residual, out_dtype, dtype, drop, seed, step, keep)


def _linear8_backward(fw, dy, need_x, need_weight, need_bias) -> LinearGrads:
    x, weight, bias = fw.tensors[:3]
    got = _lib.host().linear8_backward(fw.desc, x.q, x.scale, x.cols, weight, fw.saved, dy, need_x, need_weight, need_bias and bias is not None)
    if got is not None:
        return LinearGrads(*got)
    d = _lib.Linear.from_buffer_copy(fw.desc)
    _tensor(x.q, "x of the forward call", 2)
    dy = _rows(dy, "dy", torch.float32 if d.out_type == 0 else weight.dtype, shape=(d.rows, d.out))  # (fw.y may be gone)
    dev = x.q.device
    dx = torch.empty((d.rows, d.in_), dtype=weight.dtype, device=dev) if need_x else None
    dw = torch.empty((d.out, d.in_), dtype=weight.dtype, device=dev) if need_weight else None
    db = torch.empty(d.out, dtype=weight.dtype, device=dev) if need_bias and bias is not None else None
    L = _lib.lib()
    ws_bytes = int(L.kge_linear8_bwd_workspace(C.byref(d)))
    ws = _bytes(ws_bytes, dev)
    _lib.check(L.kge_linear8_bwd(C.byref(d), C.byref(_rows8_c(x)), _p(dy), _row_stride(dy), _p(fw.saved), fw.saved.numel() if fw.saved is not None else 0,
                                 _p(dx), _p(dw), _p(db), _p(ws), ws_bytes, _stream()), "kge_linear8_bwd")
    return LinearGrads(dx, dw, db)


def _plain_dtype(x, weight, dtype):
    """x's own type is the only one where x is a tensor."""
    if isinstance(weight, Rows8):
        raise TypeError("a weight in 8 bits goes with rows in 8 bits (pack8)")
    if dtype is not None and isinstance(x, torch.Tensor) and dtype != x.dtype:
        raise TypeError(f"dtype must be that of x, {x.dtype} (got {dtype})")


def linear(x, weight, bias=None, *, act="none", residual=None, out_dtype=None, drop=0.0, seed=0, step=0, dtype=None) -> torch.Tensor:
    """``drop(act(x weight^T + bias)) + residual``: x [rows, in], weight [out, in], bias [out], residual [rows, out].

    act: "none", "relu", "gelu" or "silu"; drop, seed, step as in :func:`dropout`.  The output has x's type, or float32 by out_dtype (or
    because the residual is); 16-bit products are summed in fp32 and nothing is rounded before the end.

    x may be :class:`Rows8`, with a weight in bfloat16 or float16, whose type the layer has, or in 8 bits too: then dtype is the layer's (that of the bias, or
    bfloat16, unless said otherwise).  What is in 8 bits is multiplied as numbers of that type: float16 rounds those below 2^-21 and makes infinity of those from
    65520 up, bfloat16 takes all as they are."""
    if isinstance(x, Rows8):
        y = _host8(x, weight, bias, act, residual, out_dtype, dtype, drop, seed, step, False)
        if y is not None:
            return y
        desc, tensors, out_dtype, weight8 = _describe8(x, weight, bias, act, drop, seed, step, residual, out_dtype, dtype)
        return _linear8_call(desc, tensors, out_dtype, weight8, False)[0]
    if dtype is not None or isinstance(weight, Rows8):
        _plain_dtype(x, weight, dtype)
    y = _lib.host().linear(x, weight, bias, _act(act), residual, out_dtype, drop, seed, step, False)
    if y is not None:
        return y
    return _linear_call(*_describe(x, weight, bias, act, drop, seed, step, residual, out_dtype), False)[0]


def linear_forward(x, weight, bias=None, *, act="none", residual=None, out_dtype=None, drop=0.0, seed=0, step=0) -> LinearForward:
    """:func:`linear`, with what :func:`linear_backward` needs.  Of a layer on :class:`Rows8` that is those rows and, in 8 bits too, the activation's
    derivative: within 0.0025, 0.0014 in the mean square (some 0.0022 of the gradients, in float16 too).  The backward pass takes such rows less than 2^26 bytes apart."""
    if isinstance(x, Rows8):
        got = _host8(x, weight, bias, act, residual, out_dtype, None, drop, seed, step, True)
        if got is not None:
            y, saved, desc = got
            return LinearForward(y, desc, saved, (x, weight, bias, residual, None))
        desc, tensors, out_dtype, weight8 = _describe8(x, weight, bias, act, drop, seed, step, residual, out_dtype, None)
        y, saved = _linear8_call(desc, tensors, out_dtype, weight8, True)
        return LinearForward(y, bytes(desc), saved, tensors)
    if isinstance(weight, Rows8):
        _plain_dtype(x, weight, None)
    got = _lib.host().linear(x, weight, bias, _act(act), residual, out_dtype, drop, seed, step, True)
    if got is not None:
        y, saved, desc = got
        return LinearForward(y, desc, saved, (x, weight, bias, residual, None))
    desc, tensors, out_dtype = _describe(x, weight, bias, act, drop, seed, step, residual, out_dtype)
    y, saved = _linear_call(desc, tensors, out_dtype, True)
    return LinearForward(y, bytes(desc), saved, tensors)


def linear_backward(fw: LinearForward, dy, need_x: bool = True, need_weight: bool = True, need_bias: bool = True) -> LinearGrads:
    """Gradients of x, weight and bias from the gradient of y (of y's type).  That of x in 8 bits is the one at the values it stands for.

    What enters the two products is rounded to the layer's type.  In float16 that makes 0 of values below 3e-8 and infinity of those above 65504: scale
    the loss of a large batch up, and the gradients down again."""
    if not isinstance(fw, LinearForward):
        raise TypeError("fw must come from linear_forward()")
    x, _, bias = fw.tensors[:3]
    if isinstance(x, Rows8):
        return _linear8_backward(fw, dy, need_x, need_weight, need_bias)
    got = _lib.host().linear_backward(fw.desc, x, fw.saved, dy, need_x, need_weight, need_bias and bias is not None)
    if got is not None:
        return LinearGrads(*got)
    d = _lib.Linear.from_buffer_copy(fw.desc)
    _tensor(x, "x of the forward call", 2)
    dy = _rows(dy, "dy", fw.y.dtype, shape=fw.y.shape)
    dx = torch.empty((d.rows, d.in_), dtype=x.dtype, device=x.device) if need_x else None
    dw = torch.empty((d.out, d.in_), dtype=x.dtype, device=x.device) if need_weight else None
    db = torch.empty(d.out, dtype=x.dtype, device=x.device) if need_bias and bias is not None else None
    L = _lib.lib()
    ws_bytes = int(L.kge_linear_bwd_workspace(C.byref(d)))
    ws = _bytes(ws_bytes, x.device)
    _lib.check(L.kge_linear_bwd(C.byref(d), _p(dy), _row_stride(dy), _p(fw.saved), fw.saved.numel() if fw.saved is not None else 0, _p(dx),
                                _p(dw), _p(db), _p(ws), ws_bytes, _stream()), "kge_linear_bwd")
    return LinearGrads(dx, dw, db)


# ---- dropout ---------------------------------------------------------------------------------------
def dropout(x, p, seed, step=0, out=None) -> torch.Tensor:
    """x [rows, cols] with each element zero with probability p, the others scaled by 1 / (1 - p) (p to 1 / 65536).

    Which elements go is a function of (seed, step, row, column) alone, defined at kge_dropout in the C header; nothing is stored.  step: an
    integer, or one int64 on the GPU that the kernel reads (a captured graph then draws a new mask at every replay).  out: where to, x
    itself or other columns of the same array included."""
    if out is None:
        y = _lib.host().dropout(x, p, seed, step)
        if y is not None:
            return y
    x = _rows(x, "x")
    p = _probability(p)
    seed, step, word = _random(seed, step)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif _rows(out, "out", x.dtype, shape=x.shape) is not out:
        raise ValueError("out must have contiguous rows: it is written in place")
    elif not _apart(x, out):
        raise ValueError("out must be x itself or lie apart from it: elsewhere, or in other columns of the same rows")
    _lib.check(_lib.lib().kge_dropout(_TYPES[x.dtype], _p(x), _row_stride(x), _p(out), _row_stride(out), x.shape[0], x.shape[1], p, seed,
                                      step, _p(word), _stream()), "kge_dropout")
    return out


def dropout_backward(dy, p, seed, step=0, out=None) -> torch.Tensor:
    """The gradient of :func:`dropout`'s x: the same elements of dy dropped, the others scaled alike."""
    return dropout(dy, p, seed, step, out)


# ---- preference loss -------------------------------------------------------------------------------
def preference_loss(pos, neg, ref_pos=None, ref_neg=None, *, beta=1.0, kind="sigmoid", smoothing=0.0, temperature=0.0, mask=None,
                    sign=1.0):
    """(loss, dpos, dneg) of positive scores [B] against negative ones [B, N], relative to a frozen reference's scores of the same triples.

    With d = sign ((pos - ref_pos) - (neg - ref_neg)) a pair costs -(1 - smoothing) log sigma(beta d) - smoothing log sigma(-beta d)
    ("sigmoid"), max(0, 1 - beta d) ("hinge") or (d - 1 / (2 beta))^2 ("square").  A row's pairs are averaged, evenly or by
    softmax(temperature sign neg) (a constant to the gradient), rows evenly.  mask [B, N] (bool or uint8): False where there is no pair; what the
    scores hold there is not looked at, and a row without a pair costs nothing.  Nor does a pair that takes no share of the softmax (an infinitely low
    score, say); NaN stays NaN.  Gradients and loss are float32."""
    code = _lib.PREFERENCES.get(kind)
    if code is None:
        raise ValueError(f"kind must be one of {sorted(_lib.PREFERENCES)} (got {kind!r})")
    got = _lib.host().preference_loss(pos, neg, ref_pos, ref_neg, mask, code, beta, sign, smoothing, temperature)
    if got is not None:
        return got
    neg = _rows(neg, "neg")
    B, N = neg.shape
    pos = _rows(pos, "pos", neg.dtype, ndim=1, shape=(B,))
    if (ref_pos is None) != (ref_neg is None):
        raise ValueError("ref_pos and ref_neg go together")
    if ref_pos is not None:
        ref_pos, ref_neg = _rows(ref_pos, "ref_pos", neg.dtype, ndim=1, shape=(B,)), _rows(ref_neg, "ref_neg", neg.dtype, shape=(B, N))
    if mask is not None:
        if isinstance(mask, torch.Tensor) and mask.dtype == torch.bool:
            mask = mask.view(torch.uint8)
        mask = _rows(mask, "mask", torch.uint8, shape=(B, N))
    desc = _lib.Preference(_TYPES[neg.dtype], code, B, N, _p(pos), _p(neg), _row_stride(neg), _p(ref_pos), _p(ref_neg),
                           _row_stride(ref_neg) if ref_neg is not None else 0, _p(mask), _row_stride(mask) if mask is not None else 0,
                           float(beta), float(sign), float(smoothing), float(temperature))
    L = _lib.lib()
    f32 = dict(dtype=torch.float32, device=neg.device)
    loss, dpos, dneg = torch.empty(1, **f32), torch.empty(B, **f32), torch.empty((B, N), **f32)
    ws_bytes = int(L.kge_preference_workspace(C.byref(desc)))
    ws = _bytes(ws_bytes, neg.device)
    _lib.check(L.kge_preference_loss(C.byref(desc), _p(loss), _p(dpos), _p(dneg), _p(ws), ws_bytes, _stream()), "kge_preference_loss")
    return loss, dpos, dneg


# ---- rows in 8 bits --------------------------------------------------------------------------------
E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _fits8(q, scale, cols) -> bool:
    if not (isinstance(q, torch.Tensor) and isinstance(scale, torch.Tensor) and q.dtype is E4M3 and scale.dtype is _E8M0 and cols >= 0):
        return False
    shape = q.shape
    return len(shape) == 2 and shape[1] == -(-cols // 32) * 32 and scale.shape == (shape[0], -(-cols // 128) * 4)


def _refuse8(q, scale, cols):
    for t, name, dtype, width in ((q, "q", E4M3, -(-cols // 32) * 32), (scale, "scale", _E8M0, -(-cols // 128) * 4)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise TypeError(f"{name} must be a tensor of {dtype} (got {t.dtype if isinstance(t, torch.Tensor) else type(t).__name__})")
        if cols < 0 or t.dim() != 2 or t.shape[1] != width or t.shape[0] != q.shape[0]:
            raise ValueError(f"rows of {cols} values need {name} of shape {(q.shape[0] if q.dim() else 0, width)} (got {tuple(t.shape)})")


class Rows8:
    """Rows of ``cols`` values in 8 bits: e4m3 numbers and one power of two for each 32 columns, a value being their product.

    q [rows, 32 ceil(cols / 32)] (float8_e4m3fn), zero behind column cols; scale [rows, 4 ceil(cols / 128)] (float8_e8m0fnu), those behind the last
    block anything but NaN.  :func:`pack8` and :func:`rms_norm` make them; arrays made elsewhere are taken as they are."""
    __slots__ = ("q", "scale", "cols")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, cols: int):
        if not _fits8(q, scale, cols):
            _refuse8(q, scale, cols)
        self.q, self.scale, self.cols = q, scale, int(cols)

    @property
    def shape(self):
        return torch.Size((self.q.shape[0], self.cols))

    def __repr__(self):
        return f"Rows8(rows={self.q.shape[0]}, cols={self.cols}, device={self.q.device})"


def _made8(q, scale, cols) -> Rows8:
    """Rows8 of arrays that were made here."""
    r = Rows8.__new__(Rows8)
    r.q, r.scale, r.cols = q, scale, cols
    return r


def _laid(t: torch.Tensor, unit: int) -> torch.Tensor:
    """t with rows that start at multiples of `unit` bytes."""
    ok = (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or (t.stride(0) >= t.shape[1] and t.stride(0) % unit == 0)) and t.data_ptr() % unit == 0
    return t if ok else t.view(torch.uint8).clone(memory_format=torch.contiguous_format).view(t.dtype)


def _rows8(r, name: str) -> Rows8:
    if not isinstance(r, Rows8):
        raise TypeError(f"{name} must be Rows8 (got {type(r).__name__})")
    _tensor(r.q, f"{name}.q", 2), _tensor(r.scale, f"{name}.scale", 2)
    q, scale = _laid(r.q, 16), _laid(r.scale, 4)
    return r if q is r.q and scale is r.scale else Rows8(q, scale, r.cols)


def _rows8_c(r: Rows8) -> _lib.Rows8:
    one = r.q.shape[0] <= 1 or r.cols == 0  # (whose stride may be anything)
    return _lib.Rows8(_p(r.q), r.q.shape[1] if one else r.q.stride(0), _p(r.scale), r.scale.shape[1] if one else r.scale.stride(0))


def _new_rows8(rows: int, cols: int, device) -> Rows8:
    return Rows8(torch.empty((rows, 32 * (-(-cols // 32))), dtype=E4M3, device=device),
                 torch.empty((rows, 4 * (-(-cols // 128))), dtype=_E8M0, device=device), cols)


def pack8(x) -> Rows8:
    """x [rows, cols] in 8 bits: half the memory of 16 bits, each value within 2^-4 of itself (less than 2^-17 of its block's largest: within
    2^-19 of that).  What is infinite becomes NaN."""
    got = _lib.host().pack8(x)
    if got is not None:
        return _made8(*got, x.shape[1])
    x = _rows(x, "x")
    out = _new_rows8(x.shape[0], x.shape[1], x.device)
    _lib.check(_lib.lib().kge_pack8(_TYPES[x.dtype], _p(x), _row_stride(x), x.shape[0], x.shape[1], C.byref(_rows8_c(out)), _stream()), "kge_pack8")
    return out


def unpack8(rows8, dtype=torch.bfloat16) -> torch.Tensor:
    """What rows in 8 bits stand for, as bfloat16, float16 or float32 (exact, but for what float16 cannot hold: it rounds below 2^-21
    and has no number from 65520 up)."""
    if isinstance(rows8, Rows8):
        y = _lib.host().unpack8(rows8.q, rows8.scale, rows8.cols, dtype)
        if y is not None:
            return y
    r = _rows8(rows8, "rows8")
    if dtype not in _TYPES:
        raise TypeError(f"dtype must be float32, bfloat16 or float16 (got {dtype})")
    y = torch.empty(tuple(r.shape), dtype=dtype, device=r.q.device)
    _lib.check(_lib.lib().kge_unpack8(C.byref(_rows8_c(r)), r.shape[0], r.cols, _TYPES[dtype], _p(y), max(r.cols, 1), _stream()), "kge_unpack8")
    return y


# ---- norm ------------------------------------------------------------------------------------------
@dataclass
class NormForward:
    """A norm's output, and what its backward pass needs (h and weight have to stay as they are until then)."""
    y: torch.Tensor | Rows8
    h: torch.Tensor     # x + residual; x itself where there is none
    rstd: torch.Tensor  # float32 [rows]; -r 2^-64 where r is 2^128 or more
    weight: torch.Tensor | None
    rest: torch.Tensor | None = None  # int32 [rows, ceil(cols / 8)]: what h lost when it was rounded to 16 bits, in four bits an element
    eps: float = 1e-6


@dataclass
class NormGrads:
    x: torch.Tensor | None       # of x, and of the residual
    weight: torch.Tensor | None


def _norm_call(x, weight, residual, eps, out_dtype, keep):
    got = _lib.host().rms_norm(x, weight, residual, eps, out_dtype, keep)
    if got is not None:
        y, scale, h, rstd, rest = got
        return NormForward(y if scale is None else _made8(y, scale, x.shape[1]), x if h is None else h, rstd, weight, rest, float(eps))
    x = _rows(x, "x")
    rows, cols = x.shape
    if weight is not None:
        weight = _rows(weight, "weight", x.dtype, ndim=1, shape=(cols,))
    if residual is not None:
        residual = _rows(residual, "residual", x.dtype, shape=x.shape)
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative (got {eps})")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES and out_dtype != E4M3:
        raise TypeError(f"out_dtype must be float32, bfloat16, float16 or float8_e4m3fn (got {out_dtype})")
    eight = out_dtype == E4M3
    y = _new_rows8(rows, cols, x.device) if eight else torch.empty((rows, cols), dtype=out_dtype, device=x.device)
    h = torch.empty((rows, cols), dtype=x.dtype, device=x.device) if residual is not None else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
    rest = torch.empty((rows, -(-cols // 8)), dtype=torch.int32, device=x.device) if keep and h is not None and x.dtype != torch.float32 else None
    desc = _lib.RmsNorm(_TYPES[x.dtype], _lib.E4M3 if eight else _TYPES[out_dtype], rows, cols, _p(x), _row_stride(x), _p(residual),
                        _row_stride(residual) if residual is not None else 0, _p(weight), eps)
    _lib.check(_lib.lib().kge_rms_norm_fwd(C.byref(desc), None if eight else _p(y), cols, C.byref(_rows8_c(y)) if eight else None, _p(h), cols,
                                           _p(rstd), _p(rest), _stream()), "kge_rms_norm_fwd")
    return NormForward(y, x if h is None else h, rstd, weight, rest, eps)


def rms_norm(x, weight=None, residual=None, *, eps=1e-6, out_dtype=None):
    """``h / sqrt(mean(h^2) + eps) * weight`` of the rows of h = x + residual: x, residual [rows, cols] and weight [cols] of one type.

    out_dtype: float32, bfloat16 or float16 (x's, unless said otherwise), or float8_e4m3fn: :class:`Rows8`, as the layers behind it take them.  Gives y, or (y, h) where
    there is a residual; h is rounded to x's type, y is made of the sum before that."""
    got = _lib.host().rms_norm(x, weight, residual, eps, out_dtype, False)
    if got is not None:
        y = got[0] if got[1] is None else _made8(got[0], got[1], x.shape[1])
        return y if residual is None else (y, got[2])
    fw = _norm_call(x, weight, residual, eps, out_dtype, False)
    return fw.y if residual is None else (fw.y, fw.h)


def rms_norm_forward(x, weight=None, residual=None, *, eps=1e-6, out_dtype=None) -> NormForward:
    """:func:`rms_norm`, with what :func:`rms_norm_backward` needs."""
    return _norm_call(x, weight, residual, eps, out_dtype, True)


def rms_norm_backward(fw: NormForward, dy, dh=None, need_x: bool = True, need_weight: bool = True) -> NormGrads:
    """Gradients from that of y (float32, bfloat16 or float16, whatever y's own type) and, where h went on by itself, that of h (x's type).  The gradient of
    the residual is that of x.  An 8-bit y's rounding counts as none."""
    if not isinstance(fw, NormForward):
        raise TypeError("fw must come from rms_norm_forward()")
    got = _lib.host().rms_norm_backward(fw.h, fw.rstd, fw.rest, fw.weight, dy, dh, need_x, need_weight, fw.eps)
    if got is not None:
        return NormGrads(*got)
    h, weight, rest = _rows(fw.h, "h of the forward call"), fw.weight, fw.rest
    dy = _rows(dy, "dy", shape=h.shape)
    if dh is not None:
        dh = _rows(dh, "dh", h.dtype, shape=h.shape)
    rows, cols = h.shape
    rstd = _rows(fw.rstd, "rstd of the forward call", torch.float32, ndim=1, shape=(rows,))
    if weight is not None:
        weight = _rows(weight, "weight of the forward call", h.dtype, ndim=1, shape=(cols,))
    if rest is not None:
        rest = _rows(rest, "rest of the forward call", torch.int32, shape=(rows, -(-cols // 8))).contiguous()
    dx = torch.empty((rows, cols), dtype=h.dtype, device=h.device) if need_x else None
    dw = torch.empty(cols, dtype=h.dtype, device=h.device) if need_weight and weight is not None else None
    desc = _lib.RmsNorm(_TYPES[h.dtype], _TYPES[h.dtype], rows, cols, None, 0, None, 0, _p(weight), fw.eps)
    L = _lib.lib()
    ws_bytes = int(L.kge_rms_norm_bwd_workspace(C.byref(desc))) if dw is not None else 0
    ws = _bytes(ws_bytes, h.device)
    _lib.check(L.kge_rms_norm_bwd(C.byref(desc), _p(h), _row_stride(h), _p(rstd), _p(rest), _TYPES[dy.dtype], _p(dy), _row_stride(dy), _p(dh),
                                  _row_stride(dh) if dh is not None else 0, _p(dx), cols, _p(dw), _p(ws), ws_bytes, _stream()), "kge_rms_norm_bwd")
    return NormGrads(dx, dw)


# ---- encoder ---------------------------------------------------------------------------------------
@dataclass
class EncoderForward:
    rows: torch.Tensor  # float32 [n, dim]
    hidden: LinearForward
    last: LinearForward
    drop: tuple | None  # (p, seed, step) of the rows


@dataclass
class EncoderGrads:
    hidden: LinearGrads
    last: LinearGrads
    base: torch.Tensor  # gradient of the free rows


class FeatureEncoder:
    """Entity rows from feature rows: ``base + drop(act(x W1^T + b1)) W2^T + b2``, dropped once more on the way out.

    w1 [hidden, features], w2 [dim, hidden] with their biases, all of one type (bfloat16, float16 or float32); the rows are float32, as
    every score function takes them.  base are the entities' free rows of a table (or None)."""

    def __init__(self, w1, b1, w2, b2, act: str = "gelu", drop: float = 0.0, row_drop: float = 0.0, seed: int = 0):
        if w2.shape[1] != w1.shape[0]:
            raise ValueError(f"w2 must have as many columns as w1 has rows (got {tuple(w2.shape)} and {tuple(w1.shape)})")
        self.w1, self.b1, self.w2, self.b2 = w1, b1, w2, b2
        self.act, self.drop, self.row_drop, self.seed = act, _probability(drop), _probability(row_drop), int(seed)

    def encode(self, x, base=None) -> torch.Tensor:
        """Rows for answering with: nothing is dropped, nothing is kept."""
        return linear(linear(x, self.w1, self.b1, act=self.act), self.w2, self.b2, residual=base, out_dtype=torch.float32)

    def forward(self, x, base=None, step=0) -> EncoderForward:
        """Rows for a training step; step (an integer, or one int64 on the GPU) draws the masks."""
        hidden = linear_forward(x, self.w1, self.b1, act=self.act, drop=self.drop, seed=self.seed, step=step)
        last = linear_forward(hidden.y, self.w2, self.b2, residual=base, out_dtype=torch.float32)
        if self.row_drop == 0.0:
            return EncoderForward(last.y, hidden, last, None)
        drop = (self.row_drop, self.seed + 1, step)
        return EncoderForward(dropout(last.y, *drop), hidden, last, drop)

    def backward(self, fw: EncoderForward, drows, need_x: bool = False) -> EncoderGrads:
        """Gradients from those of the rows."""
        d = drows if fw.drop is None else dropout_backward(drows, *fw.drop)
        last = linear_backward(fw.last, d)
        return EncoderGrads(linear_backward(fw.hidden, last.x, need_x=need_x), last, d)


@dataclass
class Block:
    """A block's weights, or their gradients: norm [width], w1 [inner, width], b1 [inner], w2 [width, inner], b2 [width]."""
    norm: torch.Tensor
    w1: torch.Tensor | Rows8
    b1: torch.Tensor
    w2: torch.Tensor | Rows8
    b2: torch.Tensor


@dataclass
class ResidualForward:
    rows: torch.Tensor  # float32 [n, dim]
    first: LinearForward
    blocks: list        # (NormForward, LinearForward, LinearForward) of each
    norm: NormForward
    last: LinearForward


@dataclass
class ResidualGrads:
    first: LinearGrads
    blocks: list        # Block of each
    norm: torch.Tensor
    last: LinearGrads
    base: torch.Tensor  # gradient of the free rows


class ResidualEncoder:
    """Entity rows from feature rows through a residual stream:  h = x W_in^T + b_in;  of each block
    ``h += drop(act(norm(h) W1^T + b1)) W2^T + b2``;  rows = base + norm(h) W_out^T + b_out.

    All weights are of one type (bfloat16 or float16), the stream too; the rows are float32.  What goes into a layer (the norms' outputs, the hidden rows) is made in 8 bits and
    kept like that; x may be rows of the weights' type or :class:`Rows8`."""

    def __init__(self, w_in, b_in, blocks, norm, w_out, b_out, act: str = "gelu", drop: float = 0.0, seed: int = 0, eps: float = 1e-6):
        width = w_in.shape[0]
        for i, b in enumerate(blocks):
            if b.w1.shape[1] != width or b.w2.shape[0] != width or b.w2.shape[1] != b.w1.shape[0]:
                raise ValueError(f"block {i} must take and give rows of {width} (got {tuple(b.w1.shape)} and {tuple(b.w2.shape)})")
        if w_out.shape[1] != width:
            raise ValueError(f"w_out must have {width} columns (got {tuple(w_out.shape)})")
        self.w_in, self.b_in, self.blocks, self.norm, self.w_out, self.b_out = w_in, b_in, list(blocks), norm, w_out, b_out
        self.act, self.drop, self.seed, self.eps = act, _probability(drop), int(seed), float(eps)

    def packed(self) -> "ResidualEncoder":
        """The same encoder for answering, its weights in 8 bits (those of w_in stay: they multiply rows that nobody has packed)."""
        blocks = [Block(b.norm, pack8(b.w1), b.b1, pack8(b.w2), b.b2) for b in self.blocks]
        return ResidualEncoder(self.w_in, self.b_in, blocks, self.norm, pack8(self.w_out), self.b_out, self.act, self.drop, self.seed, self.eps)

    def encode(self, x, base=None) -> torch.Tensor:
        """Rows for answering with: nothing is dropped, nothing is kept."""
        h, more, dt = linear(x, self.w_in, self.b_in), None, self.w_in.dtype

        def norm(weight):
            nonlocal h
            y = rms_norm(h if more is None else more, weight, None if more is None else h, eps=self.eps, out_dtype=E4M3)
            if more is not None:
                y, h = y
            return y
        for b in self.blocks:
            more = linear(pack8(linear(norm(b.norm), b.w1, b.b1, act=self.act, dtype=dt)), b.w2, b.b2, dtype=dt)
        return linear(norm(self.norm), self.w_out, self.b_out, residual=base, out_dtype=torch.float32, dtype=dt)

    def forward(self, x, base=None, step=0) -> ResidualForward:
        """Rows for a training step; step (an integer, or one int64 on the GPU) draws the masks."""
        first = linear_forward(x, self.w_in, self.b_in)
        h, more, kept = first.y, None, []
        for i, b in enumerate(self.blocks):
            n = rms_norm_forward(h if more is None else more, b.norm, None if more is None else h, eps=self.eps, out_dtype=E4M3)
            hidden = linear_forward(n.y, b.w1, b.b1, act=self.act, drop=self.drop, seed=self.seed + i, step=step)
            out = linear_forward(pack8(hidden.y), b.w2, b.b2)
            kept.append((n, hidden, out))
            h, more = n.h, out.y
            hidden.y = out.y = None  # (the one is kept in 8 bits, the other is part of the stream)
        n = rms_norm_forward(h if more is None else more, self.norm, None if more is None else h, eps=self.eps, out_dtype=E4M3)
        last = linear_forward(n.y, self.w_out, self.b_out, residual=base, out_dtype=torch.float32)
        return ResidualForward(last.y, first, kept, n, last)

    def backward(self, fw: ResidualForward, drows, need_x: bool = False) -> ResidualGrads:
        """Gradients from those of the rows."""
        last = linear_backward(fw.last, drows)
        g = rms_norm_backward(fw.norm, last.x)
        norm, d, blocks = g.weight, g.x, []
        for n, hidden, out in reversed(fw.blocks):  # d: the gradient of the stream behind the block, and of what the block adds to it
            go = linear_backward(out, d)
            gh = linear_backward(hidden, go.x)
            g = rms_norm_backward(n, gh.x, d)
            blocks.append(Block(g.weight, gh.weight, gh.bias, go.weight, go.bias))
            d = g.x
        return ResidualGrads(linear_backward(fw.first, d, need_x=need_x), blocks[::-1], norm, last, drows)
