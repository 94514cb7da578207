"""Entity rows made from features, and a loss against a frozen model.

The score functions of :mod:`cuke_amd.kge` look rows up.  The operators here stand in front of that lookup and behind the scores:

  linear / linear_forward / linear_backward   ``drop(act(x W^T + b)) + residual`` and its gradients
  dropout / dropout_backward                  rows dropped by a counter-based generator; no mask is kept
  preference_loss                             positive against negative scores, relative to a frozen reference's
  FeatureEncoder                              two linear layers that turn feature rows into entity rows

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
           "preference_loss", "FeatureEncoder", "EncoderForward", "EncoderGrads"]

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
    """A layer's output, and what its backward pass needs (x and weight have to stay as they are until then)."""
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


def linear(x, weight, bias=None, *, act="none", residual=None, out_dtype=None, drop=0.0, seed=0, step=0) -> torch.Tensor:
    """``drop(act(x weight^T + bias)) + residual``: x [rows, in], weight [out, in], bias [out], residual [rows, out].

    act: "none", "relu", "gelu" or "silu"; drop, seed, step as in :func:`dropout`.  The output has x's type, or float32 by out_dtype (or
    because the residual is); 16-bit products are summed in fp32 and nothing is rounded before the end."""
    y = _lib.host().linear(x, weight, bias, _act(act), residual, out_dtype, drop, seed, step, False)
    if y is not None:
        return y
    return _linear_call(*_describe(x, weight, bias, act, drop, seed, step, residual, out_dtype), False)[0]


def linear_forward(x, weight, bias=None, *, act="none", residual=None, out_dtype=None, drop=0.0, seed=0, step=0) -> LinearForward:
    """:func:`linear`, with what :func:`linear_backward` needs."""
    got = _lib.host().linear(x, weight, bias, _act(act), residual, out_dtype, drop, seed, step, True)
    if got is not None:
        y, saved, desc = got
        return LinearForward(y, desc, saved, (x, weight, bias, residual, None))
    desc, tensors, out_dtype = _describe(x, weight, bias, act, drop, seed, step, residual, out_dtype)
    y, saved = _linear_call(desc, tensors, out_dtype, True)
    return LinearForward(y, bytes(desc), saved, tensors)


def linear_backward(fw: LinearForward, dy, need_x: bool = True, need_weight: bool = True, need_bias: bool = True) -> LinearGrads:
    """Gradients of x, weight and bias from the gradient of y (of y's type).

    What enters the two products is rounded to the layer's type.  In float16 that makes 0 of values below 3e-8 and infinity of those above 65504: scale
    the loss of a large batch up, and the gradients down again."""
    if not isinstance(fw, LinearForward):
        raise TypeError("fw must come from linear_forward()")
    x, _, bias = fw.tensors[:3]
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
