"""The operators that a training step over a vocabulary needs beside the
products and the optimizers, over the C ABI: layer norm and its gradients,
the log probabilities of given tokens with their loss's gradient, and the
clipping of gradients by their global norm.

Matrices are Tensors or TensorViews of any rank >= 1 whose last axis has its
elements side by side; the leading axes are the rows and have to step as one
axis (any contiguous tensor, a slice of one along its first or last axis).
Results go to the `out` arguments where they are given, else to new tensors,
made in the order of the call's stream (CudaStorage says how they go back);
an argument made on another stream is the caller's to order, and to keep until
the call has run.
Shapes that do not fit raise ValueError; the library's own refusals raise
TcError.  Nothing waits for the device.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass
from typing import Sequence

from . import _native as N
from .cuda import ELEM, CudaStorage, Tensor, TensorView, _stream

NO_TOKEN = N.NO_TOKEN
MAX_TOP = N.MAX_TOP


_BYTES = {name: nbytes for name, (_, nbytes) in ELEM.items()}


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(N.lib(), name)


def _run(name: str, stream, *args) -> None:
    """N.call with the stream last, its entry point looked up once: small
    calls cost what their checks do."""
    status = _entry(name)(*args, stream if type(stream) is int else _stream(stream))
    if status:
        N.check(name, status)


def _matrix(what: str, x, dtype: str | None = None) -> tuple[int, int, int, int]:
    """(address, rows, cols, row stride) of x read as a matrix."""
    storage, shape = x.storage, x.shape
    if dtype is not None and storage.dtype != dtype:
        raise ValueError(f"{what}: element type {storage.dtype}, expected {dtype}")
    if not shape:
        raise ValueError(f"{what}: a scalar has no rows")
    cols, rows = shape[-1], 1
    for e in shape[:-1]:
        rows *= e
    if type(x) is Tensor:
        if rows * cols > storage.len:
            raise ValueError(f"{what}: shape {list(shape)} reaches past {storage.len} elements")
        return storage.ptr, rows, cols, cols
    strides = x.strides
    if cols > 1 and strides[-1] != 1:
        raise ValueError(f"{what}: the last axis steps by {strides[-1]}, call contiguous() first")
    if len(shape) == 2:
        stride = strides[0] if rows > 1 else cols
    else:
        stride, step = cols, None
        for e, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
            if e == 1:
                continue
            if step is None:
                stride = s
            elif s != step:
                raise ValueError(f"{what}: the leading axes {shape[:-1]} do not step as one, call contiguous() first")
            step = s * e
    if x.offset < 0:
        raise ValueError(f"{what}: begins before its storage, at element {x.offset}")
    if rows and cols:
        reach = x.offset + (rows - 1) * stride + cols
        if reach > storage.len:
            raise ValueError(f"{what}: reaches element {reach}, past {storage.len} elements")
    return storage.ptr + x.offset * _BYTES[storage.dtype], rows, cols, stride


def _vector(what: str, x, n: int, dtypes: Sequence[str]) -> int | None:
    """The address of x's n contiguous elements; None for None."""
    if x is None:
        return None
    kind, offset = type(x), 0
    if kind is CudaStorage:
        storage, held = x, x.len
    else:
        storage, shape = x.storage, x.shape
        held = 1
        for e in shape:
            held *= e
        if kind is TensorView:
            offset = x.offset
            if shape and (len(shape) > 1 or x.strides[0] != 1) and not x.is_contiguous():
                raise ValueError(f"{what}: not contiguous")
    if storage.dtype not in dtypes:
        raise ValueError(f"{what}: element type {storage.dtype}, expected {' or '.join(dtypes)}")
    if offset < 0:
        raise ValueError(f"{what}: begins before its storage, at element {offset}")
    if held != n or offset + n > storage.len:
        raise ValueError(f"{what}: {held} elements, expected {n}")
    return storage.ptr + offset * _BYTES[storage.dtype]


def _new(shape, dtype: str, stream) -> Tensor:
    n = 1
    for e in shape:
        n *= e
    return Tensor(CudaStorage(dtype, n, stream=stream), shape)


def _same_shape(what: str, x, y) -> None:
    if x.shape != y.shape and list(x.shape) != list(y.shape):
        raise ValueError(f"{what}: shapes {list(x.shape)} and {list(y.shape)} differ")


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None, statistics=None, stream=None):
    """(y, statistics): each row of x normalised, times weight, plus bias.
    weight and bias hold one value per column, in x's type or f32 (both in the
    same).  statistics [rows, 2] (f32) holds each row's mean and
    1/sqrt(variance + eps), for layer_norm_backward.  out may be x."""
    ptr, rows, cols, stride = _matrix("layer_norm: x", x)
    dtype = x.storage.dtype
    kinds = (dtype, "f32")
    w, b = _vector("layer_norm: weight", weight, cols, kinds), _vector("layer_norm: bias", bias, cols, kinds)
    kind = _dtype(weight) or _dtype(bias) or dtype
    if weight is not None and bias is not None and _dtype(bias) != kind:
        raise ValueError(f"layer_norm: weight is {kind}, bias {_dtype(bias)}")
    if out is None:
        out = _new(x.shape, dtype, stream)
    else:
        _same_shape("layer_norm", x, out)
    yptr, _, _, ystride = _matrix("layer_norm: out", out, dtype)
    if statistics is None:
        statistics = _new([rows, 2], "f32", stream)
    st = _vector("layer_norm: statistics", statistics, 2 * rows, ("f32",))
    _run("tc_layer_norm", stream, N.DTYPES[dtype], N.DTYPES[kind], rows, cols, ptr, stride, w, b, eps, yptr, ystride, st)
    return out, statistics


def _dtype(x) -> str | None:
    return None if x is None else x.dtype if type(x) is CudaStorage else x.storage.dtype


def layer_norm_backward(grad, x, statistics, weight=None, out=None, grad_weight=None, grad_bias=None, stream=None):
    """(grad_x, grad_weight, grad_bias) of layer_norm, from the gradient of its
    y, its x and the statistics it left.  grad_weight and grad_bias are in
    weight's type (x's without a weight); out may be grad or x."""
    ptr, rows, cols, stride = _matrix("layer_norm_backward: x", x)
    dtype = x.storage.dtype
    _same_shape("layer_norm_backward", x, grad)
    gptr, _, _, gstride = _matrix("layer_norm_backward: grad", grad, dtype)
    w = _vector("layer_norm_backward: weight", weight, cols, (dtype, "f32"))
    kind = _dtype(weight) or _dtype(grad_weight) or _dtype(grad_bias) or dtype
    st = _vector("layer_norm_backward: statistics", statistics, 2 * rows, ("f32",))
    if out is None:
        out = _new(x.shape, dtype, stream)
    else:
        _same_shape("layer_norm_backward", x, out)
    optr, _, _, ostride = _matrix("layer_norm_backward: out", out, dtype)
    if grad_weight is None:
        grad_weight = _new([cols], kind, stream)
    if grad_bias is None:
        grad_bias = _new([cols], kind, stream)
    gw = _vector("layer_norm_backward: grad_weight", grad_weight, cols, (kind,))
    gb = _vector("layer_norm_backward: grad_bias", grad_bias, cols, (kind,))
    _run("tc_layer_norm_backward", stream, N.DTYPES[dtype], N.DTYPES[kind], rows, cols, gptr, gstride, ptr, stride, st, w,
           optr, ostride, gw, gb)
    return out, grad_weight, grad_bias


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------
@dataclass
class TokenLogprobs:
    """What token_logprobs gives for each row; None: not computed.  All f32
    but top_tokens (u32); statistics is [rows, 2], the top ones [rows, top]."""

    logprobs: object = None
    entropy: object = None
    statistics: object = None
    top_tokens: object = None
    top_logprobs: object = None


def _fresh(rows: int, tokens, entropy: bool, top: int, stream) -> TokenLogprobs:
    def new(shape, dtype="f32"):
        return _new(shape, dtype, stream)

    return TokenLogprobs(new([rows]) if tokens is not None else None, new([rows]) if entropy else None, new([rows, 2]),
                         new([rows, top], "u32") if top else None, new([rows, top]) if top else None)


def _results(what: str, out: TokenLogprobs, rows: int) -> tuple:
    return (_vector(what + ": logprobs", out.logprobs, rows, ("f32",)),
            _vector(what + ": entropy", out.entropy, rows, ("f32",)),
            _vector(what + ": statistics", out.statistics, 2 * rows, ("f32",)))


def token_logprobs(logits, tokens=None, top: int = 0, entropy: bool = True, out: TokenLogprobs | None = None,
                   stream=None) -> TokenLogprobs:
    """The log probability of each row's token (tokens: u32, one per row,
    NO_TOKEN where there is none), the row's entropy and its `top` likeliest
    tokens (at most MAX_TOP), under the softmax of each row of logits.  With
    `out`, its fields that are not None are computed, and `top` is the last
    extent of out.top_tokens."""
    ptr, rows, vocab, stride = _matrix("token_logprobs: logits", logits)
    tok = _vector("token_logprobs: tokens", tokens, rows, ("u32",))
    if out is None:
        out = _fresh(rows, tokens, entropy, top, stream)
    elif (out.top_tokens is None) != (out.top_logprobs is None):
        raise ValueError("token_logprobs: top_tokens and top_logprobs go together")
    else:
        top = 0 if out.top_tokens is None else out.top_tokens.shape[-1]
    lp, ent, st = _results("token_logprobs", out, rows)
    tt = _vector("token_logprobs: top_tokens", out.top_tokens, rows * top, ("u32",))
    tl = _vector("token_logprobs: top_logprobs", out.top_logprobs, rows * top, ("f32",))
    _run("tc_token_logprobs", stream, N.DTYPES[logits.storage.dtype], rows, vocab, ptr, stride,
           tok, lp, ent, st, top, tt, tl)
    return out


def token_logprobs_backward(logits, tokens, statistics, grad_logprobs=None, entropy=None, grad_entropy=None, out=None,
                            stream=None):
    """The logits' gradient, from the gradients (f32, one per row; None: zero)
    of the logprobs and of the entropies that token_logprobs gave, its
    statistics and, where grad_entropy is given, its entropies.  out may be
    logits."""
    ptr, rows, vocab, stride = _matrix("token_logprobs_backward: logits", logits)
    dtype = logits.storage.dtype
    each = [_vector("token_logprobs_backward: " + name, v, rows, (kind,))
            for name, v, kind in (("tokens", tokens, "u32"), ("entropy", entropy, "f32"),
                                  ("grad_logprobs", grad_logprobs, "f32"), ("grad_entropy", grad_entropy, "f32"))]
    st = _vector("token_logprobs_backward: statistics", statistics, 2 * rows, ("f32",))
    if out is None:
        out = _new(logits.shape, dtype, stream)
    else:
        _same_shape("token_logprobs_backward", logits, out)
    optr, _, _, ostride = _matrix("token_logprobs_backward: out", out, dtype)
    _run("tc_token_logprobs_backward", stream, N.DTYPES[dtype], rows, vocab, ptr, stride, each[0], st, each[1], each[2],
           each[3], optr, ostride)
    return out


def token_loss(logits, tokens, grad_logprobs, grad_entropy=None, out: TokenLogprobs | None = None, grad=None,
               stream=None):
    """(TokenLogprobs, grad): token_logprobs and token_logprobs_backward in
    one call that reads the logits from memory once, for losses whose
    gradient in the logprobs (and entropies) is known beforehand.  grad may
    be logits; with `out`, its fields that are not None are computed."""
    ptr, rows, vocab, stride = _matrix("token_loss: logits", logits)
    dtype = logits.storage.dtype
    given = (_vector("token_loss: tokens", tokens, rows, ("u32",)),
             _vector("token_loss: grad_logprobs", grad_logprobs, rows, ("f32",)),
             _vector("token_loss: grad_entropy", grad_entropy, rows, ("f32",)))
    if out is None:
        out = _fresh(rows, tokens, True, 0, stream)
    elif out.top_tokens is not None or out.top_logprobs is not None:
        raise ValueError("token_loss: the top tokens are token_logprobs'")
    if grad is None:
        grad = _new(logits.shape, dtype, stream)
    else:
        _same_shape("token_loss", logits, grad)
    gptr, _, _, gstride = _matrix("token_loss: grad", grad, dtype)
    lp, ent, st = _results("token_loss", out, rows)
    _run("tc_token_loss", stream, N.DTYPES[dtype], rows, vocab, ptr, stride, *given, lp, ent, st, gptr, gstride)
    return out, grad


# ---------------------------------------------------------------------------
# the gradients' global norm, and clipping
# ---------------------------------------------------------------------------
class GradList:
    """The gradients of a step (Tensors, contiguous TensorViews or
    CudaStorages, of any of the element types), and where they go clipped:
    `outs`, or in place.  A program builds it once and passes it every step."""

    def __init__(self, grads: Sequence, outs: Sequence | None = None):
        grads, outs = list(grads), list(grads if outs is None else outs)
        if len(grads) != len(outs):
            raise ValueError(f"GradList: {len(grads)} gradients, {len(outs)} outputs")
        self._keep = (grads, outs)  # the storages live as long as the list
        self.count = len(grads)
        self.entries = (N.Gradient * max(1, self.count))()
        for e, g, o in zip(self.entries, grads, outs):
            n = g.len if isinstance(g, CudaStorage) else g.numel()
            e.g = _vector("GradList: gradient", g, n, ("f32", "f16", "bf16"))
            e.out = _vector("GradList: output", o, n, (g.dtype,))
            e.n, e.dtype = n, N.DTYPES[g.dtype]


def _list(grads) -> GradList:
    return grads if isinstance(grads, GradList) else GradList(grads)


def grad_norm(grads, out=None, stream=None):
    """The square root of the sum of all gradients' squares, one f32 on the
    device."""
    grads = _list(grads)
    if out is None:
        out = _new([1], "f32", stream)
    _run("tc_grad_norm", stream, grads.entries, grads.count, _vector("grad_norm: out", out, 1, ("f32",)))
    return out


def clip_grads(grads, norm, limit: float, stream=None) -> None:
    """Every gradient times min(1, limit / norm), norm a device f32 (grad_norm's,
    or one combined over ranks)."""
    grads = _list(grads)
    _run("tc_clip_grads", stream, grads.entries, grads.count, _vector("clip_grads: norm", norm, 1, ("f32",)), float(limit))
