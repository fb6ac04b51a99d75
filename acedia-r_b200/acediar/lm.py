"""Operators of language models over gpuTensors: token log probabilities, the
residual update with its norms, products with 4-bit weights.

They follow tensor.py: axes and tokens count from 1, storage is column-major,
computation is a call into libacediar_b200.so on the current torch stream.  The
formulas and every rule on masked, missing and empty values stand beside the C
functions in include/acd.h.  The reference has none of these operators.
"""
import ctypes
import functools
import numbers
import struct
from collections import namedtuple

import torch

from . import _lib as L
from .tensor import _TORCH, _norm_dtype, _stream, context, contiguous, gpuTensor

TokenLogprob = namedtuple("TokenLogprob", "logprob entropy logsumexp top_index top_logprob")
ResidualNorm = namedtuple("ResidualNorm", "h y rstd_h rstd_block")
ResidualNormGrad = namedtuple("ResidualNormGrad", "d_residual d_block d_w_pre d_w_post d_gate")
Quant4 = namedtuple("Quant4", "weights scales zeros")

_UNSUPPORTED = 8


# A small call's time is its host time, so what follows from a shape alone is
# worked out once a shape.
@functools.lru_cache(maxsize=4096)
def _layout(shape):
    """Elements to allocate and column-major strides."""
    n, strides = 1, []
    for s in shape:
        strides.append(n)
        n *= s
    return n or 1, tuple(strides)


def _new(shape, dtype, device):
    """An uninitialised tensor; shape is a tuple of ints.  (The attributes are set
    without the constructor's checks.)"""
    t = gpuTensor.__new__(gpuTensor)
    n, t.strides = _layout(shape)
    t.storage = torch.empty(n, dtype=_TORCH[dtype], device=device)
    t.shape, t.dtype, t.offset = shape, dtype, 0
    return t


# the layout of acd_desc in two parts: where the data is, and its form
_pack_at = struct.Struct("Pq").pack
_pack_form = struct.Struct("%dq%dqii" % (L.MAX_DIMS, L.MAX_DIMS)).pack
assert struct.calcsize("Pq%dq%dqii" % (L.MAX_DIMS, L.MAX_DIMS)) == ctypes.sizeof(L.Desc)


@functools.lru_cache(maxsize=4096)
def _form(shape, strides, dtype):
    pad = (0,) * (L.MAX_DIMS - len(shape))
    return _pack_form(*shape, *pad, *strides, *pad, len(shape), L.DTYPE_CODES[dtype])


_functions = {}


def _call(name):
    """The C function, taking descriptors as bytes: these calls have up to 14 of
    them, and a ctypes structure costs three times as much to make."""
    f = _functions.get(name)
    if f is None:
        lib = L.lib()
        f = lib[name]  # a function object of its own
        f.argtypes = [ctypes.c_char_p if t is ctypes.POINTER(L.Desc) else t for t in getattr(lib, name).argtypes]
        f.restype = ctypes.c_int32
        _functions[name] = f
    return f


def _desc(t):
    if t is None:
        return None
    return _pack_at(t.storage.data_ptr(), t.offset) + _form(t.shape, t.strides, t.dtype)


def _dense(t):
    """The tensor itself, or a column-major copy of a view.  (The caller keeps
    the copy in a variable: its memory is free again once nothing refers to it.)"""
    return t if t is None or t.is_contiguous() else contiguous(t)


def _axis0(x, axis):
    if type(axis) is int and 1 <= axis <= len(x.shape):
        return axis - 1
    if not isinstance(axis, numbers.Number) or axis != int(axis) or axis < 1 or axis > x.ndims:
        raise ValueError("axis must be a single positive integer within tensor dimensions")
    return int(axis) - 1


def _row_shape(x, a):
    return x.shape[:a] + x.shape[a + 1:] or (1,)


def _rows(x, inplace=False):
    """Views of up to two axes are taken as they are; others are made dense (never in place)."""
    return x if x is None or inplace or x.ndims <= 2 or x.is_contiguous() else contiguous(x)


def _stat_dtype(x):
    return "double" if x.dtype == "double" else "float"


def token_logprob(logits, tokens=None, axis=1, scale=1.0, top=0):
    """Log probability of one given token a row under softmax(scale * logits),
    with the row's entropy and log-sum-exp and, for top > 0, its `top` most
    likely tokens (at most 32) and their log probabilities.

    logits: "float", "double" or "float16"; a row is all elements along `axis`.
    tokens: "int32" or "int64", the logits' shape without `axis` (or 1 there),
    counted from 1; 0 asks for nothing (logprob 0), NA and tokens outside the
    vocabulary give NaN.  Masked logits are -Inf.  top_index and top_logprob
    have the logits' shape with extent `top` on the axis, equal logits in the
    order of their index.  Returns TokenLogprob; what was not asked for is
    None."""
    a = _axis0(logits, axis)
    if not isinstance(top, numbers.Number) or top != int(top) or top < 0:
        raise ValueError("top must be a whole number, 0 or more")
    st, shape, dev = _stat_dtype(logits), _row_shape(logits, a), logits.device
    logprob = _new(shape, st, dev) if tokens is not None else None
    entropy, lse = _new(shape, st, dev), _new(shape, st, dev)
    index = top_logprob = None
    if top:
        tshape = logits.shape[:a] + (int(top),) + logits.shape[a + 1:]
        index, top_logprob = _new(tshape, "int64", dev), _new(tshape, st, dev)
    f, c, s = _call("acd_token_logprob"), context(), _stream()
    out = [_desc(t) for t in (logprob, entropy, lse, index, top_logprob)]
    tokens = _dense(tokens)
    r = f(c, *out, _desc(logits), _desc(tokens), a, scale, 1, s)
    if r == _UNSUPPORTED and not logits.is_contiguous():
        logits = contiguous(logits)
        r = f(c, *out, _desc(logits), _desc(tokens), a, scale, 1, s)
    L.check(r, "token_logprob")
    return TokenLogprob(logprob, entropy, lse, index, top_logprob)


def token_logprob_grad(logits, tokens, logsumexp, entropy=None, d_logprob=None, d_entropy=None, d_logsumexp=None,
                       axis=1, scale=1.0, inplace=False):
    """The gradient of token_logprob with respect to the logits: logsumexp and
    entropy as it returned them, d_logprob, d_entropy, d_logsumexp the loss's
    gradients with respect to its outputs (None: none).  inplace=True writes
    the gradient over the logits."""
    a = _axis0(logits, axis)
    f, c, s = _call("acd_token_logprob_grad"), context(), _stream()
    grad = logits if inplace else _new(logits.shape, logits.dtype, logits.device)
    rest = [_dense(t) for t in (logsumexp, entropy, d_logprob, d_entropy, d_logsumexp)]
    tokens = _dense(tokens)
    r = f(c, _desc(grad), _desc(logits), _desc(tokens), a, scale, *[_desc(t) for t in rest], 1, s)
    if r == _UNSUPPORTED and not inplace and not logits.is_contiguous():
        logits = contiguous(logits)
        r = f(c, _desc(grad), _desc(logits), _desc(tokens), a, scale, *[_desc(t) for t in rest], 1, s)
    L.check(r, "token_logprob_grad")
    return grad


def residual_norm(residual, block, w_pre, w_post=None, gate=None, axis=1, alpha=1.0, eps=1e-6, inplace=False):
    """A residual update with the norms around it (root mean square, rows
    along `axis`):

        h = alpha * residual + gate * (block / rms(block) * w_post)
        y = h / rms(h) * w_pre

    Without w_post the block is added as it is, without gate unscaled.  gate
    has one element for each of a row, or the residual's shape with 1 on any
    leading axes other than `axis` (a gate for each sample; an axis in the
    middle leaves extents other than 1 to one side of it).  inplace=True writes
    h over the residual and y over the block.  Returns ResidualNorm;
    rstd_h and rstd_block are what residual_norm_grad takes."""
    a = _axis0(block, axis)
    dev, st, shape = block.device, _stat_dtype(block), _row_shape(block, a)
    residual, block = _rows(residual, inplace), _rows(block, inplace)
    w_pre, w_post, gate = _dense(w_pre), _dense(w_post), _dense(gate)
    h = residual if inplace else _new(block.shape, block.dtype, dev)
    y = block if inplace else _new(block.shape, block.dtype, dev)
    rh = _new(shape, st, dev)
    rb = _new(shape, st, dev) if w_post is not None else None
    L.check(_call("acd_residual_norm")(context(), _desc(h), _desc(y), _desc(rh), _desc(rb), _desc(residual),
                                       _desc(block), _desc(w_pre), _desc(w_post), _desc(gate), a, alpha, eps,
                                       _stream()), "residual_norm")
    return ResidualNorm(h, y, rh, rb)


def residual_norm_grad(d_h, d_y, h, block, rstd_h, rstd_block, w_pre, w_post=None, gate=None, axis=1, alpha=1.0):
    """The gradients of residual_norm: d_h and d_y are the loss's gradients with
    respect to h (None: none) and y; h, rstd_h, rstd_block as it returned them.
    The gradients of w_pre, w_post and gate are sums over all rows that an
    element was used for, in "float" ("double" for doubles).  Returns
    ResidualNormGrad."""
    a = _axis0(block, axis)
    dev, st = block.device, _stat_dtype(block)
    d_h, d_y, h, block = _rows(d_h), _rows(d_y), _rows(h), _rows(block)
    w_pre, w_post, gate, rstd_h, rstd_block = (_dense(t) for t in (w_pre, w_post, gate, rstd_h, rstd_block))
    dr, db = _new(block.shape, block.dtype, dev), _new(block.shape, block.dtype, dev)
    like = lambda t: None if t is None else _new(t.shape, st, dev)  # noqa: E731
    dpre, dpost, dgate = like(w_pre), like(w_post), like(gate)
    L.check(_call("acd_residual_norm_grad")(
        context(), _desc(dr), _desc(db), _desc(dpre), _desc(dpost), _desc(dgate), _desc(d_h), _desc(d_y), _desc(h),
        _desc(block), _desc(rstd_h), _desc(rstd_block), _desc(w_pre), _desc(w_post), _desc(gate), a, alpha,
        _stream()), "residual_norm_grad")
    return ResidualNormGrad(dr, db, dpre, dpost, dgate)


def quant4_encode(w, group=128, zeros=False, scale_dtype="float16"):
    """4-bit weights of an [out, in] matrix: Quant4(weights, scales, zeros) with
    one scale (and, with zeros=True, one zero point) for each `group` inputs of
    an output.  weights is an "int8" tensor [16 * ceil(in / 32), out] with two
    weights a byte along the inputs, the even one in the low half."""
    if w.ndims != 2:
        raise ValueError("quant4_encode: an [out, in] matrix required")
    if not isinstance(group, numbers.Number) or group != int(group) or group <= 0 or group % 32:
        raise ValueError("group must be a positive multiple of 32")
    out, inner = w.shape
    sd = _norm_dtype(scale_dtype)
    q = _new((16 * -(-inner // 32), out), "int8", w.device)
    s = _new((-(-inner // group), out), sd, w.device)
    z = _new(s.shape, sd, w.device) if zeros else None
    L.check(_call("acd_quant4_encode")(context(), _desc(q), _desc(s), _desc(z), _desc(w), int(group), _stream()),
            "quant4_encode")
    return Quant4(q, s, z)


def quant4_matvec(weights, scales, x, group=128, zeros=None, out_dtype=None):
    """W %*% x for weights in 4 bits (see quant4_encode) and x [in] or [in, n],
    "float" or "float16"; the result has x's dtype unless out_dtype says
    otherwise."""
    if not isinstance(group, numbers.Number) or group != int(group) or group <= 0 or group % 32:
        raise ValueError("group must be a positive multiple of 32")
    if weights.ndims != 2 or x.ndims not in (1, 2):
        raise ValueError("quant4_matvec: weights from quant4_encode and x [in] or [in, n] required")
    odt = x.dtype if out_dtype is None else _norm_dtype(out_dtype)
    weights, scales, zeros = _dense(weights), _dense(scales), _dense(zeros)
    out = _new((weights.shape[1],) + x.shape[1:], odt, x.device)
    L.check(_call("acd_quant4_matvec")(context(), _desc(out), _desc(weights), _desc(scales), _desc(zeros), _desc(x),
                                      int(group), _stream()), "quant4_matvec")
    return out
