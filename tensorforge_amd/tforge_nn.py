"""Operators of the pre-norm residual MLP block on torch tensors: the
root-mean-square norm with the residual's addition (32, 16 or 8 bits out), the
products with bias, activation and residual in 16 and 8 bits, and their
gradients.

    h, y = x + r, ...         y, h = rms_norm(x, weight, residual=r)
    8-bit rows with scales    q, s, h = rms_norm(x, weight, residual=r, quantize=True)
                              q, s = quantize_rows(x)   (e4m3; quantize=torch.int8 and
                              quantize_rows(x, torch.int8): integers)
    act(x @ w + b) + r        out = linear(x, w, b, "gelu", r)
    8-bit product             out = linear(q, wq.t(), b, "gelu", r, x_scale=s, w_scale=ws)
    kept in 8 bits            x8 = keep8(x); x8.restore(); linear(..., keep8=True),
                              rms_norm(..., keep8=True) for their gradients
    loss over a vocabulary    loss = linear_cross_entropy(x, w, target)
    gradients                 dx, dweight = rms_norm_grad(dy, h, weight, dh=...)
                              dx, dw, dbias = linear_grad(dy, x, w, z, "gelu", bias_dtype=...)
                              dx, dw = linear_cross_entropy_grad(dloss, x, w, target, lse)

Every call enqueues kernels of libtforge_hip on the tensors' device and torch's
current stream, and returns new tensors; nothing is synchronised, and a call may
be captured in a HIP graph.  A tensor last written on another stream has to be
ordered before the call as for torch's own operators.  Tensors with leading
dimensions are taken as rows.  Where an input of rms_norm or linear requires a
gradient, autograd runs the gradient calls, which have no gradient themselves: a
second derivative raises RuntimeError.  Neither have the 8-bit results: with an input
that requires a gradient, quantize_rows, rms_norm into 8 bits, 8-bit products and the
gradient calls raise ValueError unless they run under torch.no_grad(); so does keep8.

Bad arguments raise ValueError or TypeError before any work (a number past 64 bits
OverflowError); errors of the library raise RuntimeError with its message.
"""

import functools

import torch

from tensorforge_amd import _lib

_lib.lib()  # the kernels; also the check that they are built
from tensorforge_amd import _nn_torch as _C  # noqa: E402  (links libtforge_hip.so)

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


class _Refused(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t):
        return t.view_as(t)

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("trying to differentiate twice: the gradient calls have no gradient (once_differentiable)")


def _once_differentiable(backward):
    """A backward whose results raise where a second derivative reaches them.  (torch's own decorator lets one through where the
    incoming gradient is a constant: the loss itself, or a sum.)"""

    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            got = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return got
        return tuple(t if t is None else _Refused.apply(t.detach().requires_grad_()) for t in got)

    return run


def _act(activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    return code


# ---- activations kept in 8 bits -----------------------------------------------------


class Kept8:
    """A tensor of `shape` and `dtype` (float32, bfloat16 or float16) kept in 8 bits, its bytes in `data` (uint8, contiguous).

    32 neighbours of a row of the last dimension share a unit, a power of two, and are integers of -127..127 times it;
    tf_keep8 in tforge_hip.h describes the bytes.  linear_grad and rms_norm_grad take it as it is.
    """

    __slots__ = ("data", "shape", "dtype")

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, tuple(shape), dtype

    def restore(self):
        """The tensor, each value within half a unit of what it was."""
        return _C.restore8(self.data, self.shape, self.dtype)

    def __repr__(self):
        return f"Kept8({self.shape}, {self.dtype})"


def keep8(x, positive=False, masked=False):
    """x in 8 bits (Kept8), 33 bytes for 32 values.  positive: values above zero stay above zero, as relu's gradient needs.

    A group of 32 that holds an infinity or a NaN comes back as NaN.  masked: minus infinity does not count there; it
    comes back as itself, and the values beside it as without it.
    """
    return Kept8(_C.keep8(x, True if positive else False, True if masked else False), x.shape, x.dtype)


def _tensor(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is not a tensor")
    return t


def _kept(t, name, like, columns):
    """What the native layer takes for an operand that may be kept in 8 bits."""
    if type(t) is Kept8:
        if t.dtype != like.dtype:
            raise TypeError(f"{name} was {t.dtype}, not {like.dtype}")
        if not t.shape or t.shape[-1] != columns:
            raise ValueError(f"{name} was {t.shape}, not rows of {columns}")
        return t.data
    if isinstance(t, torch.Tensor) and t.dtype is torch.uint8:
        raise TypeError(f"{name} is a tensor of bytes: what keep8 gave is passed as it is")
    return t


def _like(dx, x):
    return dx.view(x.shape) if type(x) is Kept8 and dx is not None and dx.shape != x.shape else dx


# ---- norm -----------------------------------------------------------------------


def rms_norm(x, weight, residual=None, eps=1e-6, quantize=False, keep8=False):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    Returns (y, h), h None without a residual; with quantize=True or an 8-bit dtype
    (q, scale, h): y in 8 bits (float8_e4m3fn, or int8) with one scale a row, y ~ q * scale.
    x is float32, bfloat16 or float16, the weight of x's type or float32.  keep8: where the
    result gets a gradient, h is kept for it in 8 bits (Kept8).
    """
    got = _C.rms_norm(x, weight, residual, eps, quantize)
    if got is not None:
        return got
    if quantize:
        raise ValueError("the 8-bit output has no gradient: call rms_norm under torch.no_grad(), or on detached tensors")
    y, h = _RmsNorm.apply(x, weight, residual, eps, keep8)
    return y, (None if residual is None else h)


def quantize_rows(x, dtype=torch.float8_e4m3fn):
    """(q, scale): x in 8 bits (float8_e4m3fn or int8) with one float32 scale a row of the last dimension, x ~ q * scale."""
    return _C.quantize_rows(x, dtype)


def rms_norm_grad(dy, h, weight, eps=1e-6, dh=None):
    """(dx, dweight) of rms_norm from the gradient dy of y and the norm's input h (x + residual).

    dh: the gradient that reaches h past the norm, added to dx; dx is the residual's gradient too.
    h may be kept in 8 bits (Kept8).
    """
    if type(h) is not Kept8:
        return _C.rms_norm_grad(dy, h, weight, eps, dh)
    dx, dw = _C.rms_norm_grad8(dy, _kept(h, "h", dy, dy.shape[-1] if _tensor(dy, "dy").dim() else 0), weight, eps, dh)
    return _like(dx, h), dw


def _saved(t, keep, positive=False):
    """What autograd saves of t: (t, None), or its bytes and what they stand for."""
    if t is None or not keep:
        return t, None
    kept = keep8(t, positive, masked=True)
    return kept.data, (kept.shape, kept.dtype)


def _again(t, kept):
    return t if kept is None else Kept8(t, *kept)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, keep):
        with torch.no_grad():
            y, h = rms_norm(x, weight, residual, eps)
            saved, ctx.kept = _saved(x if residual is None else h, keep)
        ctx.eps, ctx.added = eps, None if residual is None else residual.shape
        ctx.save_for_backward(saved, weight)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        h = _again(h, ctx.kept)
        if dy is None:  # h's alone, past the norm
            dx, dw = dh, None
        else:
            dx, dw = rms_norm_grad(dy.contiguous(), h, weight, ctx.eps, None if dh is None else dh.contiguous())
        if ctx.added is None:
            return dx, dw, None, None, None
        # A view would be another tensor on dx's memory, and both could become a leaf's grad.
        return dx, dw, dx if ctx.added == dx.shape else dx.reshape(ctx.added).clone(), None, None


# ---- products ---------------------------------------------------------------------


def linear(x, w, bias=None, activation="none", residual=None, keep=False, x_scale=None, w_scale=None, out_dtype=None,
           tile=0, splits=0, grad_terms=0, keep8=False):
    """z = x @ w + bias;  out = activation(z) + residual, rounded once.

    x (..., k) and w (k, n) are bfloat16 or float16; w may lie row by row or column by
    column (w = weight.t() of an n x k weight).  Or both are float8_e4m3fn, or both int8
    (sums exact, k at most 131071), w column by column, with x_scale (one a row) and
    w_scale (one a column), and out_dtype (bfloat16 unless given).  bias is of the output's type or float32.  activation:
    "none", "relu", "gelu" (by the normal distribution), "silu".  Returns out, or
    (out, z) with keep=True; both are differentiable.  tile and splits override the choice by sizes
    (tf_linear_args_t in tforge_hip.h); grad_terms is linear_grad's terms under autograd.
    keep8: where the result gets a gradient, x and the pre-activation are kept for it in
    8 bits (keep8, masked), relu's with the sign of every value.  A group of 32 neighbours with a NaN or plus infinity is
    NaN in the gradient; minus infinity (a unit masked by its bias) has a slope of 0 and leaves the others alone.
    """
    got = _C.linear(x, w, bias, _act(activation), residual, True if keep else False, x_scale, w_scale, out_dtype, tile,
                    splits)
    if got is not None:
        return got
    out, z = _Linear.apply(x, w, bias, residual, activation, keep, tile, splits, grad_terms, keep8)
    return (out, z) if keep else out


def linear_grad(dy, x, w, z=None, activation="none", bias_dtype=None, want_dx=True, want_dw=True, tile=0, splits=0,
                terms=0):
    """(dx, dw, dbias) of linear from the gradient dy of its output and the kept pre-activation z.

    dw lies in memory as w does.  dbias comes in bias_dtype (x's type or float32), None
    without one; what is not wanted is None.  The residual's gradient is dy itself.
    With gelu and silu the products take dz = dy * activation'(z) rounded to x's type
    (terms=1, an error of sqrt(2) of the results' own rounding) or with what the rounding
    left as a second term (terms=2, twice the time); 0 takes two up to 1.4e8 multiply-adds.
    x and z may be kept in 8 bits (Kept8).
    """
    if type(x) is not Kept8 and type(z) is not Kept8:
        return _C.linear_grad(dy, x, w, z, _act(activation), bias_dtype, True if want_dx else False,
                              True if want_dw else False, tile, splits, terms)
    _tensor(dy, "dy")
    if _tensor(w, "w").dim() != 2:
        raise ValueError(f"w is {tuple(w.shape)}, not k x n")
    dx, dw, dbias = _C.linear_grad8(dy, _kept(x, "x", dy, w.shape[0]), w, _kept(z, "z", dy, w.shape[1]), _act(activation), bias_dtype,
                                    True if want_dx else False, True if want_dw else False, tile, splits, terms)
    return _like(dx, x), dw, dbias


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, keep, tile, splits, terms, keep8):
        smooth = activation != "none"
        with torch.no_grad():
            if keep8 and smooth and not keep:  # z is written in 8 bits alone
                out, saved_z = _C.linear_keep8(x, w, bias, _act(activation), residual, False, None, None, None, tile, splits)
                z, kept_z = None, (out.shape, out.dtype)
            else:
                got = linear(x, w, bias, activation, residual, keep=keep or smooth, tile=tile, splits=splits)
                out, z = got if keep or smooth else (got, None)
                saved_z, kept_z = _saved(z if smooth else None, keep8, activation == "relu")
            saved_x, kept_x = _saved(x, keep8)
        ctx.save_for_backward(saved_x, w, saved_z)
        ctx.kept = kept_x, kept_z
        ctx.how = activation, None if bias is None else bias.dtype, tile, splits, terms
        ctx.added = None if residual is None else residual.shape
        ctx.set_materialize_grads(False)
        return out, z if keep else None

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy, dz):
        x, w, z = ctx.saved_tensors
        x, z = _again(x, ctx.kept[0]), _again(z, ctx.kept[1])
        activation, bias_dtype, tile, splits, terms = ctx.how
        need = ctx.needs_input_grad

        def grads(g, z, activation):
            return linear_grad(g.contiguous(), x, w, z, activation, bias_dtype if need[2] else None, need[0], need[1], tile,
                               splits, terms)

        # A gradient that reaches the kept z past the activation: its own products, added to the output's.
        got = [] if dy is None else [grads(dy, z, activation)]
        got += [] if dz is None else [grads(dz, None, "none")]
        total = (None, None, None) if not got else got[0] if len(got) == 1 else [a if a is None else a + b for a, b in zip(*got)]
        return (*total, dy.reshape(ctx.added) if need[3] and dy is not None else None, None, None, None, None, None,
                None)


# ---- the loss over a vocabulary -----------------------------------------------------

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(x, w, target, ignore_index=-100, reduction="mean", keep=False):
    """The cross entropy of the logits x @ w with the classes target, without the logits in memory.

    x (..., k) and w (k, n) are bfloat16 or float16, w row by row or column by column
    (w = weight.t() of an n x k weight); target (...) is int64.  loss[i] = log(sum of
    exp(logits[i])) - logits[i][target[i]] in float32.  Rows with the target ignore_index do not
    count: their loss is 0, and the mean is over the others (0 if there are none).  Any other
    target outside of 0..n-1 gives NaN, and so does a row with a logit of plus infinity or without one above minus
    infinity (magnitudes past 2.358e38 count as these).  reduction: "mean", "sum" or "none".  Returns the
    loss, or (loss, lse, count) with keep=True: what linear_cross_entropy_grad takes (lse is
    float64: a row that is sure of its class takes small differences of it).
    """
    code = REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"reduction {reduction!r} is not one of {', '.join(REDUCTIONS)}")
    got = _C.linear_xent(x, w, target, ignore_index, code)
    return got if keep else got[0]


def linear_cross_entropy_grad(dloss, x, w, target, lse, count=None, ignore_index=-100, want_dx=True, want_dw=True):
    """(dx, dw) of linear_cross_entropy from the gradient dloss of its loss (one number, or one a row) and the kept lse.

    count: the one kept with reduction="mean", whose gradient it then is.  dw lies in memory
    as w does.  The products take the logits' gradient rounded to x's type once, which adds up to a fifth to the results' own
    rounding with one dloss and two fifths with one a row; up to 64 rows in two terms, which adds nothing.  What is not wanted is None.
    """
    return _C.linear_xent_grad(dloss, x, w, target, lse, count, ignore_index, True if want_dx else False, True if want_dw else False)
