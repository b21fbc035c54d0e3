"""Operators of the pre-norm residual MLP block on torch tensors: the
root-mean-square norm with the residual's addition (32, 16 or 8 bits out), the
products with bias, activation and residual in 16 and 8 bits, and their
gradients.

    h, y = x + r, ...         y, h = rms_norm(x, weight, residual=r)
    8-bit rows with scales    q, s, h = rms_norm(x, weight, residual=r, quantize=True)
                              q, s = quantize_rows(x)
    act(x @ w + b) + r        out = linear(x, w, b, "gelu", r)
    8-bit product             out = linear(q, wq.t(), b, "gelu", r, x_scale=s, w_scale=ws)
    gradients                 dx, dweight = rms_norm_grad(dy, h, weight, dh=...)
                              dx, dw, dbias = linear_grad(dy, x, w, z, "gelu", bias_dtype=...)

Every call enqueues kernels of libtforge_hip on the tensors' device and torch's
current stream, and returns new tensors; nothing is synchronised, and a call may
be captured in a HIP graph.  A tensor last written on another stream has to be
ordered before the call as for torch's own operators.  Tensors with leading
dimensions are taken as rows.  Where an input of rms_norm or linear requires a
gradient, autograd runs the gradient calls, which have no gradient themselves: a
second derivative raises RuntimeError.  Neither have the 8-bit results: with an input
that requires a gradient, quantize_rows, rms_norm into 8 bits, 8-bit products and the
gradient calls raise ValueError unless they run under torch.no_grad().

Bad arguments raise ValueError or TypeError before any work; errors of the
library raise RuntimeError with its message.
"""

import torch
from torch.autograd.function import once_differentiable

from tensorforge_amd import _lib

_lib.lib()  # the kernels; also the check that they are built
from tensorforge_amd import _nn_torch as _C  # noqa: E402  (links libtforge_hip.so)

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _act(activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    return code


# ---- norm -----------------------------------------------------------------------


def rms_norm(x, weight, residual=None, eps=1e-6, quantize=False):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    Returns (y, h), h None without a residual; with quantize=True (q, scale, h): y in
    8 bits (float8_e4m3fn) with one scale a row, y ~ q * scale.  x is float32,
    bfloat16 or float16, the weight of x's type or float32.
    """
    got = _C.rms_norm(x, weight, residual, eps, True if quantize else False)
    if got is not None:
        return got
    if quantize:
        raise ValueError("the 8-bit output has no gradient: call rms_norm under torch.no_grad(), or on detached tensors")
    y, h = _RmsNorm.apply(x, weight, residual, eps)
    return y, (None if residual is None else h)


def quantize_rows(x):
    """(q, scale): x in 8 bits (float8_e4m3fn) with one float32 scale a row of the last dimension, x ~ q * scale."""
    return _C.quantize_rows(x)


def rms_norm_grad(dy, h, weight, eps=1e-6, dh=None):
    """(dx, dweight) of rms_norm from the gradient dy of y and the norm's input h (x + residual).

    dh: the gradient that reaches h past the norm, added to dx; dx is the residual's gradient too.
    """
    return _C.rms_norm_grad(dy, h, weight, eps, dh)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        with torch.no_grad():
            y, h = rms_norm(x, weight, residual, eps)
        ctx.eps, ctx.added = eps, None if residual is None else residual.shape
        ctx.save_for_backward(x if residual is None else h, weight)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        if dy is None:  # h's alone, past the norm
            dx, dw = dh, None
        else:
            dx, dw = rms_norm_grad(dy.contiguous(), h, weight, ctx.eps, None if dh is None else dh.contiguous())
        if ctx.added is None:
            return dx, dw, None, None
        # A view would be another tensor on dx's memory, and both could become a leaf's grad.
        return dx, dw, dx if ctx.added == dx.shape else dx.reshape(ctx.added).clone(), None


# ---- products ---------------------------------------------------------------------


def linear(x, w, bias=None, activation="none", residual=None, keep=False, x_scale=None, w_scale=None, out_dtype=None,
           tile=0, splits=0, grad_terms=0):
    """z = x @ w + bias;  out = activation(z) + residual, rounded once.

    x (..., k) and w (k, n) are bfloat16 or float16; w may lie row by row or column by
    column (w = weight.t() of an n x k weight).  Or both are float8_e4m3fn, w column by
    column, with x_scale (one a row) and w_scale (one a column), and out_dtype
    (bfloat16 unless given).  bias is of the output's type or float32.  activation:
    "none", "relu", "gelu" (by the normal distribution), "silu".  Returns out, or
    (out, z) with keep=True; both are differentiable.  tile and splits override the choice by sizes
    (tf_linear_args_t in tforge_hip.h); grad_terms is linear_grad's terms under autograd.
    """
    got = _C.linear(x, w, bias, _act(activation), residual, True if keep else False, x_scale, w_scale, out_dtype, tile,
                    splits)
    if got is not None:
        return got
    out, z = _Linear.apply(x, w, bias, residual, activation, keep, tile, splits, grad_terms)
    return (out, z) if keep else out


def linear_grad(dy, x, w, z=None, activation="none", bias_dtype=None, want_dx=True, want_dw=True, tile=0, splits=0,
                terms=0):
    """(dx, dw, dbias) of linear from the gradient dy of its output and the kept pre-activation z.

    dw lies in memory as w does.  dbias comes in bias_dtype (x's type or float32), None
    without one; what is not wanted is None.  The residual's gradient is dy itself.
    With gelu and silu the products take dz = dy * activation'(z) rounded to x's type
    (terms=1, an error of sqrt(2) of the results' own rounding) or with what the rounding
    left as a second term (terms=2, twice the time); 0 takes two up to 1.4e8 multiply-adds.
    """
    return _C.linear_grad(dy, x, w, z, _act(activation), bias_dtype, True if want_dx else False,
                          True if want_dw else False, tile, splits, terms)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, keep, tile, splits, terms):
        smooth = activation != "none"
        with torch.no_grad():
            got = linear(x, w, bias, activation, residual, keep=keep or smooth, tile=tile, splits=splits)
        out, z = got if keep or smooth else (got, None)
        ctx.save_for_backward(x, w, z if smooth else None)
        ctx.how = activation, None if bias is None else bias.dtype, tile, splits, terms
        ctx.added = None if residual is None else residual.shape
        ctx.set_materialize_grads(False)
        return out, z if keep else None

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        x, w, z = ctx.saved_tensors
        activation, bias_dtype, tile, splits, terms = ctx.how
        need = ctx.needs_input_grad

        def grads(g, z, activation):
            return linear_grad(g.contiguous(), x, w, z, activation, bias_dtype if need[2] else None, need[0], need[1], tile,
                               splits, terms)

        # A gradient that reaches the kept z past the activation: its own products, added to the output's.
        got = [] if dy is None else [grads(dy, z, activation)]
        got += [] if dz is None else [grads(dz, None, "none")]
        total = (None, None, None) if not got else got[0] if len(got) == 1 else [a if a is None else a + b for a, b in zip(*got)]
        return (*total, dy.reshape(ctx.added) if need[3] and dy is not None else None, None, None, None, None, None)
