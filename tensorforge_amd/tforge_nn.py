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
gradient, autograd runs the gradient calls.

Bad arguments raise ValueError or TypeError before any work; errors of the
library raise RuntimeError with its message.
"""

import ctypes
import functools
import struct

import torch

from tensorforge_amd import _lib

F8 = torch.float8_e4m3fn
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, F8: 3}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _packer(cls):
    """struct.pack for a ctypes structure: several times faster than filling one."""
    code = {ctypes.c_void_p: "P", ctypes.c_longlong: "q", ctypes.c_int: "i", ctypes.c_float: "f"}
    s = struct.Struct("@" + "".join(code[t] for _, t in cls._fields_))
    assert s.size == ctypes.sizeof(cls), cls
    return s.pack


_pack_norm = _packer(_lib.RmsNormArgs)
_pack_norm_grad = _packer(_lib.RmsNormGradArgs)
_pack_linear = _packer(_lib.LinearArgs)
_pack_linear_grad = _packer(_lib.LinearGradArgs)

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _launch(call, device, *args):
    """Calls a library function on `device`'s current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _raw_stream(index))
    if rc < 0:
        _lib.check(rc)


def _rows(t, name):
    """(tensor, rows, row length, elements between rows) of a tensor taken as rows."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f"{name} has no dimension")
        n = t.shape[-1]
        t = t.view(t.numel() // n if n else 0, n)
    m, n = t.shape
    s0, s1 = t.stride()
    if s1 != 1 and n > 1:
        raise ValueError(f"{name}: the elements of a row are not next to each other (strides {tuple(t.stride())})")
    if m > 1 and s0 < n:
        raise ValueError(f"{name}: rows overlap (strides {tuple(t.stride())})")
    return t, m, n, (s0 if m > 1 else n)


def _like(t, name, shape, dtypes, device):
    """_rows of a tensor that has to have this shape (as rows), one of these types and this device."""
    _on(t, name, dtypes, device)
    t, m, n, ld = _rows(t, name)
    if (m, n) != shape:
        raise ValueError(f"{name} is {m} x {n}, not {shape[0]} x {shape[1]}")
    return t, ld


def _on(t, name, dtypes, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is not a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")


def _vector(t, name, n, dtypes, device):
    _on(t, name, dtypes, device)
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} is not a contiguous vector of {n}")
    return t.data_ptr()


def _gpu(t, name, dtypes):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is not a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    if t.device.type != "cuda":
        raise ValueError(f"{name} is on {t.device}, not on a GPU")


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


_NORM_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_HALF_TYPES = (torch.bfloat16, torch.float16)
_F32 = (torch.float32,)


# ---- norm -----------------------------------------------------------------------


def rms_norm(x, weight, residual=None, eps=1e-6, quantize=False):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    Returns (y, h), h None without a residual; with quantize=True (q, scale, h): y in
    8 bits (float8_e4m3fn) with one scale a row, y ~ q * scale.  x is float32,
    bfloat16 or float16, the weight of x's type or float32.
    """
    if _wants_grad(x, weight, residual):
        if quantize:
            raise ValueError("the 8-bit output has no gradient: call rms_norm under torch.no_grad()")
        y, h = _RmsNorm.apply(x, weight, residual, eps)
        return y, (None if residual is None else h)
    _gpu(x, "x", _NORM_TYPES)
    dev, dt = x.device, x.dtype
    x2, m, d, x_ld = _rows(x, "x")
    w = _vector(weight, "weight", d, (dt, torch.float32), dev)
    y = torch.empty(x.shape, dtype=F8 if quantize else dt, device=dev)
    r = r_ld = h_ptr = 0
    h = scale = None
    if residual is not None:
        r2, r_ld = _like(residual, "residual", (m, d), (dt,), dev)
        r = r2.data_ptr()
        h = torch.empty(x.shape, dtype=dt, device=dev)
        h_ptr = h.data_ptr()
    if quantize:
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    args = _pack_norm(x2.data_ptr(), r, w, y.data_ptr(), h_ptr, scale.data_ptr() if quantize else 0, x_ld, r_ld, d, d, m, d,
                      TYPES[dt], TYPES[weight.dtype], 3 if quantize else TYPES[dt], eps)
    _launch(_lib.lib().tf_rms_norm, dev, args)
    return (y, scale, h) if quantize else (y, h)


def quantize_rows(x):
    """(q, scale): x in 8 bits (float8_e4m3fn) with one float32 scale a row of the last dimension, x ~ q * scale."""
    _gpu(x, "x", _NORM_TYPES)
    dev = x.device
    x2, m, d, x_ld = _rows(x, "x")
    q = torch.empty(x.shape, dtype=F8, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    _launch(_lib.lib().tf_quantize_rows, dev, x2.data_ptr(), x_ld, m, d, TYPES[x.dtype], q.data_ptr(), d,
            scale.data_ptr())
    return q, scale


@functools.lru_cache(maxsize=4096)
def _norm_grad_bytes(rows, d):
    n = ctypes.c_longlong()
    _lib.check(_lib.lib().tf_rms_norm_grad_workspace(rows, d, ctypes.byref(n)))
    return n.value


def rms_norm_grad(dy, h, weight, eps=1e-6, dh=None):
    """(dx, dweight) of rms_norm from the gradient dy of y and the norm's input h (x + residual).

    dh: the gradient that reaches h past the norm, added to dx; dx is the residual's gradient too.
    """
    _gpu(h, "h", _NORM_TYPES)
    dev, dt = h.device, h.dtype
    h2, m, d, h_ld = _rows(h, "h")
    dy2, dy_ld = _like(dy, "dy", (m, d), (dt,), dev)
    w = _vector(weight, "weight", d, (dt, torch.float32), dev)
    g = g_ld = 0
    if dh is not None:
        dh2, g_ld = _like(dh, "dh", (m, d), (dt,), dev)
        g = dh2.data_ptr()
    dx = torch.empty(h.shape, dtype=dt, device=dev)
    dw = torch.empty(d, dtype=weight.dtype, device=dev)
    n = _norm_grad_bytes(m, d)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    args = _pack_norm_grad(dy2.data_ptr(), h2.data_ptr(), g, w, dx.data_ptr(), dw.data_ptr(), dy_ld, h_ld, g_ld, d, m, d,
                           TYPES[dt], TYPES[weight.dtype], eps, 0, ws.data_ptr(), n)
    _launch(_lib.lib().tf_rms_norm_grad, dev, args)
    return dx, dw


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        with torch.no_grad():
            y, h = rms_norm(x, weight, residual, eps)
        ctx.eps, ctx.added = eps, residual is not None
        ctx.save_for_backward(h if ctx.added else x, weight)
        if not ctx.added:
            h = y.new_empty(0)
            ctx.mark_non_differentiable(h)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        dx, dw = rms_norm_grad(dy.contiguous(), h, weight, ctx.eps, dh.contiguous() if ctx.added else None)
        return dx, dw, dx if ctx.added else None, None


# ---- products ---------------------------------------------------------------------


def _weights(w, k, dtypes, dev):
    """(order, elements between rows) of a k x n matrix in either memory order."""
    _on(w, "w", dtypes, dev)
    if w.dim() != 2 or w.shape[0] != k:
        raise ValueError(f"w is {tuple(w.shape)}, not {k} x n")
    n, (s0, s1) = w.shape[1], w.stride()
    if (s0 == 1 or k <= 1) and (s1 >= k or n <= 1):
        return 1, (s1 if n > 1 else k)
    if (s1 == 1 or n <= 1) and (s0 >= n or k <= 1):
        return 0, (s0 if k > 1 else n)
    raise ValueError(f"w: neither its rows nor its columns are contiguous (strides {(s0, s1)})")


def _act(activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is not one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[activation]


@functools.lru_cache(maxsize=4096)
def _linear_bytes(m, n, k, t, to, tile, splits):
    args = _lib.LinearArgs(m=m, n=n, k=k, type=t, out_type=to, tile=tile, splits=splits)
    b = ctypes.c_longlong()
    _lib.check(_lib.lib().tf_linear_workspace(ctypes.byref(args), ctypes.byref(b)))
    return b.value


@functools.lru_cache(maxsize=4096)
def _linear_grad_bytes(m, n, k, order, t, act, tile, splits):
    args = _lib.LinearGradArgs(m=m, n=n, k=k, w_order=order, type=t, act=act, tile=tile, splits=splits)
    b = ctypes.c_longlong()
    _lib.check(_lib.lib().tf_linear_grad_workspace(ctypes.byref(args), ctypes.byref(b)))
    return b.value


def linear(x, w, bias=None, activation="none", residual=None, keep=False, x_scale=None, w_scale=None, out_dtype=None,
           tile=0, splits=0):
    """z = x @ w + bias;  out = activation(z) + residual, rounded once.

    x (..., k) and w (k, n) are bfloat16 or float16; w may lie row by row or column by
    column (w = weight.t() of an n x k weight).  Or both are float8_e4m3fn, w column by
    column, with x_scale (one a row) and w_scale (one a column), and out_dtype
    (bfloat16 unless given).  bias is of the output's type or float32.  activation:
    "none", "relu", "gelu" (by the normal distribution), "silu".  Returns out, or
    (out, z) with keep=True.  tile and splits override the choice by sizes
    (tf_linear_args_t in tforge_hip.h).
    """
    _gpu(x, "x", _HALF_TYPES + (F8,))
    dev, dt = x.device, x.dtype
    act = _act(activation)
    if dt == F8:
        to = torch.bfloat16 if out_dtype is None else out_dtype
        if to not in _HALF_TYPES:
            raise TypeError(f"out_dtype is {to}, not {' or '.join(str(d) for d in _HALF_TYPES)}")
    else:
        to = dt
        if out_dtype not in (None, dt):
            raise TypeError(f"out_dtype is {out_dtype}: 16-bit products keep x's type, {dt}")
        if _wants_grad(x, w, bias, residual):
            out, z = _Linear.apply(x, w, bias, residual, activation, keep, tile, splits)
            return (out, z) if keep else out
    x2, m, k, x_ld = _rows(x, "x")
    order, w_ld = _weights(w, k, (dt,), dev)
    n = w.shape[1]
    b = bt = r = r_ld = z_ptr = sx = sw = 0
    if bias is not None:
        b, bt = _vector(bias, "bias", n, (to, torch.float32), dev), TYPES[bias.dtype]
    if residual is not None:
        r2, r_ld = _like(residual, "residual", (m, n), (to,), dev)
        r = r2.data_ptr()
    if dt == F8:
        if order != 1:
            raise ValueError("8-bit weights have to lie column by column: pass weight.t() of an n x k weight")
        if x_scale is None or w_scale is None:
            raise ValueError("an 8-bit product needs x_scale and w_scale")
        sx = _vector(x_scale if x_scale.dim() == 1 else x_scale.reshape(-1), "x_scale", m, _F32, dev)
        sw = _vector(w_scale, "w_scale", n, _F32, dev)
    elif x_scale is not None or w_scale is not None:
        raise ValueError("scales belong to 8-bit products")
    shape = (m, n) if x.dim() == 2 else (*x.shape[:-1], n)
    out = torch.empty(shape, dtype=to, device=dev)
    if keep:
        z = torch.empty(shape, dtype=to, device=dev)
        z_ptr = z.data_ptr()
    t, tt = TYPES[dt], TYPES[to]
    size = _linear_bytes(m, n, k, t, tt, tile, splits)
    ws = torch.empty(size, dtype=torch.uint8, device=dev).data_ptr() if size else 0
    args = _pack_linear(x2.data_ptr(), w.data_ptr(), b, r, sx, sw, out.data_ptr(), z_ptr, ws, size, x_ld, w_ld, r_ld, n, n,
                        m, n, k, order, t, tt, bt, act, tile, splits, 0)
    _launch(_lib.lib().tf_linear, dev, args)
    return (out, z) if keep else out


def linear_grad(dy, x, w, z=None, activation="none", bias_dtype=None, want_dx=True, want_dw=True, tile=0, splits=0):
    """(dx, dw, dbias) of linear from the gradient dy of its output and the kept pre-activation z.

    dw lies in memory as w does.  dbias comes in bias_dtype (x's type or float32), None
    without one; what is not wanted is None.  The residual's gradient is dy itself.
    """
    _gpu(x, "x", _HALF_TYPES)
    dev, dt = x.device, x.dtype
    act = _act(activation)
    x2, m, k, x_ld = _rows(x, "x")
    order, w_ld = _weights(w, k, (dt,), dev)
    n = w.shape[1]
    dy2, dy_ld = _like(dy, "dy", (m, n), (dt,), dev)
    z_ptr = z_ld = 0
    if act:
        if z is None:
            raise ValueError("an activation's gradient needs z: call linear with keep=True")
        z2, z_ld = _like(z, "z", (m, n), (dt,), dev)
        z_ptr = z2.data_ptr()
    if bias_dtype not in (None, dt, torch.float32):
        raise TypeError(f"bias_dtype is {bias_dtype}, not {dt} or torch.float32")
    dx = torch.empty(x.shape, dtype=dt, device=dev) if want_dx else None
    dw = None
    if want_dw:
        dw = torch.empty((n, k), dtype=dt, device=dev).t() if order else torch.empty((k, n), dtype=dt, device=dev)
    db = None if bias_dtype is None else torch.empty(n, dtype=bias_dtype, device=dev)
    size = _linear_grad_bytes(m, n, k, order, TYPES[dt], act, tile, splits)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    args = _pack_linear_grad(dy2.data_ptr(), x2.data_ptr(), w.data_ptr(), z_ptr, dx.data_ptr() if want_dx else 0,
                             dw.data_ptr() if want_dw else 0, 0 if db is None else db.data_ptr(), ws.data_ptr(), size,
                             dy_ld, x_ld, w_ld, z_ld, k, k if order else n, m, n, k, order, TYPES[dt],
                             TYPES[bias_dtype] if db is not None else 0, act, tile, splits)
    _launch(_lib.lib().tf_linear_grad, dev, args)
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, keep, tile, splits):
        smooth = activation != "none"
        with torch.no_grad():
            got = linear(x, w, bias, activation, residual, keep=keep or smooth, tile=tile, splits=splits)
        out, z = got if keep or smooth else (got, None)
        ctx.save_for_backward(x, w, z if smooth else None)
        ctx.how = activation, None if bias is None else bias.dtype, tile, splits
        if z is None or not keep:
            return out, None
        ctx.mark_non_differentiable(z)
        return out, z

    @staticmethod
    def backward(ctx, dy, _):
        x, w, z = ctx.saved_tensors
        activation, bias_dtype, tile, splits = ctx.how
        need = ctx.needs_input_grad
        dy = dy.contiguous()
        dx, dw, db = linear_grad(dy, x, w, z, activation, bias_dtype if need[2] else None, need[0], need[1], tile, splits)
        return dx, dw, db, dy if need[3] else None, None, None, None, None
