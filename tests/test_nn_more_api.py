"""Without a GPU: what the calls with 8-bit integers, kept activations and the loss over
a vocabulary refuse, before any device work, and the launches they make."""

import ctypes

import pytest
import torch

from tensorforge_amd import _lib
from tensorforge_amd import tforge_nn as nn
from test_nn_api import STUB, HEAD, without_gpu  # noqa: F401


def _refused(rc, words):
    assert rc == -4  # TF_E_ARG
    assert words in _lib.lib().tf_last_error().decode(), _lib.lib().tf_last_error()


def _linear(**kw):
    base = dict(x=256, w=256, out=256, x_scale=256, w_scale=256, x_ld=64, w_ld=64, out_ld=32, m=8, n=32, k=64, w_order=1, type=4, out_type=1)
    return ctypes.byref(_lib.LinearArgs(**{**base, **kw}))


@pytest.mark.parametrize("change,words", [
    (dict(k=131072, x_ld=131072, w_ld=131072), "k = 131072"), (dict(out_type=4), "out_type = 4"), (dict(out_type=0), "out_type = 0"),
    (dict(w_order=0), "8-bit weights"), (dict(x_scale=0), "x_scale is a null pointer"), (dict(w_scale=0), "w_scale is a null pointer"),
    (dict(x_ld=63), "x: 63 elements"), (dict(type=5), "type = 5"), (dict(bias=256, bias_type=4), "bias_type = 4"),
])
def test_integer_product_refusals(change, words):
    _refused(_lib.lib().tf_linear(_linear(**change), None), words)
    n = ctypes.c_longlong()
    if "k" in change:
        _refused(_lib.lib().tf_linear_workspace(_linear(**change), ctypes.byref(n)), words)


def test_integer_rows_refusals():
    lib = _lib.lib()
    _refused(lib.tf_quantize_rows_to(256, 64, 4, 64, 1, 256, 64, 1, 256, None), "y_type = 1")
    _refused(lib.tf_quantize_rows_to(256, 64, 4, 64, 4, 256, 64, 4, 256, None), "type = 4")
    _refused(lib.tf_quantize_rows_to(256, 64, 4, 64, 1, 256, 64, 4, 0, None), "scale is a null pointer")
    a = _lib.RmsNormArgs(x=256, weight=256, y=256, x_ld=64, y_ld=64, rows=4, d=64, type=1, weight_type=1, y_type=4, eps=1e-6)
    _refused(lib.tf_rms_norm(ctypes.byref(a), None), "scale is a null pointer")
    g = _lib.LinearGradArgs(dy=256, x=256, w=256, dx=256, dy_ld=32, x_ld=64, w_ld=32, dx_ld=64, m=8, n=32, k=64, type=4, bias_type=1)
    _refused(lib.tf_linear_grad(ctypes.byref(g), None), "type = 4")


def test_integer_python_refusals():
    h, v = torch.zeros(4, 16, dtype=torch.int8), torch.ones(16)
    w = torch.zeros(8, 16, dtype=torch.int8)
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    for call, error, words in [
            (lambda: nn.linear(h, w.t(), x_scale=v[:4], w_scale=v[:8]), ValueError, "not on a GPU"),
            (lambda: nn.linear(h, w.t()), ValueError, "needs x_scale"),
            (lambda: nn.linear(h, w.to(torch.float8_e4m3fn).t(), x_scale=v[:4], w_scale=v[:8]), TypeError, "w is Float8"),
            (lambda: nn.linear(h.to(torch.uint8), w.t(), x_scale=v[:4], w_scale=v[:8]), TypeError, "x is Byte"),
            (lambda: nn.linear(h, w.t().contiguous(), x_scale=v[:4], w_scale=v[:8]), ValueError, "column by column"),
            (lambda: nn.linear(h, w.t(), x_scale=v[:5], w_scale=v[:8]), ValueError, "x_scale is not"),
            (lambda: nn.linear(h, w.t(), x_scale=v[:4], w_scale=v[:8], out_dtype=torch.float32), TypeError, "out_dtype is Float"),
            (lambda: nn.linear(h, w.t(), x_scale=v[:4], w_scale=v[:8].clone().requires_grad_()), ValueError, "no gradient"),
            (lambda: nn.quantize_rows(x, torch.int8), ValueError, "not on a GPU"),
            (lambda: nn.quantize_rows(x, torch.uint8), TypeError, "not Byte"),
            (lambda: nn.quantize_rows(x, None), TypeError, "not a dtype"),
            (lambda: nn.quantize_rows(x.clone().requires_grad_(), torch.int8), ValueError, "no gradient"),
            (lambda: nn.rms_norm(x, v, quantize=torch.int8), ValueError, "not on a GPU"),
            (lambda: nn.rms_norm(x, v, quantize=torch.float16), TypeError, "not Half"),
            (lambda: nn.rms_norm(x.clone().requires_grad_(), v, quantize=torch.int8), ValueError, "no gradient")]:
        with pytest.raises(error, match=words):
            call()


def test_integer_products_of_extreme_sizes_launch(without_gpu):  # noqa: F811
    """No launch has 2^32 threads."""
    without_gpu("""
big = 1 << 30
def linear8(m, n, k, **kw):
    a = _lib.LinearArgs(x=256, w=256, out=256, x_scale=256, w_scale=256, x_ld=k, w_ld=k, out_ld=n, m=m, n=n, k=k, w_order=1, type=4,
                        out_type=1, workspace=256, **kw)
    size = ctypes.c_longlong()
    assert lib.tf_linear_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    return lib.tf_linear(ref(a), None)
for m, n, k in ((1, big, 1), (big, 1, 16), (64, big, 64), (1 << 20, 1 << 16, 5), (1, 1 << 26, 131071), (1, 1, 131071)):
    for tile in (0, 1, 2, 3, 4, 5):
        assert linear8(m, n, k, tile=tile) == 0, (m, n, k, tile)
    assert linear8(m, n, k, tile=3, splits=2) == 0
for rows, d in ((1 << 24, 4), (big, 1), (big, 0), (1 << 22, 20000)):
    assert norm(d, rows, 256, 4) == 0 and lib.tf_quantize_rows_to(256, d, rows, d, 1, 256, d, 4, 256, None) == 0
""")
