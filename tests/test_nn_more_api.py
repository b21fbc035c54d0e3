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
    (dict(kept=1, type=1), "kept = 1"), (dict(kept=2, z=256), "do not keep z in 8 bits"),
    (dict(kept=2, type=1, x_scale=0, w_scale=0, z=0), "z is a null pointer"),
    (dict(kept=2, type=1, x_scale=0, w_scale=0, z=264), "z, kept in 8 bits, is not 16-byte"),
    (dict(kept=2, type=1, x_scale=0, w_scale=0, z=256), "are needed"),
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


# ---- kept in 8 bits -------------------------------------------------------------


def test_keep8_refusals():
    lib, n = _lib.lib(), ctypes.c_longlong()
    for rows, d, bytes_ in ((0, 5, 0), (5, 0, 0), (3, 1, 99), (3, 32, 99), (3, 33, 198), (1 << 30, 1 << 30, (1 << 55) * 33)):
        assert lib.tf_keep8_bytes(rows, d, ctypes.byref(n)) == 0 and n.value == bytes_
    _refused(lib.tf_keep8_bytes(-1, 5, ctypes.byref(n)), "rows = -1")
    _refused(lib.tf_keep8_bytes(1, (1 << 30) + 1, ctypes.byref(n)), "d = 1073741825")
    _refused(lib.tf_keep8_bytes(1, 1, None), "null")
    _refused(lib.tf_keep8(256, 64, 4, 64, 3, 0, 256, None), "type = 3")
    _refused(lib.tf_keep8(256, 63, 4, 64, 1, 0, 256, None), "x: 63 elements")
    _refused(lib.tf_keep8(257, 64, 4, 64, 1, 0, 256, None), "x is not aligned")
    _refused(lib.tf_keep8(256, 64, 4, 64, 1, 2, 256, None), "positive = 2")
    _refused(lib.tf_keep8(256, 64, 4, 64, 1, 0, 264, None), "kept, kept in 8 bits, is not 16-byte aligned")
    _refused(lib.tf_keep8(256, 64, 4, 64, 1, 0, None, None), "kept is a null pointer")
    _refused(lib.tf_restore8(256, 4, 64, 4, 256, 64, None), "type = 4")
    _refused(lib.tf_restore8(256, 4, 64, 1, 256, 32, None), "x: 32 elements")
    _refused(lib.tf_restore8(None, 4, 64, 1, 256, 64, None), "kept is a null pointer")
    assert lib.tf_keep8(None, 0, 0, 64, 1, 0, None, None) == lib.tf_restore8(None, 4, 0, 1, None, 0, None) == 0
    base = dict(dy=256, x=256, w=256, z=256, dx=256, dw=256, workspace=256, workspace_bytes=1 << 30, dy_ld=32, w_ld=32, dx_ld=64,
                dw_ld=32, m=8, n=32, k=64, type=1, bias_type=1, act=2)
    for change, words in ((dict(kept=4), "kept = 4"), (dict(kept=3, x=264), "x, kept in 8 bits"), (dict(kept=3, z=0), "z is a null pointer"),
                          (dict(kept=1), "z: 0 elements"), (dict(kept=2), "x: 0 elements"), (dict(kept=3, workspace_bytes=16), "are needed")):
        _refused(lib.tf_linear_grad(ctypes.byref(_lib.LinearGradArgs(**{**base, **change})), None), words)
    a = dict(dy=256, h=256, weight=256, dx=256, dweight=256, dy_ld=64, dx_ld=64, rows=4, d=64, type=1, weight_type=1, workspace=256,
             workspace_bytes=1 << 20)
    for change, words in ((dict(kept=2), "kept = 2"), (dict(kept=1, h=264), "h, kept in 8 bits"), (dict(kept=0), "h: 0 elements")):
        _refused(lib.tf_rms_norm_grad(ctypes.byref(_lib.RmsNormGradArgs(**{**a, **change})), None), words)


def test_products_that_keep_z_launch(without_gpu):  # noqa: F811
    """Whichever of their launches fails, the call says so; no launch has 2^32 threads."""
    without_gpu("""
def kept(m, n, k, order, tile=0, splits=0, fail=-1):
    a = _lib.LinearArgs(x=256, w=256, out=256, z=256, x_ld=k, w_ld=k if order else n, out_ld=n, m=m, n=n, k=k, w_order=order, type=1, out_type=1,
                        workspace=256, tile=tile, splits=splits, kept=2, act=1)
    size = ctypes.c_longlong()
    assert lib.tf_linear_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    stub.arm(fail)
    return lib.tf_linear(ref(a), None)
big = 1 << 30
for order in (0, 1):
    for m, n, k in ((big, 1, 1), (big, 64, 64), (1, big, 8), (64, 1 << 28, 7), (1 << 20, 1 << 16, 8)):
        for tile in (0, 1, 2, 3, 4, 5):
            assert kept(m, n, k, order, tile) == 0, (m, n, k, tile)
    for m, n, k in ((4096, 4096, 512), (16, 512, 4096), (777, 1111, 333), (300, 300, 8000)):
        for tile, splits in ((0, 0), (3, 2), (4, 1)):
            assert kept(m, n, k, order, tile, splits) == 0
            for i in range(stub.arm(-1)):
                assert kept(m, n, k, order, tile, splits, i) == -5, (m, n, k, tile, i)
""")


def test_kept_python_refusals():
    h, w, v = (torch.zeros(n, dtype=torch.bfloat16) for n in ((4, 40), (40, 16), (40,)))
    dy, half = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(4, 16, dtype=torch.float16)
    kept = lambda m, n, t=torch.bfloat16, more=0: nn.Kept8(torch.zeros(m * (-(-n // 32)) * 33 + more, dtype=torch.uint8), (m, n), t)  # noqa: E731
    for call, error, words in [
            (lambda: nn.keep8(h), ValueError, "not on a GPU"),
            (lambda: nn.keep8(h.int()), TypeError, "x is Int"),
            (lambda: nn.keep8(h.t()), ValueError, "next to each other"),
            (lambda: nn.keep8(h.clone().requires_grad_()), ValueError, "no gradient"),
            (lambda: kept(4, 40).restore(), ValueError, "not on a GPU"),
            (lambda: kept(4, 40, more=1).restore(), ValueError, "is not 264 contiguous bytes"),
            (lambda: nn.Kept8(kept(4, 40).data, (4, 40), torch.int8).restore(), TypeError, "not Char"),
            (lambda: nn.Kept8(kept(4, 40).data.char(), (4, 40), torch.bfloat16).restore(), TypeError, "kept is Char"),
            (lambda: nn.Kept8(kept(4, 40).data, (-4, 40), torch.bfloat16).restore(), ValueError, "out of range"),
            (lambda: nn.Kept8(kept(4, 40).data, (), torch.bfloat16).restore(), ValueError, "no dimension"),
            (lambda: nn.linear_grad(dy, kept(4, 40), w), ValueError, "not on a GPU"),
            (lambda: nn.linear_grad(dy, kept(4, 39), w), ValueError, "not rows of 40"),
            (lambda: nn.linear_grad(dy, kept(5, 40), w), ValueError, "x, 4 x 40 kept in 8 bits"),
            (lambda: nn.linear_grad(dy, kept(4, 40, torch.float16), w), TypeError, "x was torch.float16"),
            (lambda: nn.linear_grad(half, kept(4, 40), w), TypeError, "x was torch.bfloat16"),
            (lambda: nn.linear_grad(dy, kept(4, 40).data, w), TypeError, "x is Byte"),
            (lambda: nn.linear_grad(dy, h, w, kept(4, 17), "gelu"), ValueError, "not rows of 16"),
            (lambda: nn.linear_grad(dy, kept(4, 40), w, None, "gelu"), ValueError, "keep=True"),
            (lambda: nn.linear_grad(dy, kept(4, 40), w[0]), ValueError, "not k x n"),
            (lambda: nn.linear_grad(dy, kept(4, 40), w, kept(4, 16).data, "gelu"), TypeError, "a tensor of bytes"),
            (lambda: nn.linear_grad(dy, h, w, kept(4, 16).data, "gelu"), TypeError, "z is Byte"),
            (lambda: nn.linear_grad(dy, kept(4, 40), w.clone().requires_grad_()), ValueError, "no gradient"),
            (lambda: nn.rms_norm_grad(h, kept(4, 40), v), ValueError, "not on a GPU"),
            (lambda: nn.rms_norm_grad(h, kept(4, 33), v), ValueError, "not rows of 40"),
            (lambda: nn.rms_norm_grad(h, kept(3, 40), v), ValueError, "kept in 8 bits"),
            (lambda: nn.rms_norm_grad(h.half(), kept(4, 40), v.half()), TypeError, "h was torch.bfloat16"),
            (lambda: nn.rms_norm_grad(h, kept(4, 40).data, v), TypeError, "h is Byte")]:
        with pytest.raises(error, match=words):
            call()


def test_keeping_extreme_sizes_launches(without_gpu):  # noqa: F811
    without_gpu("""
big = 1 << 30
for rows, d in ((1, big), (big, 1), (big, 33), (1 << 22, 20000), (1 << 15, big)):
    for ld in (d, d + 8):
        assert lib.tf_keep8(256, ld, rows, d, 1, 0, 256, None) == 0 and lib.tf_restore8(256, rows, d, 1, 256, ld, None) == 0, (rows, d)
    if rows * d < 1 << 40:
        a = _lib.RmsNormGradArgs(dy=256, h=256, weight=256, dx=256, dweight=256, dy_ld=d, dx_ld=d, rows=rows, d=d, type=1, weight_type=1,
                                 workspace=256, workspace_bytes=1 << 60, kept=1)
        assert lib.tf_rms_norm_grad(ref(a), None) == 0
def grad8(m, n, k, order, act):
    a = _lib.LinearGradArgs(dy=256, x=256, w=256, z=256, dx=256, dw=256, dbias=256, workspace=256, dy_ld=n, w_ld=k if order else n,
                            dx_ld=k, dw_ld=k if order else n, m=m, n=n, k=k, w_order=order, type=1, bias_type=1, act=act, kept=3)
    size = ctypes.c_longlong()
    assert lib.tf_linear_grad_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    return lib.tf_linear_grad(ref(a), None)
for m, n, k in ((1, 1 << 26, 8), (64, big, 64), (big, 9, 8), (big, 1, 1), (1, 1, big), (64, 8, 1 << 27), (4096, 8, 1 << 22)):
    for order in (0, 1):
        for act in (0, 1, 2):
            assert grad8(m, n, k, order, act) == 0, (m, n, k, order, act)
""")


# ---- the loss over a vocabulary ---------------------------------------------------


def _xent(**kw):
    base = dict(x=256, w=256, target=256, loss=256, lse=256, workspace=256, workspace_bytes=1 << 40, x_ld=64, w_ld=100, m=8, n=100, k=64,
                ignore=-100, type=1)
    return ctypes.byref(_lib.LinearXentArgs(**{**base, **kw}))


def _xent_grad(**kw):
    base = dict(x=256, w=256, target=256, lse=256, dloss=256, dx=256, dw=256, workspace=256, workspace_bytes=1 << 40, x_ld=64, w_ld=100,
                dx_ld=64, dw_ld=100, m=8, n=100, k=64, ignore=-100, type=1, dloss_rows=1)
    return ctypes.byref(_lib.LinearXentGradArgs(**{**base, **kw}))


@pytest.mark.parametrize("change,words", [
    (dict(type=0), "type = 0"), (dict(type=3), "type = 3"), (dict(w_order=2), "w_order = 2"), (dict(n=0), "no class"), (dict(m=-1), "m = -1"),
    (dict(k=(1 << 30) + 1), "k = 1073741825"), (dict(x=0), "x is a null"), (dict(w=0), "w is a null"), (dict(target=0), "target is null"),
    (dict(target=260), "target is null or not aligned"), (dict(loss=0), "loss is a null"), (dict(lse=0), "lse is null"), (dict(lse=260), "lse is null or not aligned"),
    (dict(x_ld=63), "x: 63"), (dict(w_ld=99), "w: 99"), (dict(w_order=1, w_ld=63), "w: 63"), (dict(workspace=0), "workspace is null"),
    (dict(workspace=264), "not 16-byte aligned"), (dict(sum=258), "sum is not aligned"), (dict(mean=258), "mean is not aligned"),
    (dict(count=258), "count is not aligned"), (dict(m=1 << 30, n=1 << 27, w_ld=1 << 27), "are too many"), (dict(workspace_bytes=16), "are needed"), (dict(x=257), "x is not aligned")])
def test_xent_refusals(change, words):
    _refused(_lib.lib().tf_linear_xent(_xent(**change), None), words)


@pytest.mark.parametrize("change,words", [
    (dict(type=4), "type = 4"), (dict(n=0), "no class"), (dict(dloss=0), "dloss is a null"), (dict(lse=0), "lse is null"), (dict(lse=260), "lse is null or not aligned"),
    (dict(dloss_rows=2), "dloss_rows = 2"), (dict(target=0), "target is null"), (dict(dx_ld=63), "dx: 63"), (dict(dw_ld=99), "dw: 99"),
    (dict(count=258), "count is not aligned"), (dict(workspace_bytes=16), "are needed"), (dict(m=(1 << 30) + 1), "m = 1073741825")])
def test_xent_grad_refusals(change, words):
    _refused(_lib.lib().tf_linear_xent_grad(_xent_grad(**change), None), words)
    lib, n = _lib.lib(), ctypes.c_longlong()
    assert lib.tf_linear_xent(None, None) == lib.tf_linear_xent_grad(None, None) == -4
    assert lib.tf_linear_xent_workspace(None, ctypes.byref(n)) == lib.tf_linear_xent_grad_workspace(_xent_grad(), None) == -4


def test_xent_python_refusals():
    h, w, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    one, dl, rows = torch.ones(()), torch.zeros(4), torch.zeros(4, dtype=torch.float64)
    for call, error, words in [
            (lambda: nn.linear_cross_entropy(h, w, t), ValueError, "not on a GPU"),
            (lambda: nn.linear_cross_entropy(h, w, t, reduction="max"), ValueError, "not one of none, sum, mean"),
            (lambda: nn.linear_cross_entropy(h.float(), w.float(), t), TypeError, "x is Float"),
            (lambda: nn.linear_cross_entropy(h, w.half(), t), TypeError, "w is Half"),
            (lambda: nn.linear_cross_entropy(h, w, t.int()), TypeError, "target is Int"),
            (lambda: nn.linear_cross_entropy(h, w, t[:3]), ValueError, "target is not"),
            (lambda: nn.linear_cross_entropy(h, w, t[None]), ValueError, "target is not"),
            (lambda: nn.linear_cross_entropy(h, w, t.repeat(2)[::2]), ValueError, "target is not"),
            (lambda: nn.linear_cross_entropy(h, w[:4], t), ValueError, "not 8 x n"),
            (lambda: nn.linear_cross_entropy(h, w[:, :0], t), ValueError, "not on a GPU|no class"),
            (lambda: nn.linear_cross_entropy(h.clone().requires_grad_(), w, t), ValueError, "not on a GPU"),
            (lambda: nn.linear_cross_entropy(h.clone().requires_grad_(), w, t[:3]), ValueError, "target is not"),
            (lambda: nn.linear_cross_entropy_grad(one, h, w, t, rows), ValueError, "not on a GPU"),
            (lambda: nn.linear_cross_entropy_grad(dl[:3], h, w, t, rows), ValueError, "dloss is not"),
            (lambda: nn.linear_cross_entropy_grad(one.double(), h, w, t, rows), TypeError, "dloss is Double"),
            (lambda: nn.linear_cross_entropy_grad(one, h, w, t, rows[:2]), ValueError, "lse is not"),
            (lambda: nn.linear_cross_entropy_grad(one, h, w, t, rows, dl), ValueError, "count is not one"),
            (lambda: nn.linear_cross_entropy_grad(one, h, w, t, dl), TypeError, "lse is Float"),
            (lambda: nn.linear_cross_entropy_grad(one, h, w.clone().requires_grad_(), t, rows), ValueError, "no gradient")]:
        with pytest.raises(error, match=words):
            call()


def test_xent_struct_layouts_match_c(tmp_path):
    import subprocess
    header = _lib.PKG.parent / "include" / "tforge_hip.h"
    structs = {"tf_linear_xent_args_t": _lib.LinearXentArgs, "tf_linear_xent_grad_args_t": _lib.LinearXentGradArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        lines += [f'  printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    (tmp_path / "sizes.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", str(tmp_path / "sizes.c"), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True).stdout.split()]
    want = [v for py in structs.values() for v in [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]]
    assert got == want


XENT = """
def xent(m, n, k, order, type=1, fail=None):
    a = _lib.LinearXentArgs(x=256, w=256, target=256, loss=256, lse=256, mean=256, count=256, workspace=256, x_ld=k, w_ld=k if order else n,
                            m=m, n=n, k=k, w_order=order, type=type, ignore=-100)
    size = ctypes.c_longlong()
    assert lib.tf_linear_xent_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    if fail is not None: stub.arm(fail)
    return lib.tf_linear_xent(ref(a), None)
def xent_grad(m, n, k, order, type=1, fail=None):
    a = _lib.LinearXentGradArgs(x=256, w=256, target=256, lse=256, dloss=256, count=256, dx=256, dw=256, workspace=256, x_ld=k,
                                w_ld=k if order else n, dx_ld=k, dw_ld=k if order else n, m=m, n=n, k=k, w_order=order, type=type, ignore=-100)
    size = ctypes.c_longlong()
    assert lib.tf_linear_xent_grad_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    if fail is not None: stub.arm(fail)
    return lib.tf_linear_xent_grad(ref(a), None)
"""


def test_failed_launches_of_the_loss(without_gpu):  # noqa: F811
    """Whichever of its launches fails, the call says so."""
    without_gpu(XENT + """
for m, n, k in ((1, 5, 64), (70, 1001, 333), (4096, 4096, 4096), (20000, 40000, 72), (1, 70000, 2048)):
    for order in (0, 1):
        for type in (1, 2):
            for call in (xent, xent_grad):
                assert call(m, n, k, order, type, -1) == 0
                for i in range(stub.arm(-1)):
                    assert call(m, n, k, order, type, i) == -5, (call, m, n, k, order, i)
""")


def test_losses_of_extreme_sizes_launch(without_gpu):  # noqa: F811
    """One side as long as memory may hold: no launch has 2^32 threads."""
    without_gpu(XENT + """
big = 1 << 30
for m, n, k in ((1, big, 8), (big, 1, 1), (big, 9, 8), (1 << 24, 1 << 18, 64), (1 << 20, 1 << 20, 1000), (1, 1, big), (64, 1 << 28, 7), (0, 100, 64)):
    for order in (0, 1):
        for type in (1, 2):
            assert xent(m, n, k, order, type) == 0, (m, n, k, order)
            assert xent_grad(m, n, k, order, type) == 0, (m, n, k, order)
""")


def test_second_order_with_constant_gradients():
    """A sum's gradient is a constant: a penalty on what it gives is refused all the same."""
    from test_nn_autograd import Plain
    plain, native = Plain(), nn._C
    nn._C = plain
    try:
        x, w, w1 = (torch.randn(s, dtype=torch.float64, requires_grad=True) for s in ((6, 8), (8,), (8, 5)))
        for loss, of in ((nn.rms_norm(x, w)[0].sum(), w), (nn.linear(x, w1, None, "gelu").sum(), w1), (nn.linear(x, w1).sum(), x)):
            g, = torch.autograd.grad(loss, of, create_graph=True)
            with pytest.raises(RuntimeError, match="twice"):
                (loss.detach() + g.pow(2).sum()).backward()
    finally:
        nn._C = native
