"""The residual block's operators without a GPU: the argument structs' layout, and
what the C ABI and the Python functions refuse (before any device work)."""

import ctypes
import os
import pathlib
import subprocess
import sys

import pytest
import torch

from tensorforge_amd import _lib
from tensorforge_amd import tforge_nn as nn

F8 = torch.float8_e4m3fn
HEADER = pathlib.Path(__file__).resolve().parent.parent / "include" / "tforge_hip.h"
STRUCTS = {"tf_rms_norm_args_t": _lib.RmsNormArgs, "tf_rms_norm_grad_args_t": _lib.RmsNormGradArgs,
           "tf_linear_args_t": _lib.LinearArgs, "tf_linear_grad_args_t": _lib.LinearGradArgs}


def test_struct_layouts_match_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    (tmp_path / "sizes.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", str(tmp_path / "sizes.c"), "-o", str(tmp_path / "sizes")], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True).stdout.splitlines())
    for cname, py in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(py, f).offset, (cname, f)


def test_kernels_do_not_spill():
    import json
    res = json.loads((_lib.PKG / "kernel_resources.json").read_text())
    ours = {n: r for n, r in res.items() if "4tfnn" in n}
    for kernel in ("gemm_wide_kernel", "gemm_tile_kernel", "gemm_rows_kernel", "gemm_pair_kernel", "gemm_join_kernel",
                   "pack_kernel", "act_slope_kernel", "rms_norm_kernel", "rms_norm_grad_kernel", "share_sum_kernel"):
        assert any(kernel in n for n in ours), kernel
    for name, r in ours.items():
        assert r["scratch_bytes"] == 0 and r["vgpr_spill"] == 0, name


def _refused(call, args, words):
    assert call(ctypes.byref(args), None) == -4  # TF_E_ARG
    assert words in _lib.lib().tf_last_error().decode(), _lib.lib().tf_last_error()


def _linear(**kw):
    base = dict(x=256, w=256, out=256, x_ld=64, w_ld=32, out_ld=32, m=8, n=32, k=64, type=1, out_type=1)
    return _lib.LinearArgs(**{**base, **kw})


@pytest.mark.parametrize("change,words", [
    (dict(type=0), "type = 0"), (dict(out_type=2), "out_type = 2"), (dict(act=4), "act = 4"), (dict(m=-1), "m = -1"),
    (dict(k=(1 << 30) + 1), "k = 1073741825"), (dict(x=0), "x is a null pointer"), (dict(out=0), "out is a null pointer"),
    (dict(x=257), "x is not aligned"), (dict(x_ld=63), "x: 63 elements between rows of 64"),
    (dict(w_ld=31), "w: 31 elements between rows of 32"), (dict(w_order=1), "w: 32 elements between rows of 64"),
    (dict(w_order=2), "w_order = 2"), (dict(out_ld=31), "out: 31"), (dict(z=256, z_ld=8), "z: 8"),
    (dict(residual=256, residual_ld=3), "residual: 3"), (dict(bias=256, bias_type=2), "bias_type = 2"),
    (dict(x_scale=256), "scales belong to 8-bit"), (dict(type=3), "8-bit weights"),
    (dict(type=3, w_order=1, w_ld=64), "x_scale is a null pointer"), (dict(tile=6), "tile = 6"),
    (dict(splits=65), "splits = 65"), (dict(workspace=8, workspace_bytes=64), "not 16-byte aligned"),
    (dict(x_ld=1 << 41), "are too many"),
])
def test_linear_refusals(change, words):
    _refused(_lib.lib().tf_linear, _linear(**change), words)


@pytest.mark.parametrize("change,words", [
    (dict(type=3), "type = 3"), (dict(dy=0), "dy is a null pointer"), (dict(act=1), "z is a null pointer"),
    (dict(x=0), "x is a null pointer"), (dict(w=0), "w is a null pointer"), (dict(dx_ld=63), "dx: 63"),
    (dict(dw_ld=31), "dw: 31"), (dict(bias_type=3), "bias_type = 3"), (dict(act=1, z=256, z_ld=32, workspace_bytes=16), "bytes, "),
    (dict(act=1, z=256, z_ld=32, workspace=0), "workspace is null"), (dict(n=-2), "n = -2"),
])
def test_linear_grad_refusals(change, words):
    base = dict(dy=256, x=256, w=256, dx=256, dw=256, dbias=256, workspace=256, workspace_bytes=1 << 30, dy_ld=32, x_ld=64,
                w_ld=32, dx_ld=64, dw_ld=32, m=8, n=32, k=64, type=1, bias_type=1)
    _refused(_lib.lib().tf_linear_grad, _lib.LinearGradArgs(**{**base, **change}), words)


@pytest.mark.parametrize("change,words", [
    (dict(type=3), "type = 3"), (dict(weight_type=2), "weight_type = 2"), (dict(y_type=2), "y_type = 2"),
    (dict(rows=-1), "rows = -1"), (dict(weight=0), "weight is a null pointer"), (dict(y=0), "y is a null pointer"),
    (dict(y_type=3), "scale is a null pointer"), (dict(residual=256, residual_ld=64), "h is a null pointer"),
    (dict(h=256, h_ld=64), "h without a residual"), (dict(x_ld=8), "x: 8"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=258, type=0, weight_type=0, y_type=0), "x is not aligned"),
])
def test_rms_norm_refusals(change, words):
    base = dict(x=256, weight=256, y=256, x_ld=64, y_ld=64, rows=4, d=64, type=1, weight_type=1, y_type=1, eps=1e-6)
    _refused(_lib.lib().tf_rms_norm, _lib.RmsNormArgs(**{**base, **change}), words)


def test_other_refusals():
    lib = _lib.lib()
    assert lib.tf_quantize_rows(256, 8, 4, 64, 1, 256, 64, 256, None) == -4
    assert lib.tf_quantize_rows(256, 64, 4, 64, 3, 256, 64, 256, None) == -4
    assert lib.tf_rms_norm(None, None) == lib.tf_linear(None, None) == lib.tf_linear_grad(None, None) == -4
    n = ctypes.c_longlong()
    assert lib.tf_rms_norm_grad_workspace(-1, 8, ctypes.byref(n)) == -4
    assert lib.tf_linear_workspace(ctypes.byref(_linear(m=-1)), ctypes.byref(n)) == -4
    a = dict(dy=256, h=256, weight=256, dx=256, dweight=256, dy_ld=64, h_ld=64, dx_ld=64, rows=4, d=64, type=1,
             weight_type=1, workspace=256, workspace_bytes=4)
    _refused(lib.tf_rms_norm_grad, _lib.RmsNormGradArgs(**a), "bytes, ")


def test_workspace_sizes():
    lib, n = _lib.lib(), ctypes.c_longlong()
    assert lib.tf_linear_workspace(ctypes.byref(_linear(m=8192, n=8192, k=8192)), ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tf_linear_workspace(ctypes.byref(_linear(m=5, n=7, k=512, tile=3, splits=2)), ctypes.byref(n)) == 0
    assert n.value == 2 * 5 * 8 * 4
    assert lib.tf_rms_norm_grad_workspace(0, 64, ctypes.byref(n)) == 0 and n.value == 0


def test_python_refusals():
    """On CPU tensors: what is wrong with the tensors comes first, the missing GPU last."""
    h = torch.zeros(4, 8, dtype=torch.bfloat16)
    w, v = torch.zeros(8, 16, dtype=torch.bfloat16), torch.zeros(16)
    for call, error, words in [
            (lambda: nn.linear(h, w), ValueError, "not on a GPU"),
            (lambda: nn.rms_norm(h, h[0]), ValueError, "not on a GPU"),
            (lambda: nn.rms_norm_grad(h, h, h[0]), ValueError, "not on a GPU"),
            (lambda: nn.linear_grad(h[:, :1].expand(4, 16).contiguous(), h, w), ValueError, "not on a GPU"),
            (lambda: nn.quantize_rows(h), ValueError, "not on a GPU"),
            (lambda: nn.quantize_rows(None), TypeError, "x is not a tensor"),
            (lambda: nn.rms_norm(h.double(), h[0]), TypeError, "x is Double"),
            (lambda: nn.rms_norm(h, h[0].half()), TypeError, "weight is Half"),
            (lambda: nn.rms_norm(h, w[0]), ValueError, "not a contiguous vector of 8"),
            (lambda: nn.rms_norm(h, h[0], residual=w), ValueError, "residual is 8 x 16, not 4 x 8"),
            (lambda: nn.rms_norm(h.requires_grad_(False).clone().requires_grad_(), h[0], quantize=True), ValueError, "gradient"),
            (lambda: nn.linear(h.float(), w.float()), TypeError, "x is Float"),
            (lambda: nn.linear(h, w.half()), TypeError, "w is Half"),
            (lambda: nn.linear(h, h), ValueError, "not 8 x n"),
            (lambda: nn.linear(h, w, h[0]), ValueError, "bias is not"),
            (lambda: nn.linear(h, w, activation="tanh"), ValueError, "not one of none, relu, gelu, silu"),
            (lambda: nn.linear(h, w, residual=h), ValueError, "residual is 4 x 8, not 4 x 16"),
            (lambda: nn.linear(h, w, x_scale=v), ValueError, "scales belong"),
            (lambda: nn.linear(h, w, out_dtype=torch.float16), TypeError, "keep x's type"),
            (lambda: nn.linear(h.to(F8), w.to(F8), x_scale=v[:4], w_scale=v), ValueError, "column by column"),
            (lambda: nn.linear(h.to(F8), w.to(F8).t().contiguous().t()), ValueError, "needs x_scale"),
            (lambda: nn.linear(torch.zeros(8, 4, dtype=torch.bfloat16).t(), w), ValueError, "next to each other"),
            (lambda: nn.linear(h[0].expand(4, 8), w), ValueError, "rows overlap"),
            (lambda: nn.linear(h, torch.zeros(16, 32, dtype=torch.bfloat16)[::2, ::2]), ValueError, "neither its rows"),
            (lambda: nn.linear(torch.zeros(2, 3, 9, dtype=torch.bfloat16)[:, :2, :8], w), ValueError, "one run of rows"),
            (lambda: nn.linear_grad(w[:4], h, w, activation="gelu"), ValueError, "keep=True"),
            (lambda: nn.linear_grad(w[:4], h, w, bias_dtype=torch.float64), TypeError, "bias_dtype is Double")]:
        with pytest.raises(error, match=words):
            call()


# Stands in for HIP's launches in a process without a GPU: refuses what HIP refuses (2^32 threads or more along a side)
# and the launch that arm() names, and keeps the last error as HIP does.  arm() returns the launches since the last.
STUB = """
#include <stddef.h>
typedef struct { unsigned x, y, z; } dim3;
static int last, launches, fail = -1;
static dim3 grid, block;
static size_t shared;
static void *stream;
int arm(int fail_at) { int n = launches; launches = 0; last = 0; fail = fail_at; return n; }
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t n, void *s) { grid = g; block = b; shared = n; stream = s; return 0; }
int __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *n, void **s) { *g = grid; *b = block; *n = shared; *s = stream; return 0; }
int hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t n, void *s) {
  int bad = (unsigned long long)g.x * b.x >> 32 || (unsigned long long)g.y * b.y >> 32 || launches == fail;
  ++launches;
  if (bad) last = 9;
  return bad ? 9 : 0;
}
int hipGetLastError(void) { int e = last; last = 0; return e; }
"""

HEAD = """
import ctypes
from tensorforge_amd import _lib
lib, stub, ref = _lib.lib(), ctypes.CDLL(None), ctypes.byref

def norm(d, rows, residual=0, y_type=1):
    a = _lib.RmsNormArgs(x=256, weight=256, y=256, scale=256, residual=residual, h=residual, x_ld=d, y_ld=d, residual_ld=d, h_ld=d,
                         rows=rows, d=d, type=1, weight_type=1, y_type=y_type)
    return lib.tf_rms_norm(ref(a), None)

def norm_grad(d, rows):
    a = _lib.RmsNormGradArgs(dy=256, h=256, weight=256, dx=256, dweight=256, dy_ld=d, h_ld=d, dx_ld=d, rows=rows, d=d, type=1,
                             weight_type=1, workspace=256, workspace_bytes=1 << 60)
    return lib.tf_rms_norm_grad(ref(a), None)

def linear(m, n, k, order, type=1, **kw):
    a = _lib.LinearArgs(x=256, w=256, out=256, x_scale=256 * (type == 3), w_scale=256 * (type == 3), x_ld=k, w_ld=k if order else n, out_ld=n,
                        m=m, n=n, k=k, w_order=order, type=type, out_type=1, workspace=256, **kw)
    size = ctypes.c_longlong()
    assert lib.tf_linear_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    return lib.tf_linear(ref(a), None)

def linear_grad(m, n, k, order, act=0, **kw):
    a = _lib.LinearGradArgs(dy=256, x=256, w=256, z=256, dx=256, dw=256, dbias=256, workspace=256, dy_ld=n, x_ld=k, z_ld=n,
                            w_ld=k if order else n, dx_ld=k, dw_ld=k if order else n, m=m, n=n, k=k, w_order=order, type=1, bias_type=1,
                            act=act, **kw)
    size = ctypes.c_longlong()
    assert lib.tf_linear_grad_workspace(ref(a), ref(size)) == 0
    a.workspace_bytes = size.value
    return lib.tf_linear_grad(ref(a), None)
"""


@pytest.fixture(scope="module")
def without_gpu(tmp_path_factory):
    """Runs code, after HEAD, in a process with the stub before HIP."""
    at = tmp_path_factory.mktemp("stub")
    (at / "stub.c").write_text(STUB)
    subprocess.run(["gcc", "-shared", "-fPIC", str(at / "stub.c"), "-o", str(at / "stub.so")], check=True)
    preload = " ".join([str(at / "stub.so"), os.environ.get("LD_PRELOAD", "")]).strip()
    env = {**os.environ, "LD_PRELOAD": preload, "HIP_VISIBLE_DEVICES": "-1", "ROCR_VISIBLE_DEVICES": "-1",
           "PYTHONPATH": str(_lib.PKG.parent)}

    def run(code):
        r = subprocess.run([sys.executable, "-c", HEAD + code], env=env, capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


def test_failed_launches_of_the_norm_gradient(without_gpu):
    """Whichever of its launches fails, the call says so."""
    without_gpu("""
for rows, d in ((4, 64), (4000, 64), (4000, 4000), (5, 4), (70, 20000), (0, 64)):
    stub.arm(-1)
    assert norm_grad(d, rows) == 0
    launches = stub.arm(-1)
    assert 1 <= launches <= 2
    for i in range(launches):
        stub.arm(i)
        assert norm_grad(d, rows) == -5, (rows, d, i)
""")


def test_norms_of_many_rows_launch(without_gpu):
    """No launch has 2^32 threads, up to the largest sizes that fit a memory of 288 GB."""
    without_gpu("""
for rows, d in ((1 << 24, 4), (1 << 30, 1), (1 << 30, 7), (1 << 30, 0), (1 << 30, 64), (1 << 26, 2000), (1 << 22, 20000)):
    for residual in (0, 256):
        for y_type in (1, 3):
            assert norm(d, rows, residual, y_type) == 0, (rows, d)
    assert lib.tf_quantize_rows(256, d, rows, d, 1, 256, d, 256, None) == 0
    assert norm_grad(d, rows) == 0, (rows, d)
""")


def test_products_of_extreme_sizes_launch(without_gpu):
    """One side as long as the header allows: no launch has 2^32 threads."""
    without_gpu("""
big = 1 << 30
sizes = [(1, 1 << 26, 8), (16, 1 << 26, 64), (1, 1 << 27, 8), (64, 1 << 28, 8), (1, big, 1), (3, big, 7), (64, big, 64), (big, 1, 1),
         (big, 9, 8), (big, 64, 64), (big, 64, 8), (big - 63, 8, 16), (100, 1 << 29, 8), (65, big, 9), (1 << 20, 1 << 16, 5), (1, 1, big)]
for m, n, k in sizes:
    for order in (0, 1):
        for tile in (0, 1, 2, 3, 4, 5):
            assert linear(m, n, k, order, tile=tile) == 0, (m, n, k, order, tile)
        for act in (0, 1, 2):
            assert linear_grad(m, n, k, order, act) == 0, (m, n, k, order, act)
        assert linear_grad(m, n, k, order, 2, tile=3, splits=2) == 0, (m, n, k, order)
    assert linear(m, n, k, 1, type=3) == 0 and linear(m, n, k, 1, type=3, tile=3, splits=2) == 0, (m, n, k)
assert norm_grad(big, 1) == 0 and norm_grad(big, 2) == 0
""")


def test_copies_of_short_lines_stay_small():
    """Aligned copies of odd operands take at most four times their memory, or 256 MB."""
    lib, size = _lib.lib(), ctypes.c_longlong()
    for m, n, k in ((1 << 30, 1, 1), (1 << 28, 64, 5), (1 << 26, 300, 3), (1 << 22, 4096, 1), (5, 1 << 28, 7), (4096, 4096, 5)):
        for order in (0, 1):
            for type_ in (1, 3)[:1 + order]:
                for tile in (0, 2):
                    a = _lib.LinearArgs(x=256, w=256, out=256, x_ld=k, w_ld=k if order else n, out_ld=n, m=m, n=n, k=k, w_order=order,
                                        type=type_, out_type=1, tile=tile, splits=1)
                    assert lib.tf_linear_workspace(ctypes.byref(a), ctypes.byref(size)) == 0
                    assert size.value <= max(4 * (m + n) * k * 2, 256 << 20), (m, n, k, order, type_, tile)


def test_terms_refusals():
    base = dict(dy=256, x=256, w=256, dx=256, dw=256, dbias=256, workspace=256, workspace_bytes=1 << 30, dy_ld=32, x_ld=64,
                w_ld=32, dx_ld=64, dw_ld=32, m=8, n=32, k=64, type=1, bias_type=1)
    for terms in (-1, 3):
        _refused(_lib.lib().tf_linear_grad, _lib.LinearGradArgs(**base, terms=terms), f"terms = {terms}")
