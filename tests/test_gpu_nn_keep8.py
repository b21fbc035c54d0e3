"""Activations kept in 8 bits: their bytes against the definition, back again, and the
gradients that take them against 64-bit references at the restored values."""

import ctypes

import numpy as np
import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu"]


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _bytes(x, positive=False):
    """(codes rows x groups x 32, exponents rows x groups) from the definition, in 64 bits."""
    rows, d = x.shape
    groups = -(-d // 32)
    v = np.zeros((rows, groups * 32))
    v[:, :d] = x.double().numpy()
    v = v.reshape(rows, groups, 32)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(top)
    mantissa, exponent = np.frexp(np.where(bad, 1.0, top))
    e = np.maximum(np.where(mantissa * 128 < 127.5, exponent - 7, exponent - 6), -126)
    e = np.where(top == 0, -126, e)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = np.rint(np.ldexp(v, -e[..., None]))
    if positive:
        codes = np.where((v > 0) & (codes < 1), 1, codes)
    codes = np.where(bad[..., None], 0, codes)
    return torch.from_numpy(codes.astype(np.int8)), torch.from_numpy(np.where(bad, 255, e + 127).astype(np.uint8))


def _values(codes, exponents, d):
    unit = np.where(exponents.numpy() == 255, np.nan, np.ldexp(1.0, exponents.numpy().astype(int) - 127))
    return torch.from_numpy((codes.numpy() * unit[..., None]).reshape(codes.shape[0], -1)[:, :d])


def _check_kept(kept, x, positive=False):
    codes, exponents = _bytes(x.cpu().reshape(-1, x.shape[-1]), positive)
    want = torch.cat([codes.reshape(-1).view(torch.uint8), exponents.reshape(-1)])
    assert torch.equal(kept.data.cpu(), want)
    v = _values(codes, exponents, x.shape[-1]).view(x.shape)
    got = kept.restore()
    assert got.dtype == x.dtype == kept.dtype and got.shape == x.shape == kept.shape
    if x.dtype == torch.float16:
        v = torch.where(v.isnan(), v, v.clamp(-65504, 65504))
    v = v.to(x.dtype)
    assert torch.equal(got.cpu().isnan(), v.isnan()) and torch.equal(got.cpu().nan_to_num(), v.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 7, 8, 31, 32, 33, 64, 100, 1111, 4096, 20000])
def test_bytes(d, dtype):
    nn = _nn()
    for rows in (1, 5, 130):
        g = torch.Generator().manual_seed(d + rows)
        x = (torch.randn(rows, d, generator=g) * torch.exp(3 * torch.randn(rows, d, generator=g))).to(dtype)
        for positive in (False, True):
            _check_kept(nn.keep8(x.cuda(), positive), x, positive)


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_borders(dtype):
    """Largest values on both sides of a unit's change, ties, zeros, the smallest and largest numbers, infinities and NaN."""
    nn = _nn()
    top = torch.tensor([127, 127.49, 127.5, 127.51, 126.5, 64, 63.5, 63.75, 63.99, 128, 1, 0.996, 255, 254.9])
    x = torch.zeros(len(top), 64)
    x[:, 3] = top
    x[:, 4:32] = torch.arange(28) / 2 - 7
    x[:, 33] = -top
    x[:, 40:60] = torch.arange(20) * 0.25
    for scale in (1.0, 2.0 ** -9, 2.0 ** 8, 2.0 ** -14):
        _check_kept(nn.keep8((x * scale).to(dtype).cuda()), (x * scale).to(dtype))
        _check_kept(nn.keep8((x * scale).to(dtype).cuda(), True), (x * scale).to(dtype), True)
    info = torch.finfo(dtype)
    y = torch.zeros(8, 96, dtype=dtype)
    y[0, ::5] = info.max
    y[1, ::5] = -info.max
    y[2, 0], y[2, 1], y[2, 33] = info.tiny, info.tiny / 2, info.smallest_normal / 4
    y[3, 7], y[3, 40] = float("inf"), 1
    y[4, 31], y[4, 32] = float("nan"), 2
    y[5, 64], y[5, 65] = float("-inf"), float("nan")
    y[6] = -0.0
    y[7, 0], y[7, 1] = 1, info.tiny
    _check_kept(nn.keep8(y.cuda()), y)
    _check_kept(nn.keep8(y.cuda(), True), y, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_neighbours(dtype):
    nn = _nn()
    for d in (32, 100, 1111):
        g = torch.Generator().manual_seed(d)
        x = torch.randn(7, d, generator=g).to(dtype)
        wide = torch.full((7, d + 4), float("nan"), dtype=dtype)
        wide[:, 1:1 + d] = x
        plain = nn.keep8(x.cuda())
        assert torch.equal(nn.keep8(wide.cuda()[:, 1:1 + d]).data, plain.data)
        # back into rows of a wider matrix: nothing beside them changes
        from tensorforge_amd import _lib
        out = torch.full((7, d + 4), 5.0, dtype=dtype, device="cuda")
        kind = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
        assert _lib.lib().tf_restore8(plain.data.data_ptr(), 7, d, kind, out[:, 1:].data_ptr(), d + 4,
                                      torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[:, 1:1 + d], plain.restore()) and (out[:, 0] == 5).all() and (out[:, 1 + d:] == 5).all()
    y = torch.randn(2, 3, 40, device="cuda").to(dtype)
    assert nn.keep8(y).restore().shape == (2, 3, 40)
    assert torch.equal(nn.keep8(y).data, nn.keep8(y.view(6, 40)).data)
    for shape in ((0, 40), (3, 0), (0, 0)):
        e = nn.keep8(torch.empty(shape, dtype=dtype, device="cuda"))
        assert e.data.numel() == 0 and e.restore().shape == shape


@pytest.mark.parametrize("rows,d", [((1 << 25) + 3, 64), ((1 << 25) + 3, 63)])
def test_many_elements(rows, d):
    """More than 2^31 elements, as one run of groups and row by row: the ends and a few rows between."""
    nn = _nn()
    x = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 1 << 22):
        n = min(1 << 22, rows - i)
        x[i:i + n] = (torch.arange(i, i + n, device="cuda") % 251)[:, None] * 0.5 - torch.arange(d, device="cuda")
    kept = nn.keep8(x)
    back = kept.restore()
    groups = -(-d // 32)
    for i in (0, 1, 12345, rows // 2, rows - 2, rows - 1):
        codes, exponents = _bytes(x[i:i + 1].cpu())
        at, e = i * groups * 32, rows * groups * 32 + i * groups
        assert torch.equal(kept.data[at:at + groups * 32].cpu(), codes.reshape(-1).view(torch.uint8))
        assert torch.equal(kept.data[e:e + groups].cpu(), exponents.reshape(-1))
    for i in range(0, rows, 1 << 22):
        a, b = x[i:i + (1 << 22)].float(), back[i:i + (1 << 22)].float()
        assert bool(((a - b).abs() <= 0.5 * 2.0 ** -6 * 128).all())  # half of the largest unit: values up to 128
    del x, kept, back
    torch.cuda.empty_cache()


def _matrix(g, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


def _check_grad(got, dy, x, w, z, activation, dtype, bias_dtype):
    """As linear_grad's tests, at the restored x and z."""
    m, k = x.shape
    n = w.shape[1]
    dx, dw, db = got
    dz = dy.double() * (ref.slope(z.double(), activation) if activation != "none" else 1)
    off = 2e-6 * dy.double().abs() * (activation != "none")
    rounded = off + (ref.U[dtype] * dz.abs() + ref.FLOOR[dtype]) * (activation != "none")
    size = dz.abs() + rounded
    if dx is not None:
        ref.close(dx, dz @ w.double().t(), (rounded + (2 * n + 8) * ref.u * size) @ w.double().abs().t(), dtype)
    if dw is not None:
        ref.close(dw, x.double().t() @ dz, x.double().abs().t() @ (rounded + (2 * m + 8) * ref.u * size), dtype)
    if db is not None:
        ref.close(db, dz.sum(0), (off + (2 * m + 8) * ref.u * size).sum(0), bias_dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("activation", ACTS)
def test_linear_grad(activation, order, dtype):
    nn = _nn()
    for m, n, k in ((1, 1, 1), (3, 40, 33), (64, 64, 64), (130, 72, 200), (65, 129, 77), (300, 257, 130), (700, 520, 264)):
        g = torch.Generator().manual_seed(m + n + k)
        dy, x, z = _matrix(g, m, n, dtype), _matrix(g, m, k, dtype), _matrix(g, m, n, dtype, 1.5)
        w = _matrix(g, k, n, dtype, k ** -0.5)
        wc = w.cuda() if order == 0 else w.t().contiguous().cuda().t()
        x8 = nn.keep8(x.cuda())
        z8 = nn.keep8(z.cuda(), activation == "relu") if activation != "none" else None
        xr, zr = x8.restore().cpu(), None if z8 is None else z8.restore().cpu()
        if activation == "relu":
            assert torch.equal(zr > 0, z > 0)
        for bias in (None, dtype, torch.float32):
            got = nn.linear_grad(dy.cuda(), x8, wc, z8, activation, bias_dtype=bias)
            _check_grad(got, dy, xr, w, zr, activation, dtype, bias)
            assert got[1].stride() == wc.stride()
        # one of the two alone, and one result alone
        _check_grad(nn.linear_grad(dy.cuda(), xr.cuda(), wc, z8, activation), dy, xr, w, zr, activation, dtype, None)
        if activation != "none":
            _check_grad(nn.linear_grad(dy.cuda(), x8, wc, zr.cuda(), activation, want_dx=False), dy, xr, w, zr, activation, dtype, None)
        for tile, splits in ((1, 1), (2, 2), (3, 1), (5, 1)):
            _check_grad(nn.linear_grad(dy.cuda(), x8, wc, z8, activation, dtype, tile=tile, splits=splits), dy, xr, w, zr, activation, dtype,
                        dtype)


@pytest.mark.parametrize("order", [0, 1])
def test_gradients_of_no_rows(order):
    nn = _nn()
    w = torch.ones(40, 24, dtype=torch.bfloat16, device="cuda")
    wc = w if order == 0 else w.t().contiguous().t()
    empty = lambda n: torch.empty(0, n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    dx, dw, db = nn.linear_grad(empty(24), nn.keep8(empty(40)), wc, nn.keep8(empty(24)), "gelu", torch.float32)
    assert dx.shape == (0, 40) and (dw == 0).all() and dw.shape == (40, 24) and (db == 0).all()
    dx, dw = nn.rms_norm_grad(empty(40), nn.keep8(empty(40)), torch.ones(40, device="cuda"))
    assert dx.shape == (0, 40) and (dw == 0).all()
    dy = torch.ones(3, 24, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(3, 0, dtype=torch.bfloat16, device="cuda")
    dx, dw, db = nn.linear_grad(dy, nn.keep8(none), w[:0], nn.keep8(dy), "relu", torch.float32)
    assert dx.shape == (3, 0) and dw.shape == (0, 24) and (db == 3).all()


def test_large_linear_grad_is_that_of_the_restored():
    """Aligned sizes run the same products: the same bits."""
    nn = _nn()
    g = torch.Generator().manual_seed(1)
    m, n, k = 1024, 1536, 768
    dy, x, z, w = (_matrix(g, *s, torch.bfloat16).cuda() for s in ((m, n), (m, k), (m, n), (k, n)))
    x8, z8 = nn.keep8(x), nn.keep8(z)
    for a, b in zip(nn.linear_grad(dy, x8, w, z8, "gelu", torch.float32),
                    nn.linear_grad(dy, x8.restore(), w, z8.restore(), "gelu", torch.float32)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 4, 9, 40, 64, 520, 1111, 2048, 4096, 8200, 20000])
def test_norm_grad(d, dtype):
    """The same bits as from the restored rows (float16 restores what this holds exactly)."""
    nn = _nn()
    for rows in (1, 3, 40, 700):
        if rows * d > 4_000_000:
            continue
        g = torch.Generator().manual_seed(d + rows)
        h, dy, dh = (_matrix(g, rows, d, dtype) for _ in range(3))
        w = 1 + 0.1 * torch.randn(d, generator=g)
        h8 = nn.keep8(h.cuda())
        for more in (None, dh.cuda()):
            dx, dw = nn.rms_norm_grad(dy.cuda(), h8, w.cuda(), dh=more)
            a, b = nn.rms_norm_grad(dy.cuda(), h8.restore(), w.cuda(), dh=more)
            assert torch.equal(dx, a) and torch.equal(dw, b)
    want, ww = ref.norm_grad(dy, h8.restore().cpu(), w, dh=dh)
    off = (dx.cpu().double() - want).norm() / want.norm()
    assert float(off) < ref.U[dtype] + 1e-6  # every value is off by half a step and what float32 sums lose


@pytest.mark.parametrize("activation", ACTS)
def test_autograd_keeps_bytes(activation):
    """What the block saves with keep8 is bytes and weights, and its gradients are those of the kept values."""
    nn = _nn()
    g = torch.Generator().manual_seed(5)
    m, d, f = 50, 96, 200
    x, r = (torch.randn(2, m // 2, d, generator=g).bfloat16().cuda().requires_grad_() for _ in range(2))
    nw = torch.ones(d, device="cuda", requires_grad=True)
    w, b = _matrix(g, d, f, torch.bfloat16, d ** -0.5).cuda().requires_grad_(), torch.randn(f, generator=g).cuda().requires_grad_()
    saved = []

    def pack(t):
        saved.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y, h = nn.rms_norm(x, nw, residual=r, keep8=True)
        out = nn.linear(y, w, b, activation, keep8=True)
    params = {t.data_ptr() for t in (nw, w)}
    assert all(t.dtype == torch.uint8 or t.data_ptr() in params for t in saved)
    assert sum(t.dtype == torch.uint8 for t in saved) == (2 if activation == "none" else 3)
    with torch.no_grad():
        plain, z = nn.linear(y, w, b, activation, keep=True)
        assert torch.equal(out, plain)
        dy, dh = (_matrix(g, m, c, torch.bfloat16).view(2, m // 2, c).cuda() for c in (f, d))
        y8, h8, z8 = nn.keep8(y), nn.keep8(h), nn.keep8(z, activation == "relu")
        gy, gw, gb = nn.linear_grad(dy, y8, w, None if activation == "none" else z8, activation, torch.float32)
        gx, gn = nn.rms_norm_grad(gy, h8, nw, dh=dh)
        assert gy.shape == y.shape and gx.shape == x.shape
    got = torch.autograd.grad([out, h], [x, r, nw, w, b], [dy, dh])
    for a, c in zip(got, (gx, gx, gn, gw, gb)):
        assert torch.equal(a, c)


def test_streams_and_graphs():
    """Kept, and used in both gradients, on another stream and in a graph replayed with other inputs."""
    nn = _nn()
    g = torch.Generator().manual_seed(8)
    m, n, k = 96, 200, 130
    w, nw = _matrix(g, k, n, torch.bfloat16).cuda(), torch.ones(k, device="cuda")

    def step(x, z, dy):
        dx, dw, db = nn.linear_grad(dy, nn.keep8(x), w, nn.keep8(z), "silu", torch.float32)
        return (dx, dw, db, *nn.rms_norm_grad(dx, nn.keep8(x), nw))

    inputs = [[_matrix(g, *s, torch.bfloat16).cuda() for s in ((m, k), (m, n), (m, n))] for _ in range(4)]
    want = [step(*i) for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(*inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, want[0]))
    held = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for i, expected in zip(inputs, want):
        for a, b in zip(held, i):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))
        step(*i)


def test_workspaces_of_the_gradient():
    """The C call with exactly the workspace it asks for; less is refused."""
    from tensorforge_amd import _lib
    nn = _nn()
    g = torch.Generator().manual_seed(9)
    for m, n, k in ((100, 72, 50), (600, 512, 768)):
        dy, x, z, w = (_matrix(g, *s, torch.bfloat16).cuda() for s in ((m, n), (m, k), (m, n), (k, n)))
        x8, z8 = nn.keep8(x), nn.keep8(z)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        a = _lib.LinearGradArgs(dy=dy.data_ptr(), x=x8.data.data_ptr(), w=w.data_ptr(), z=z8.data.data_ptr(), dx=dx.data_ptr(),
                                dw=dw.data_ptr(), dy_ld=n, w_ld=n, dx_ld=k, dw_ld=n, m=m, n=n, k=k, type=1, bias_type=1, act=2, kept=3)
        size = ctypes.c_longlong()
        assert _lib.lib().tf_linear_grad_workspace(ctypes.byref(a), ctypes.byref(size)) == 0
        space = torch.full((size.value + 64,), 0xaa, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = space.data_ptr(), size.value - 1
        stream = torch.cuda.current_stream().cuda_stream
        assert _lib.lib().tf_linear_grad(ctypes.byref(a), stream) == -4
        a.workspace_bytes = size.value
        assert _lib.lib().tf_linear_grad(ctypes.byref(a), stream) == 0
        want = nn.linear_grad(dy, x8, w, z8, "gelu")
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]) and (space[size.value:] == 0xaa).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("tile,splits", [(0, 0), (1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (2, 2), (3, 3)])
def test_products_that_keep_z(tile, splits, order, dtype):
    """The product's result as without, and the bytes that keep8 gives of the kept z: written with the product or after it."""
    nn = _nn()
    for i, (m, n, k) in enumerate([(1, 1, 1), (2, 40, 64), (16, 96, 128), (70, 72, 200), (130, 136, 72), (300, 520, 136), (257, 1032, 264),
                                   (65, 257, 77), (600, 200, 0)]):
        g = torch.Generator().manual_seed(m + n + k)
        x, w, r = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, max(k, 1) ** -0.5), _matrix(g, m, n, dtype)
        if i == 4:
            x[3, 5], x[100, 0] = float("inf"), float("nan")
        b = torch.randn(n, generator=g).to(dtype if i % 2 else torch.float32).cuda()
        wc = w.cuda() if order == 0 else w.t().contiguous().cuda().t()
        for activation in ACTS:
            args = (x.cuda(), wc, b if i != 2 else None, nn._act(activation), r.cuda() if i % 3 else None)
            out, kept = nn._C.linear_keep8(*args, False, None, None, None, tile, splits)
            want, z = nn._C.linear(*args, True, None, None, None, tile, splits)
            assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
            assert torch.equal(kept, nn.keep8(z, activation == "relu").data), (m, n, k, activation)


def test_large_products_that_keep_z():
    """Sizes that the choice by sizes gives to each tile, and the C call's refusal of less workspace than it asks for."""
    from tensorforge_amd import _lib
    nn = _nn()
    g = torch.Generator().manual_seed(0)
    for m, n, k in ((4096, 4096, 256), (1000, 4096, 512), (512, 1536, 768), (2048, 2048, 2048), (100, 4096, 4096), (40, 512, 4096), (700, 1001, 300)):
        x, w, b = _matrix(g, m, k, torch.bfloat16).cuda(), _matrix(g, k, n, torch.bfloat16, k ** -0.5).cuda(), torch.randn(n, generator=g).cuda()
        out, kept = nn._C.linear_keep8(x, w, b, 2, None, False, None, None, None, 0, 0)
        want, z = nn.linear(x, w, b, "gelu", keep=True)
        assert torch.equal(out, want) and torch.equal(kept, nn.keep8(z).data), (m, n, k)
    a = _lib.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), out=out.data_ptr(), z=kept.data_ptr(), x_ld=k, w_ld=n, out_ld=n, m=m, n=n, k=k, type=1,
                        out_type=1, kept=2)
    size = ctypes.c_longlong()
    assert _lib.lib().tf_linear_workspace(ctypes.byref(a), ctypes.byref(size)) == 0 and size.value >= 2 * m * n
    assert _lib.lib().tf_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == -4
