"""linear (16 and 8 bits) and linear_grad against 64-bit references: every tile,
loader and split of k, both memory orders, one row to several tiles, odd sizes,
strides, unaligned rows, special values, streams and graphs."""

import ctypes

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu"]


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _matrix(g, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


def _ordered(w, order):
    """w (k x n) on the GPU, row by row or column by column."""
    return w.cuda() if order == 0 else w.t().contiguous().cuda().t()


def _check(out, x, w, b, activation, r, z, dtype, scales=None):
    size = x.double().abs() @ w.double().abs()
    zz = x.double() @ w.double()
    if scales is not None:
        size, zz = size * scales, zz * scales
    if b is not None:
        zz, size = zz + b.double(), size + b.double().abs()
    off = (2 * x.shape[1] + 8) * ref.u * size
    if z is not None:
        ref.close(z, zz, off, dtype)
    want = ref.act(zz, activation)
    off = 1.13 * off + (4e-7 * zz.abs() if activation in ("gelu", "silu") else 0)
    if r is not None:
        want = want + r.double()
        off = off + ref.u * want.abs()
    ref.close(out, want, off, dtype)


# One element, vectors, sizes around 16 and 64, around the tiles (64, 128, 256) and slabs (64 of k), odd ones.
SHAPES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (1, 200, 1000), (16, 16, 32), (17, 48, 72), (64, 64, 64), (63, 65, 63),
          (5, 257, 130), (33, 264, 520), (130, 120, 200), (129, 300, 8), (257, 264, 136), (300, 250, 77)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, order, dtype):
    nn = _nn()
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    x, w, r = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, k ** -0.5), _matrix(g, m, n, dtype)
    for i, activation in enumerate(ACTS):
        for bt in (None, dtype, torch.float32):
            b = None if bt is None else torch.randn(n, generator=g).to(bt)
            res = r if (i + (bt is None)) % 2 else None
            out, z = nn.linear(x.cuda(), _ordered(w, order), None if b is None else b.cuda(), activation,
                               None if res is None else res.cuda(), keep=True)
            assert out.dtype == z.dtype == dtype
            _check(out, x, w, b, activation, res, z, dtype)
            again = nn.linear(x.cuda(), _ordered(w, order), None if b is None else b.cuda(), activation,
                              None if res is None else res.cuda())
            assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("tile", [1, 2, 3, 5])
@pytest.mark.parametrize("splits", [1, 3])
def test_linear_tiles(tile, splits, order, dtype):
    """Every tile over its edges, whole and ragged k, aligned (loads straight into LDS) and not."""
    nn = _nn()
    for m, n, k in ((256, 256, 256), (264, 520, 200), (1, 8, 64), (300, 260, 392), (259, 261, 131)):
        g = torch.Generator().manual_seed(tile + m)
        x, w, r = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, k ** -0.5), _matrix(g, m, n, dtype)
        b = torch.randn(n, generator=g).to(dtype)
        out = nn.linear(x.cuda(), _ordered(w, order), b.cuda(), "gelu", r.cuda(), tile=tile, splits=splits)
        _check(out, x, w, b, "gelu", r, None, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
def test_linear_few_rows(order, dtype):
    """The few-row kernel over its three heights, with fewer and more slabs of k than a workgroup's waves hold."""
    nn = _nn()
    for m in (1, 2, 15, 16, 17, 32, 33, 64):
        for n, k in ((8, 64), (16, 1024), (31, 67), (33, 2200), (40, 5000), (100, 513)):
            g = torch.Generator().manual_seed(m + n + k)
            x, w, r = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, k ** -0.5), _matrix(g, m, n, dtype)
            b = torch.randn(n, generator=g)
            out, z = nn.linear(x.cuda(), _ordered(w, order), b.cuda(), "silu", r.cuda(), keep=True, tile=4)
            _check(out, x, w, b, "silu", r, z, dtype)


@pytest.mark.parametrize("out_dtype", HALF)
@pytest.mark.parametrize("tile,splits", [(0, 0), (1, 1), (2, 1), (3, 1), (5, 1), (2, 2), (3, 3)])
def test_linear_8bit(tile, splits, out_dtype):
    nn = _nn()
    for m, n, k in ((1, 1, 1), (1, 64, 128), (16, 48, 256), (17, 257, 144), (30, 70, 9000), (64, 130, 1040), (257, 264, 272), (40, 72, 100)):
        g = torch.Generator().manual_seed(m + n + k)
        q, s = nn.quantize_rows(_matrix(g, m, k, torch.float32).cuda())
        wq, ws = nn.quantize_rows(_matrix(g, n, k, torch.float32, k ** -0.5).cuda())
        b, r = torch.randn(n, generator=g), _matrix(g, m, n, out_dtype)
        out, z = nn.linear(q, wq.t(), b.cuda(), "silu", r.cuda(), keep=True, x_scale=s, w_scale=ws, out_dtype=out_dtype,
                           tile=tile, splits=splits)
        scales = s.cpu().double()[:, None] * ws.cpu().double()
        _check(out, q.cpu().float(), wq.cpu().float().t(), b, "silu", r, z, out_dtype, scales)


def _grad_want(dy, x, w, z, activation, dtype):
    dz = dy.double() * (ref.slope(z.double(), activation) if activation != "none" else 1)
    # the slope's own error; then one rounding to dtype
    off = 2e-6 * dy.double().abs() * (activation != "none")
    return dz, off, off + (ref.U[dtype] * dz.abs() + ref.FLOOR[dtype]) * (activation != "none")


def _check_grad(got, dy, x, w, z, activation, dtype, bias_dtype):
    m, k = x.shape
    n = w.shape[1]
    dx, dw, db = got
    dz, off, rounded = _grad_want(dy, x, w, z, activation, dtype)
    size = dz.abs() + rounded
    ref.close(dx, dz @ w.double().t(), (rounded + (2 * n + 8) * ref.u * size) @ w.double().abs().t(), dtype)
    ref.close(dw, x.double().t() @ dz, x.double().abs().t() @ (rounded + (2 * m + 8) * ref.u * size), dtype)
    ref.close(db, dz.sum(0), (off + (2 * m + 8) * ref.u * size).sum(0), bias_dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("activation", ACTS)
def test_linear_grad(activation, order, dtype):
    nn = _nn()
    for m, n, k in ((1, 1, 1), (1, 64, 40), (64, 64, 64), (70, 130, 33), (130, 264, 136), (257, 72, 200)):
        g = torch.Generator().manual_seed(m + n + k)
        dy, x, w, z = (_matrix(g, *s, dtype) for s in ((m, n), (m, k), (k, n), (m, n)))
        for bias_dtype in (dtype, torch.float32):
            got = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda() if activation != "none" else None,
                                 activation, bias_dtype=bias_dtype)
            assert got[1].stride() == _ordered(w, order).stride() or min(k, n) == 1
            _check_grad(got, dy, x, w, z, activation, dtype, bias_dtype)
        only = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda() if activation != "none" else None,
                              activation, want_dx=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1], got[1])


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("tile", [1, 2, 3, 5])
@pytest.mark.parametrize("splits", [1, 2])
def test_linear_grad_tiles(tile, splits, order):
    nn = _nn()
    for m, n, k in ((256, 264, 200), (136, 520, 264), (200, 77, 130)):
        g = torch.Generator().manual_seed(m + n + k)
        dy, x, w, z = (_matrix(g, *s, torch.bfloat16) for s in ((m, n), (m, k), (k, n), (m, n)))
        got = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), "silu", bias_dtype=torch.float32, tile=tile,
                             splits=splits)
        _check_grad(got, dy, x, w, z, "silu", torch.bfloat16, torch.float32)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_small_gradients_round_once(activation, dtype):
    """Small gradients carry what dz's rounding leaves: their error is their own rounding's (5% for the few elements, and
    the float sums' share)."""
    nn = _nn()
    for m, n, k in ((1, 300, 200), (64, 64, 64), (100, 264, 136), (130, 77, 65), (600, 128, 128), (2, 1000, 3000)):
        for order in (0, 1):
            g = torch.Generator().manual_seed(m + n)
            dy, x, w, z = (_matrix(g, *s, dtype) for s in ((m, n), (m, k), (k, n), (m, n)))
            dx, dw, _ = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), activation)
            dz = dy.double() * ref.slope(z.double(), activation)
            for got, want in ((dx, dz @ w.double().t()), (dw, x.double().t() @ dz)):
                own = (want.to(dtype).double() - want).norm()
                assert float((got.cpu().double() - want).norm()) <= 1.05 * float(own) + 4e-6 * float(want.norm()), (m, n, k)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_small_gradients_with_long_sums(activation, order, dtype):
    """One side's sum is long and the other's results are few: ranges of k in the products' one launch, odd operands
    copied beside dz, the bias gradient's shares added with the products."""
    nn = _nn()
    for m, n, k in ((2100, 141, 150), (17, 2071, 67), (33, 64, 1030), (1, 1216, 791), (300, 513, 72), (768, 256, 344)):
        g = torch.Generator().manual_seed(m + n + k)
        dy, x, w, z = (_matrix(g, *s, dtype) for s in ((m, n), (m, k), (k, n), (m, n)))
        args = dy.cuda(), x.cuda(), _ordered(w, order), z.cuda() if activation != "none" else None, activation
        _check_grad(nn.linear_grad(*args, bias_dtype=torch.float32), dy, x, w, z, activation, dtype, torch.float32)
        dx, dw, _ = nn.linear_grad(*args)
        assert torch.equal(dx, nn.linear_grad(*args)[0]) and torch.equal(dw, nn.linear_grad(*args)[1])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
def test_few_rows_of_two_terms(order, dtype):
    """dx of up to 32 rows on the few-row kernel: what dz's rounding leaves goes in as further rows."""
    nn = _nn()
    for m, n, k in ((1, 300, 200), (5, 1024, 96), (16, 129, 64), (17, 520, 131), (32, 264, 264), (33, 200, 64)):
        g = torch.Generator().manual_seed(m + n)
        dy, x, w, z = (_matrix(g, *s, dtype) for s in ((m, n), (m, k), (k, n), (m, n)))
        dx, _, _ = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), "silu", want_dw=False, tile=4)
        want = (dy.double() * ref.slope(z.double(), "silu")) @ w.double().t()
        own = (want.to(dtype).double() - want).norm()
        assert float((dx.cpu().double() - want).norm()) <= 1.05 * float(own) + 4e-6 * float(want.norm()), (m, n, k)


@pytest.mark.parametrize("order", [0, 1])
def test_large_ragged(order):
    """Sizes whose unaligned operands are copied to aligned rows first, in both directions."""
    nn = _nn()
    m, n, k = 1031, 1045, 1003
    g = torch.Generator().manual_seed(1)
    x, w, dy, z = (_matrix(g, *s, torch.bfloat16, sc) for s, sc in (((m, k), 1), ((k, n), .03), ((m, n), 1), ((m, n), 1)))
    out = nn.linear(x.cuda(), _ordered(w, order), None, "silu", dy.cuda())
    _check(out, x, w, None, "silu", dy, None, torch.bfloat16)
    for activation in ("none", "gelu"):
        got = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), activation, bias_dtype=torch.float32)
        _check_grad(got, dy, x, w, z, activation, torch.bfloat16, torch.float32)
    q, s = nn.quantize_rows(x.float().cuda())
    wq, ws = nn.quantize_rows(w.t().contiguous().float().cuda())
    out = nn.linear(q, wq.t(), None, "none", None, x_scale=s, w_scale=ws)
    _check(out, q.cpu().float(), wq.cpu().float().t(), None, "none", None, None, torch.bfloat16,
           s.cpu().double()[:, None] * ws.cpu().double())


def test_without_workspace():
    """Through the C ABI with no workspace: unsplit, operands as they are."""
    from tensorforge_amd import _lib
    g = torch.Generator().manual_seed(7)
    for m, n, k in ((70, 64, 4096), (300, 301, 515)):
        x, w = _matrix(g, m, k, torch.bfloat16), _matrix(g, k, n, torch.bfloat16, k ** -0.5)
        xc, wc, out = x.cuda(), w.cuda(), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        a = _lib.LinearArgs(x=xc.data_ptr(), w=wc.data_ptr(), out=out.data_ptr(), x_ld=k, w_ld=n, out_ld=n, m=m, n=n, k=k,
                            type=1, out_type=1)
        _lib.check(_lib.lib().tf_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
        _check(out, x, w, None, "none", None, None, torch.bfloat16)


def test_linear_grad_against_differences():
    """Along random directions: (f(+e) - f(-e)) / 2e in 64 bits against the kernels' inner products."""
    nn = _nn()
    g = torch.Generator().manual_seed(5)
    m, n, k, dtype = 20, 40, 30, torch.float16
    x, w, dy = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, k ** -0.5), _matrix(g, m, n, dtype)
    b = torch.randn(n, generator=g).to(dtype)
    _, z = nn.linear(x.cuda(), w.cuda(), b.cuda(), "gelu", keep=True)
    grads = [t.cpu().double() for t in nn.linear_grad(dy.cuda(), x.cuda(), w.cuda(), z, "gelu", bias_dtype=dtype)]
    f = lambda a, c, d: float((ref.act(a @ c + d, "gelu") * dy.double()).sum())  # noqa: E731
    at = [x.double(), w.double(), b.double()]
    for _ in range(4):
        for i in range(3):
            v = torch.randn(at[i].shape, generator=g).double()
            plus, minus = list(at), list(at)
            plus[i], minus[i] = at[i] + 1e-6 * v, at[i] - 1e-6 * v
            want = (f(*plus) - f(*minus)) / 2e-6
            # z, dz and the result are each rounded to 11 bits
            assert abs(float((grads[i] * v).sum()) - want) <= 3 * 2.0 ** -11 * float((grads[i] * v).abs().sum())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
def test_strides_alignment_and_neighbours(order, dtype):
    """Operands inside larger matrices, on and off 16-byte boundaries, NaN all around them."""
    nn = _nn()
    g = torch.Generator().manual_seed(4)

    def inside(t, before, after):
        nan = lambda c: torch.full((t.shape[0], c), float("nan")).to(t)  # noqa: E731
        big = torch.cat([nan(before), t, nan(after)], 1).cuda()
        big = torch.cat([big, torch.full_like(big[:1], float("nan"))], 0)
        return big[:t.shape[0], before:before + t.shape[1]]

    for m, n, k in ((70, 72, 136), (130, 264, 200), (3, 40, 72), (70, 70, 70)):
        for before, after in ((8, 8), (1, 2), (8, 1)):
            x, w, r = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, k ** -0.5), _matrix(g, m, n, dtype)
            wi = inside(w, before, after) if order == 0 else inside(w.t().contiguous(), before, after).t()
            out, z = nn.linear(inside(x, before, after), wi, None, "relu", inside(r, before, after), keep=True)
            _check(out, x, w, None, "relu", r, z, dtype)
            dy = _matrix(g, m, n, dtype)
            got = nn.linear_grad(inside(dy, before, after), inside(x, before, after), wi, inside(z.cpu(), before, after),
                                 "relu", bias_dtype=dtype)
            _check_grad(got, dy, x, w, z.cpu(), "relu", dtype, dtype)


@pytest.mark.parametrize("splits", [1, 2, 3])
@pytest.mark.parametrize("order", [0, 1])
def test_odd_slabs_and_edges(order, splits):
    """Loads through registers, NaN around the operands: sums of k that end inside a slab (one slab is read back into
    the matrix), ranges of k that are nothing but that slab, tiles wider than the matrix, rows shorter than a piece."""
    nn = _nn()
    g = torch.Generator().manual_seed(splits)
    for m, n, k in ((70, 69, 129), (65, 9, 71), (200, 63, 191), (67, 65, 65), (131, 7, 330), (65, 70, 63), (66, 130, 449)):
        x, w = _matrix(g, m, k, torch.bfloat16), _matrix(g, k, n, torch.bfloat16, k ** -0.5)
        r, dy, z = (_matrix(g, m, n, torch.bfloat16) for _ in range(3))

        def inside(t):
            big = torch.full((t.shape[0] + 2, t.shape[1] + 4), float("nan"), dtype=t.dtype, device="cuda")
            big[1:-1, 1:-3] = t.cuda()
            return big[1:-1, 1:-3]

        wi = inside(w) if order == 0 else inside(w.t()).t()
        out = nn.linear(inside(x), wi, None, "silu", inside(r), tile=3, splits=splits)
        _check(out, x, w, None, "silu", r, None, torch.bfloat16)
        got = nn.linear_grad(inside(dy), inside(x), wi, inside(z), "relu", bias_dtype=torch.float32, tile=3, splits=splits)
        _check_grad(got, dy, x, w, z, "relu", torch.bfloat16, torch.float32)
        got = nn.linear_grad(inside(dy), inside(x), wi, inside(z), "relu", bias_dtype=torch.float32)
        _check_grad(got, dy, x, w, z, "relu", torch.bfloat16, torch.float32)


@pytest.mark.parametrize("tile,splits", [(0, 0), (1, 1), (2, 1), (3, 1), (5, 1), (3, 2)])
def test_writes_stay_inside(tile, splits):
    """Through the C ABI: out and z inside wider matrices; nothing else changes."""
    from tensorforge_amd import _lib
    nn = _nn()
    g = torch.Generator().manual_seed(6)
    for m, n, k in ((1, 5, 64), (67, 70, 64), (130, 263, 72)):
        x, w = _matrix(g, m, k, torch.bfloat16).cuda(), _matrix(g, k, n, torch.bfloat16).cuda()
        for pad in (3, 8):
            out = torch.full((m + 2, n + pad), 7.0, dtype=torch.bfloat16, device="cuda")
            z = out.clone()
            ws = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
            a = _lib.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), out=out[1].data_ptr(), z=z[1].data_ptr(),
                                workspace=ws.data_ptr(), workspace_bytes=ws.numel(), x_ld=k, w_ld=n, out_ld=n + pad,
                                z_ld=n + pad, m=m, n=n, k=k, type=1, out_type=1, tile=tile, splits=splits)
            _lib.check(_lib.lib().tf_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
            want = nn.linear(x, w, tile=tile, splits=splits)
            for t in (out, z):
                assert torch.equal(t[1:-1, :n], want)
                assert (t[0] == 7).all() and (t[-1] == 7).all() and (t[1:-1, n:] == 7).all()


def test_special_values_stay_in_their_rows_and_columns():
    nn = _nn()
    inf, nan = float("inf"), float("nan")
    for m, n, k in ((70, 72, 64), (5, 40, 33)):
        g = torch.Generator().manual_seed(8)
        x, w = _matrix(g, m, k, torch.bfloat16), _matrix(g, k, n, torch.bfloat16)
        x[1, 3], x[2, 0], w[4, 6] = inf, nan, nan
        for order in (0, 1):
            for activation in ACTS:
                out = nn.linear(x.cuda(), _ordered(w, order), None, activation).cpu().float()
                want = ref.act(x.double() @ w.double(), activation)
                want[want.isnan()] = nan
                z = x.double() @ w.double()
                if activation == "relu":
                    want = torch.where(z.isnan(), z, want)
                if activation in ("gelu", "silu"):
                    want = torch.where(z == -inf, torch.zeros_like(z), want)
                assert torch.equal(out.isnan(), want.isnan()), (order, activation)
                assert torch.equal(out.isinf(), want.isinf()), (order, activation)
    z = torch.tensor([[-inf, inf, nan, 0.0, -0.0, -200.0, 200.0, 1e30]], dtype=torch.bfloat16)
    dy = torch.ones_like(z)
    for activation, want in (("relu", [0, 1, nan, 0, 0, 0, 1, 1]), ("gelu", [0, 1, nan, .5, .5, 0, 1, 1]),
                             ("silu", [0, 1, nan, .5, .5, 0, 1, 1])):
        _, _, db = nn.linear_grad(dy.cuda(), torch.ones(1, 8, dtype=torch.bfloat16, device="cuda"),
                                  torch.ones(8, 8, dtype=torch.bfloat16, device="cuda"), z.cuda(), activation,
                                  bias_dtype=torch.float32)
        assert torch.allclose(db.cpu(), torch.tensor(want), atol=1e-6, equal_nan=True), activation


def test_leading_dimensions_and_views():
    """Leading dimensions are rows; a slice of rows, every other row and a matrix's transpose are taken where they lie."""
    nn = _nn()
    g = torch.Generator().manual_seed(13)
    x, w = _matrix(g, 24, 64, torch.bfloat16).cuda(), _matrix(g, 64, 48, torch.bfloat16).cuda()
    want = nn.linear(x, w)
    assert torch.equal(nn.linear(x.view(2, 3, 4, 64), w), want.view(2, 3, 4, 48))
    assert torch.equal(nn.linear(x[0], w), nn.linear(x[:1], w)[0])
    assert torch.equal(nn.linear(x[::2], w), nn.linear(x[::2].contiguous(), w))
    assert torch.equal(nn.linear(x.view(4, 6, 64)[1:3], w), want[6:18].view(2, 6, 48))
    wide = _matrix(g, 64, 96, torch.bfloat16).cuda()
    assert torch.equal(nn.linear(x, wide[:, 48:]), nn.linear(x, wide[:, 48:].contiguous()))
    dx, _, _ = nn.linear_grad(want.view(2, 12, 48), x.view(2, 12, 64), w)
    assert dx.shape == (2, 12, 64) and torch.equal(dx.view(24, 64), nn.linear_grad(want, x, w)[0])


def test_empty_sizes():
    nn = _nn()
    e = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    assert nn.linear(e(0, 8), e(8, 16)).shape == (0, 16)
    assert nn.linear(e(4, 8), e(8, 0)).shape == (4, 0)
    b = torch.randn(16, device="cuda")
    out = nn.linear(e(4, 0), e(0, 16), b, "relu")
    assert torch.equal(out, b.clamp_min(0).to(torch.bfloat16).expand(4, 16))
    dx, dw, db = nn.linear_grad(e(0, 16), e(0, 8), e(8, 16), e(0, 16), "relu", bias_dtype=torch.float32)
    assert dx.shape == (0, 8) and (dw == 0).all() and dw.shape == (8, 16) and (db == 0).all()
    dx, dw, db = nn.linear_grad(e(3, 0), e(3, 8), e(8, 0))
    assert (dx == 0).all() and dx.shape == (3, 8) and dw.shape == (8, 0)


def test_streams_and_graphs():
    """On a side stream, and captured once and replayed between eager calls: the eager bits every time."""
    nn = _nn()
    g = torch.Generator().manual_seed(2)
    x, w, r = (_matrix(g, *s, torch.bfloat16).cuda() for s in ((64, 1024), (1024, 256), (64, 256)))
    nw = torch.ones(1024, device="cuda")
    wq, ws = nn.quantize_rows(w.t().contiguous())

    def chain():
        y, h = nn.rms_norm(x, nw, residual=x)
        out, z = nn.linear(y, w, None, "gelu", r, keep=True, splits=4)
        q, s = nn.quantize_rows(y)
        o8 = nn.linear(q, wq.t(), None, "none", r, x_scale=s, w_scale=ws)
        return [out, o8, h, *nn.linear_grad(r, y, w, z, "gelu", bias_dtype=torch.float32, splits=2),
                *nn.rms_norm_grad(y, h, nw)]

    want = chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for _ in range(4):
        for t in captured:
            t.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        eager = chain()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        assert all(torch.equal(a, b) for a, b in zip(eager, want))


def test_small_gradients_in_a_graph():
    """The small gradients' launches (copies of odd operands, ranges of k, their join, the bias shares) and the norm's
    one, captured once and replayed between eager calls."""
    nn = _nn()
    g = torch.Generator().manual_seed(8)
    cases = [[_matrix(g, *s, torch.bfloat16).cuda() for s in ((m, n), (m, k), (k, n), (m, n))]
             for m, n, k in ((2100, 141, 150), (17, 2071, 67), (256, 256, 128))]
    h, nw = _matrix(g, 9, 999, torch.bfloat16).cuda(), torch.ones(999, device="cuda")

    def chain():
        out = [t for dy, x, w, z in cases for t in nn.linear_grad(dy, x, w, z, "gelu", bias_dtype=torch.float32)]
        return out + list(nn.rms_norm_grad(h, h, nw))

    want = chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for _ in range(4):
        for t in captured:
            t.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        eager = chain()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        assert all(torch.equal(a, b) for a, b in zip(eager, want))


def test_autograd():
    nn = _nn()
    g = torch.Generator().manual_seed(11)
    x, w, r = _matrix(g, 30, 64, torch.float16), _matrix(g, 64, 48, torch.float16, 0.125), _matrix(g, 30, 48, torch.float16)
    b = torch.randn(48, generator=g)
    gy = _matrix(g, 30, 48, torch.float16)
    for activation in ("none", "gelu"):
        leaves = [t.clone().cuda().requires_grad_() for t in (x, w, b, r)]
        nn.linear(*leaves[:3], activation, leaves[3]).backward(gy.cuda())
        same = [t.clone().double().requires_grad_() for t in (x, w, b, r)]
        z = same[0] @ same[1] + same[2]
        ((torch.nn.functional.gelu(z) if activation == "gelu" else z) + same[3]).backward(gy.double())
        for a, c in zip(leaves, same):
            # z, dz and the gradient are each rounded to 11 bits
            assert float((a.grad.cpu().double() - c.grad).norm() / c.grad.norm()) < 3 * 2.0 ** -11
