"""Corners of the residual block's operators, each against its definition: infinities in the gradients' second term,
rows of no elements, sizes near the limits, second-order and forward-mode gradients."""

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _matrix(g, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


def _ordered(w, order):
    """w (k x n) on the GPU, row by row or column by column."""
    return w.cuda() if order == 0 else w.t().contiguous().cuda().t()


# On both sides of 1.4e8 multiply-adds: below, dz of a smooth activation goes into the products in two terms.
GRAD_SIZES = [(4, 16, 8, 2), (40, 130, 77, 2), (300, 264, 200, 2), (528, 528, 528, 1)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_infinite_dy(activation, order, dtype):
    """An infinity in dy: infinities of the right sign in its row of dx and its column of dw, nothing else changed."""
    nn = _nn()
    for m, n, k, _ in GRAD_SIZES:
        g = torch.Generator().manual_seed(m + n)
        x, w, dy = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype), _matrix(g, m, n, dtype)
        z = torch.ones(m, n, dtype=dtype)
        x[x == 0], w[w == 0] = 1, 1
        dy[1, 3], dy[2, 5] = float("inf"), -float("inf")
        dz = dy.double() * ref.slope(z.double(), activation)
        args = dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), activation
        dx, dw, _ = nn.linear_grad(*args)
        for how in ({}, {"want_dw": False, "tile": 4}, {"want_dw": False}):
            dx = nn.linear_grad(*args, **how)[0]
            for got, want in ((dx, dz @ w.double().t()), (dw, x.double().t() @ dz)):
                got = got.cpu().double()
                assert not got.isnan().any(), (m, how)
                assert torch.equal(got[want.isinf()], want[want.isinf()])
                assert got[want.isfinite()].isfinite().all()


@pytest.mark.parametrize("order", [0, 1])
def test_dz_past_float16(order):
    """dy * act'(z) past float16's largest value.  Two terms hold it; one is rounded to an infinity."""
    nn = _nn()
    for m, n, k, terms in GRAD_SIZES:
        g = torch.Generator().manual_seed(m + n)
        x, w, dy = _matrix(g, m, k, torch.float16, 1 / 64), _matrix(g, k, n, torch.float16, 1 / 64), _matrix(g, m, n, torch.float16)
        x[x == 0], w[w == 0] = 0.01, 0.01
        z = torch.ones(m, n, dtype=torch.float16)
        dy[1, 3], z[1, 3], dy[2, 5], z[2, 5] = 60000, 1.5, -65504, 1.4
        dz = dy.double() * ref.slope(z.double(), "gelu")
        assert dz[1, 3] > 65520 and dz[2, 5] < -65520
        if terms == 1:
            dz = dz.half().double()
        dx, dw, _ = nn.linear_grad(dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), "gelu")
        # dz is off by its slope (2e-6 of dy) and, in one term, its rounding; then float sums and the result's rounding
        off = 2e-6 * dy.double().abs()
        if terms == 1:
            off = off + ref.U[torch.float16] * torch.where(dz.isinf(), torch.zeros_like(dz), dz.abs())
        size = torch.where(dz.isinf(), torch.zeros_like(dz), dz.abs())
        ref.close(dx, dz @ w.double().t(), (off + (2 * n + 8) * ref.u * size) @ w.double().abs().t(), torch.float16)
        ref.close(dw, x.double().t() @ dz, x.double().abs().t() @ (off + (2 * m + 8) * ref.u * size), torch.float16)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_infinite_operands_of_a_gradient(activation, order, dtype):
    """An infinity in x reaches dw's row, one in w dx's column, with the sign of dz; a NaN stays one."""
    nn = _nn()
    for m, n, k, _ in GRAD_SIZES:
        g = torch.Generator().manual_seed(m * n)
        x, w, dy = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype), _matrix(g, m, n, dtype)
        z = torch.rand(m, n, generator=g).to(dtype)  # the slope is above 0
        dy[dy == 0] = 1
        x[1, 2], x[3, 5], w[4, 6], w[6, 1], w[7, 7] = float("inf"), float("nan"), -float("inf"), float("nan"), float("inf")
        dz = dy.double() * ref.slope(z.double(), activation)
        args = dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), activation
        _, dw, _ = nn.linear_grad(*args)
        for how in ({}, {"want_dw": False, "tile": 4}, {"want_dw": False}, {"want_dw": False, "splits": 2}):
            dx = nn.linear_grad(*args, **how)[0]
            for got, want in ((dx, dz @ w.double().t()), (dw, x.double().t() @ dz)):
                got = got.cpu().double()
                assert torch.equal(got.isnan(), want.isnan()), (m, how)
                assert torch.equal(got[want.isinf()], want[want.isinf()])
                assert got[want.isfinite()].isfinite().all()


def test_scales_of_rows_without_elements():
    """Rows of no elements have the scale of zeros, and a product over no k of them is the bias."""
    nn = _nn()
    scale = torch.tensor(ref.TINY / ref.F8_MAX).cuda()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for rows in (1, 5, 9000):
            torch.full((rows,), float("nan"), device="cuda")  # what the allocator may hand out next
            q, s = nn.quantize_rows(torch.empty(rows, 0, dtype=dtype, device="cuda"))
            assert q.shape == (rows, 0) and s.shape == (rows,) and (s == scale).all()
            torch.full((rows,), float("nan"), device="cuda")
            x = torch.empty(rows, 0, dtype=dtype, device="cuda")
            _, s, h = nn.rms_norm(x, x[0], residual=x, quantize=True)
            assert (s == scale).all() and h.shape == (rows, 0)
    q, s = nn.quantize_rows(torch.empty(40, 0, device="cuda"))
    wq, ws = nn.quantize_rows(torch.empty(24, 0, device="cuda"))
    b = torch.randn(24, device="cuda")
    assert torch.equal(nn.linear(q, wq.t(), b, x_scale=s, w_scale=ws), b.bfloat16().expand(40, 24))


def test_forward_mode_is_refused():
    """A tangent is not dropped in silence: the calls have no forward-mode derivative."""
    import torch.autograd.forward_ad as fwd
    nn = _nn()
    x, w, v = (torch.ones(s, dtype=torch.bfloat16, device="cuda") for s in ((4, 8), (8, 8), (8,)))
    with fwd.dual_level():
        for call in (lambda t: nn.linear(t, w, None, "gelu"), lambda t: nn.rms_norm(t, v)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                    call(fwd.make_dual(x, x))


@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_gradient_of_the_kept_pre_activation(activation):
    nn = _nn()
    g = torch.Generator().manual_seed(12)
    x, w, gy, gz = (_matrix(g, *s, torch.float16, sc) for s, sc in (((30, 64), 1), ((64, 48), .125), ((30, 48), 1), ((30, 48), 1)))
    b = torch.randn(48, generator=g)
    leaves = [t.clone().cuda().requires_grad_() for t in (x, w, b)]
    out, z = nn.linear(*leaves, activation, keep=True)
    torch.autograd.backward([out, z], [gy.cuda(), gz.cuda()])
    same = [t.clone().double().requires_grad_() for t in (x, w, b)]
    zz = same[0] @ same[1] + same[2]
    torch.autograd.backward([torch.nn.functional.gelu(zz) if activation == "gelu" else zz + 0, zz], [gy.double(), gz.double()])
    for a, c in zip(leaves, same):
        # z and dz are each rounded to 11 bits, then both gradients and their sum
        assert float((a.grad.cpu().double() - c.grad).norm() / c.grad.norm()) < 5 * 2.0 ** -11


def test_a_residual_of_other_leading_dimensions():
    nn = _nn()
    g = torch.Generator().manual_seed(3)
    x, r, w, v = (_matrix(g, *s, torch.bfloat16).cuda() for s in ((6, 64), (6, 64), (64, 64), (1, 64)))
    grads = []
    for shape in ((6, 64), (2, 3, 64)):
        a, b = x.view(shape).clone().requires_grad_(), r.clone().requires_grad_()
        y, h = nn.rms_norm(a, v[0], residual=b)
        out = nn.linear(y, w, None, "gelu", b)
        torch.autograd.backward([out, h], [torch.ones_like(out), torch.ones_like(h)])
        assert a.grad.shape == a.shape and b.grad.shape == b.shape
        grads.append((a.grad.view(6, 64), b.grad))
    assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("d", [1, 4, 7])
def test_many_short_rows(d):
    """More rows than a launch has places for workgroups of one row each; every row's result."""
    nn = _nn()
    rows = (1 << 24) + 5
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(rows, d, generator=g, device="cuda").bfloat16()
    w = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    with torch.no_grad():
        f = x.float()
        r = torch.rsqrt((f * f).mean(1, keepdim=True) + 1e-6)
        want = f * r * w
    y, _ = nn.rms_norm(x, w)
    assert ((y.float() - want).abs() <= (ref.U[torch.bfloat16] + 64 * ref.u) * want.abs()).all()
    q, s = nn.quantize_rows(x)
    top = f.abs().amax(1).clamp_min(ref.TINY)
    assert ((s * 448 - top).abs() <= 4 * ref.u * top).all()
    # codes are off by half a spacing, 1/16 of the value at most, or of the smallest normal number
    assert ((q.float() * s[:, None] - f).abs() <= 0.0626 * torch.maximum(f.abs(), s[:, None] * 2.0 ** -6)).all()
    dy = torch.randn(rows, d, generator=g, device="cuda").bfloat16()
    dx, dw = nn.rms_norm_grad(dy, x, w)
    gw = dy.float() * w
    size = r * (gw.abs() + (f * r).abs() * (gw * f * r).abs().mean(1, keepdim=True))
    want = r * (gw - f * r * (gw * f * r).mean(1, keepdim=True))
    assert ((dx.float() - want).abs() <= ref.U[torch.bfloat16] * want.abs() + 64 * ref.u * size + 2.0 ** -133).all()
    want = (dy.double() * f * r).sum(0)
    # 512 shares of 8192 rows each
    assert ((dw - want).abs() <= 2 * (rows // 2048 + 64) * ref.u * (dy.double() * f * r).abs().sum(0)).all()


def _normal(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def test_sums_of_many_columns():
    """The shares' sums over more columns than one side of a launch has places for."""
    nn = _nn()
    d = (1 << 28) + 24
    h, dy, w = _normal(1, 1, d), _normal(2, 1, d), torch.ones(d, dtype=torch.bfloat16, device="cuda")
    dx, dw = nn.rms_norm_grad(dy, h, w)
    r = torch.rsqrt(h.float().square().mean() + 1e-6)
    want = dy[0].float() * h[0].float() * r
    # the row's sum: 2^20 additions a thread and the joining, halved by its root
    assert ((dw.float() - want).abs() <= (ref.U[torch.bfloat16] + (1 << 18) * ref.u) * want.abs()).all()
    assert dx.isfinite().all()
    del h, dx, dw, w, want
    n = (1 << 29) + 8
    dy = dy.new_empty(1, n).normal_()
    x = torch.full((1, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    _, dw, db = nn.linear_grad(dy, x, torch.zeros(1, n, dtype=torch.bfloat16, device="cuda"), want_dx=False, bias_dtype=torch.bfloat16)
    assert torch.equal(db, dy[0]) and torch.equal(dw, 2 * dy)


@pytest.mark.parametrize("order", [0, 1])
def test_few_rows_of_many_columns(order):
    """More columns than the few-row kernel's launch has places for."""
    nn = _nn()
    for m, n, k in ((1, (1 << 27) + 8, 8), (3, (1 << 26) + 3, 7)):
        x = _normal(m, m, k)
        w = _normal(5, k, n) if order == 0 else _normal(5, n, k).t()
        out = nn.linear(x, w)
        want, size = 0, 0
        for j in range(k):
            term = x[:, j:j + 1].float() * w[j].float()
            want, size = want + term, size + term.abs()
        assert ((out.float() - want).abs() <= ref.U[torch.bfloat16] * want.abs() + 4 * (k + 4) * ref.u * size).all()
        del w, out, want, size


def test_a_product_of_very_many_rows():
    """More tiles than one side of a launch has places for: rows of one element, multiplied where they lie."""
    nn = _nn()
    m = 1 << 30
    x = torch.empty(m, 1, dtype=torch.bfloat16, device="cuda").normal_()
    out = nn.linear(x, torch.full((1, 1), 2.0, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, device="cuda"), "none")
    assert torch.equal(out, 2 * x)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_activations_of_every_value(activation, dtype):
    """Every finite z: the value and the slope off by their rounding and 1e-5 of themselves (exponents of up to 126 halvings,
    each rounded in float: 126 * ln 2 * 2^-24), 1e-6 where the slope crosses zero.  A factor below the smallest normal
    number may be flushed to zero before z multiplies it."""
    nn = _nn()
    z = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    z = z[z.isfinite()]
    z = torch.cat([z, torch.zeros(-len(z) % 8, dtype=dtype)]).view(-1, 8)
    zd = z.double()
    eye = torch.eye(8, dtype=dtype).cuda()
    out = nn.linear(z.cuda(), eye, None, activation)
    flushed = lambda v: torch.finfo(torch.float32).tiny * (1 + v.abs().clamp_max(200))  # noqa: E731
    want = ref.act(zd, activation)
    ref.close(out, want, 1e-5 * want.abs() + flushed(zd), dtype)
    dy = torch.ones_like(z)
    _, _, db = nn.linear_grad(dy[:1].cuda(), dy[:1].cuda(), eye, z[:1].cuda(), activation, bias_dtype=torch.float32)
    assert db.shape == (8,)
    # dx of one row through the unit matrix: dz itself, in two terms
    step = 2048
    for at in range(0, len(z), step):
        part = z[at:at + step]
        dx, _, _ = nn.linear_grad(dy[at:at + step].cuda(), part.cuda(), eye, part.cuda(), activation, want_dw=False)
        want = ref.slope(part.double(), activation)
        ref.close(dx, want, 1e-5 * want.abs() + 1e-6 * (part.abs() < 3) + flushed(part.double()), dtype)


def test_bad_numbers_are_value_errors():
    """What the library refuses, and numbers that its arguments do not hold, before any work."""
    nn = _nn()
    x, w, v = _normal(1, 4, 8), _normal(2, 8, 16), _normal(3, 8)
    dy = _normal(4, 4, 16)
    for call, words in (
            (lambda: nn.linear(x, w, tile=9), "tile = 9"), (lambda: nn.linear(x, w, tile=1 << 32), "tile = 4294967296"),
            (lambda: nn.linear(x, w, splits=-1), "splits = -1"), (lambda: nn.linear(x, w, splits=(1 << 32) + 2), "splits = 4294967298"),
            (lambda: nn.linear_grad(dy, x, w, tile=-(1 << 40)), "tile = -1099511627776"),
            (lambda: nn.linear_grad(dy, x, w, splits=65), "splits = 65"), (lambda: nn.rms_norm(x, v, eps=-1.0), "eps"),
            (lambda: nn.rms_norm(x, v, eps=float("nan")), "eps"), (lambda: nn.rms_norm_grad(x, x, v, eps=-1e-3), "eps")):
        with pytest.raises(ValueError, match=words):
            call()
    for call in (lambda: nn.linear(x, w, tile=1 << 70), lambda: nn.linear(x, w, tile="2"), lambda: nn.rms_norm(x, v, eps=None)):
        with pytest.raises((TypeError, OverflowError)):
            call()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_terms_of_dz(activation, dtype):
    """The caller's choice on both sides of the sizes': in two terms the products err by their own rounding (5% for few
    elements, and the float sums' share), in one they are those of the rounded dz."""
    nn = _nn()
    for m, n, k in ((64, 72, 40), (130, 77, 65), (528, 528, 528), (700, 520, 515)):
        for order in (0, 1):
            g = torch.Generator().manual_seed(m + n)
            dy, x, w, z = (_matrix(g, *s, dtype) for s in ((m, n), (m, k), (k, n), (m, n)))
            args = dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), activation
            dz = dy.double() * ref.slope(z.double(), activation)
            got = {t: nn.linear_grad(*args, terms=t)[:2] for t in (0, 1, 2)}
            for i, (a, b) in enumerate(((dz, w.double().t()), (x.double().t(), dz))):
                want, own = a @ b, ((a @ b).to(dtype).double() - a @ b).norm()
                assert float((got[2][i].cpu().double() - want).norm()) <= 1.05 * float(own) + 4e-6 * float(want.norm()), (m, n, k)
                # sqrt(2) of the own rounding, and as much above one as 5% leaves
                assert 1.05 * float(own) < float((got[1][i].cpu().double() - want).norm()) < 1.6 * float(own), (m, n, k)
                assert torch.equal(got[0][i], got[2 if m * n * k <= 1.4e8 else 1][i])
            leaves = [t.detach().requires_grad_() for t in args[1:3]]
            out, zk = nn.linear(*leaves, None, activation, keep=True, grad_terms=2)
            out.backward(args[0])
            for a, b in zip(leaves, nn.linear_grad(args[0], *args[1:3], zk.detach(), activation, terms=2)):
                assert torch.equal(a.grad, b)
    for terms in (-1, 3):
        with pytest.raises(ValueError, match="terms = "):
            nn.linear_grad(*args, terms=terms)


@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4, 5])
def test_sums_of_8bit_products(tile):
    """What the sums inside an 8-bit product lose, seen where the bias takes the exact sum away.  Eight neighbouring k are
    aligned to the largest of their products and cut off 13 bits below it; the rest is float32 (one rounding for each eight
    products, one for the bias).  Signs being random, the cuts' root mean square is under one cut a product."""
    nn = _nn()
    for k in (128, 1024, 4096):
        g = torch.Generator().manual_seed(k)
        x = (100 * torch.randn(1, k, generator=g)).clamp(-448, 448).to(ref.F8)
        w = (100 * torch.randn(256, k, generator=g)).clamp(-448, 448).to(ref.F8)
        products = x.float().double() * w.float().double()
        want, size = products.sum(1), products.abs().sum(1)
        cut = 2.0 ** -13 * products.abs().view(256, -1, 8).amax(2)
        rows = 1 if tile in (0, 4) else 256
        one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
        out = nn.linear(x.expand(rows, k).contiguous().cuda(), w.cuda().t(), (-want).float().cuda(), x_scale=one(rows), w_scale=one(256),
                        tile=tile, splits=1)
        off = out.cpu().double()
        assert (off == off[:1]).all()
        off = off[0]
        rest = (k // 8 + 4) * ref.u * size
        assert (off.abs() <= 1.01 * (8 * cut.sum(1) + rest)).all()
        least = (8 * cut.square().sum(1)).mean().sqrt()
        assert float(off.square().mean().sqrt()) <= 1.01 * float(least + rest.square().mean().sqrt()), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 6, 3000])
def test_norms_in_place(rows, dtype):
    """Through the C ABI: h over x or the residual, dx over dy or dh, at whole and odd lengths of every kernel."""
    import ctypes

    from tensorforge_amd import _lib
    nn, lib = _nn(), _lib.lib()
    stream = torch.cuda.current_stream().cuda_stream
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    for d in (5, 64, 333, 1024, 1111, 2056, 4100, 8193, 16387):
        if rows * d > 8000000:
            continue
        x, r, dy, dh = (_normal(i, rows, d, dtype=torch.float32).to(dtype) for i in range(4))
        w = 1 + 0.1 * _normal(9, d, dtype=torch.float32)
        y, h = nn.rms_norm(x, w, r)
        for over in (0, 1):
            a, b, got = x.clone(), r.clone(), torch.empty_like(x)
            args = _lib.RmsNormArgs(x=a.data_ptr(), residual=b.data_ptr(), weight=w.data_ptr(), y=got.data_ptr(),
                                    h=(a, b)[over].data_ptr(), x_ld=d, residual_ld=d, y_ld=d, h_ld=d, rows=rows, d=d, type=code,
                                    weight_type=0, y_type=code, eps=1e-6)
            _lib.check(lib.tf_rms_norm(ctypes.byref(args), stream))
            assert torch.equal(got, y) and torch.equal((a, b)[over], h) and torch.equal((a, b)[1 - over], (x, r)[1 - over]), (d, over)
        dx, dw = nn.rms_norm_grad(dy, h, w, dh=dh)
        space = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
        for over in (0, 1):
            a, b, got = dy.clone(), dh.clone(), torch.empty_like(w)
            args = _lib.RmsNormGradArgs(dy=a.data_ptr(), h=h.data_ptr(), dh=b.data_ptr(), weight=w.data_ptr(), dx=(a, b)[over].data_ptr(),
                                        dweight=got.data_ptr(), dy_ld=d, h_ld=d, dh_ld=d, dx_ld=d, rows=rows, d=d, type=code,
                                        weight_type=0, eps=1e-6, workspace=space.data_ptr(), workspace_bytes=space.numel())
            _lib.check(lib.tf_rms_norm_grad(ctypes.byref(args), stream))
            assert torch.equal((a, b)[over], dx) and torch.equal(got, dw), (d, over)


def test_rows_with_infinities():
    nn = _nn()
    inf, nan = float("inf"), float("nan")
    for d in (6, 64, 1111, 20000):
        x = torch.ones(4, d, device="cuda")
        x[0, 3], x[1, 4], x[1, 5], x[2, 2] = inf, -inf, inf, nan
        w = torch.ones(d, device="cuda")
        y, _ = nn.rms_norm(x, w)
        at = x[:2].isinf()
        assert y[:2][at].isnan().all() and (y[:2][~at] == 0).all() and y[2].isnan().all() and y[3].isfinite().all()
        for q, s in (nn.rms_norm(x, w, quantize=True)[:2], nn.quantize_rows(x)):
            v = q.float() * s[:, None]
            assert v[:3].isnan().all() and v[3].isfinite().all(), d


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_are_those_of_the_formula(dtype):
    """Bit by bit: scale = top/448, code = nearest(x * (448 * (1/top))), each step in float32."""
    nn = _nn()
    for rows, d in ((4000, 6), (3000, 64), (700, 1111), (300, 4096), (90, 20000)):
        x = (_normal(d, rows, d, dtype=torch.float32) * torch.exp(_normal(7, rows, 1, dtype=torch.float32))).to(dtype)
        x[1] = 0
        q, s = nn.quantize_rows(x)
        f = x.float()
        top = f.abs().amax(1, keepdim=True).clamp_min(ref.TINY)
        factor = ref.F8_MAX * (torch.ones_like(top) / top)
        assert torch.equal(q.view(torch.uint8), (f * factor).to(ref.F8).view(torch.uint8)), (rows, d)
        assert torch.equal(s, (top / torch.full_like(top, ref.F8_MAX))[:, 0])


@pytest.mark.parametrize("dtype", HALF)
def test_8bit_products_of_few_k(dtype):
    """Element by element within what tforge_hip.h says of 8-bit sums, where few products make that visible: for each
    eight k 2^-10 of their largest product, then float32."""
    nn = _nn()
    for m, n, k in ((70, 61, 2), (33, 130, 8), (130, 40, 14), (5, 100, 30), (64, 64, 59), (3, 7, 130)):
        g = torch.Generator().manual_seed(m + n + k)
        q, s = nn.quantize_rows(_matrix(g, m, k, torch.float32).cuda())
        wq, ws = nn.quantize_rows(_matrix(g, n, k, torch.float32).cuda())
        b = torch.randn(n, generator=g)
        x, w, scales = q.cpu().double(), wq.cpu().double(), s.cpu().double()[:, None] * ws.cpu().double()
        cut = sum(2.0 ** -10 * (x[:, None, i:i + 8] * w[None, :, i:i + 8]).abs().amax(2) for i in range(0, k, 8))
        z = (x @ w.t()) * scales + b.double()
        off = (cut + (2 * k + 8) * ref.u * (x.abs() @ w.abs().t())) * scales + 4 * ref.u * (z.abs() + b.double().abs())
        for tile, splits in ((0, 0), (1, 1), (2, 1), (3, 1), (3, 2), (4, 1), (5, 1)):
            out = nn.linear(q, wq.t(), b.cuda(), x_scale=s, w_scale=ws, out_dtype=dtype, tile=tile, splits=splits)
            ref.close(out, z, off, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
def test_infinite_operands_where_nothing_is_rounded(order, dtype):
    """dz that is exact has a second term of zeros, and zero times infinity is no number: x's and w's infinities stay."""
    nn = _nn()
    for m, n, k, _ in GRAD_SIZES:
        g = torch.Generator().manual_seed(m)
        x, w, dy = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype), _matrix(g, m, n, dtype)
        dy[dy == 0] = 1
        z = torch.zeros(m, n, dtype=dtype)  # the slope is 1/2
        x[1, 2], x[3, 5], w[4, 6], w[6, 1] = float("inf"), -float("inf"), -float("inf"), float("inf")
        dz = dy.double() / 2
        args = dy.cuda(), x.cuda(), _ordered(w, order), z.cuda(), "gelu"
        _, dw, _ = nn.linear_grad(*args, terms=2)
        for how in ({}, {"want_dw": False, "tile": 4}, {"want_dw": False}, {"want_dw": False, "splits": 2}):
            dx = nn.linear_grad(*args, **how, terms=2)[0]
            for got, want in ((dx, dz @ w.double().t()), (dw, x.double().t() @ dz)):
                got = got.cpu().double()
                assert not got.isnan().any() and torch.equal(got[want.isinf()], want[want.isinf()]), (m, how)
