"""The residual block's operators on offsets past 2^31 elements: rows far apart, in every operand and result, and
matrices of more elements than that."""

import ctypes

import pytest
import torch

import nn_reference as ref
from test_gpu_nn_linear import _check, _check_grad

pytestmark = pytest.mark.gpu

B = torch.bfloat16
ROWS = 70


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


class Far:
    """Matrices of up to 70 rows whose distance puts the last ones past 2^31 elements, side by side in one memory."""

    def __init__(self, ld):
        self.ld, self.at = ld, 0
        self.memory = torch.empty(ROWS * ld, dtype=B, device="cuda")

    def room(self, rows, cols):
        v = self.memory.as_strided((rows, cols), (self.ld, 1), self.at)
        assert rows <= ROWS and self.at + (rows - 1) * self.ld + cols <= self.memory.numel()
        self.at += (cols + 7) // 8 * 8
        return v

    def put(self, t):
        v = self.room(*t.shape)
        v.copy_(t)
        return v


@pytest.fixture(params=[(1 << 25) + 8, (1 << 25) + 3], ids=["aligned", "odd"])
def far(request):
    assert (ROWS - 1) * request.param > 1 << 31
    return Far(request.param)


def _matrix(g, rows, cols, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(B)


def test_norms(far):
    nn = _nn()
    g = torch.Generator().manual_seed(1)
    for d in (5, 64, 1111, 20000):
        x, r, dy, dh = (_matrix(g, ROWS, d) for _ in range(4))
        w = 1 + 0.1 * torch.randn(d, generator=g)
        far.at = 0
        xf, rf, yf, hf = (far.put(t) for t in (x, r, dy, dh))
        for a, b in ((nn.rms_norm(xf, w.cuda(), rf), nn.rms_norm(x.cuda(), w.cuda(), r.cuda())),
                     (nn.rms_norm(xf, w.cuda(), rf, quantize=True), nn.rms_norm(x.cuda(), w.cuda(), r.cuda(), quantize=True)),
                     (nn.quantize_rows(xf), nn.quantize_rows(x.cuda())),
                     (nn.rms_norm_grad(yf, xf, w.cuda(), dh=hf), nn.rms_norm_grad(dy.cuda(), x.cuda(), w.cuda(), dh=dh.cuda()))):
            assert all(torch.equal(p.float(), q.float()) for p, q in zip(a, b)), d
        want, _ = ref.norm(x, w, r)
        ref.close(nn.rms_norm(xf, w.cuda(), rf)[0], want, 112 * ref.u * want.abs(), B)


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("tile", [0, 1, 2, 3, 4, 5])
def test_operands(tile, order, far):
    nn = _nn()
    for m, n, k in ((70, 64, 70), (70, 70, 64), (7, 70, 70)):
        g = torch.Generator().manual_seed(m + n + k)
        x, w, r, dy, z = (_matrix(g, *s, sc) for s, sc in (((m, k), 1), ((k, n), k ** -0.5), ((m, n), 1), ((m, n), 1), ((m, n), 1)))
        far.at = 0
        wf = far.put(w) if order == 0 else far.put(w.t()).t()
        xf, rf, yf, zf = (far.put(t) for t in (x, r, dy, z))
        out, kept = nn.linear(xf, wf, None, "gelu", rf, keep=True, tile=tile)
        _check(out, x, w, None, "gelu", r, kept, B)
        for terms in (1, 2):
            got = nn.linear_grad(yf, xf, wf, zf, "gelu", bias_dtype=torch.float32, tile=tile, terms=terms)
            _check_grad(got, dy, x, w, z, "gelu", B, torch.float32)


def test_results(far):
    """Through the C ABI: results in rows far apart, and nothing written between them."""
    from tensorforge_amd import _lib
    lib, nn = _lib.lib(), _nn()
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(3)
    m, n, k = 70, 61, 64
    x, w, dy, r = (t.cuda() for t in (_matrix(g, m, k), _matrix(g, k, n), _matrix(g, m, n), _matrix(g, m, k)))
    v = torch.ones(k, dtype=B, device="cuda")
    space = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    far.memory.fill_(7)
    out, z, dx, dw, y, h, nx = (far.room(*s) for s in ((m, n), (m, n), (m, k), (k, n), (m, k), (m, k), (m, k)))
    at = dict(workspace=space.data_ptr(), workspace_bytes=space.numel())
    for tile, splits in ((0, 0), (1, 1), (2, 1), (3, 1), (3, 2), (5, 1)):
        a = _lib.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), out=out.data_ptr(), z=z.data_ptr(), x_ld=k, w_ld=n, out_ld=far.ld,
                            z_ld=far.ld, m=m, n=n, k=k, type=1, out_type=1, act=3, tile=tile, splits=splits, **at)
        _lib.check(lib.tf_linear(ctypes.byref(a), stream))
        want = nn.linear(x, w, None, "silu", keep=True, tile=tile, splits=splits)
        assert torch.equal(out, want[0]) and torch.equal(z, want[1]), (tile, splits)
        b = _lib.LinearGradArgs(dy=dy.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), z=z.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(),
                                dy_ld=n, x_ld=k, w_ld=n, z_ld=far.ld, dx_ld=far.ld, dw_ld=far.ld, m=m, n=n, k=k, type=1, bias_type=1,
                                act=3, tile=tile, splits=splits, **at)
        _lib.check(lib.tf_linear_grad(ctypes.byref(b), stream))
        want = nn.linear_grad(dy, x, w, want[1], "silu", tile=tile, splits=splits)
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1]), (tile, splits)
    a = _lib.RmsNormArgs(x=x.data_ptr(), residual=r.data_ptr(), weight=v.data_ptr(), y=y.data_ptr(), h=h.data_ptr(), x_ld=k,
                         residual_ld=k, y_ld=far.ld, h_ld=far.ld, rows=m, d=k, type=1, weight_type=1, y_type=1, eps=1e-6)
    _lib.check(lib.tf_rms_norm(ctypes.byref(a), stream))
    want = nn.rms_norm(x, v, r)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    dv = torch.empty_like(v)
    b = _lib.RmsNormGradArgs(dy=r.data_ptr(), h=x.data_ptr(), weight=v.data_ptr(), dx=nx.data_ptr(), dweight=dv.data_ptr(), dy_ld=k,
                             h_ld=k, dx_ld=far.ld, rows=m, d=k, type=1, weight_type=1, eps=1e-6, **at)
    _lib.check(lib.tf_rms_norm_grad(ctypes.byref(b), stream))
    want = nn.rms_norm_grad(r, x, v)
    assert torch.equal(nx, want[0]) and torch.equal(dv, want[1])
    written = sum(t.numel() for t in (out, z, dx, dw, y, h, nx))
    assert int((far.memory != 7).sum()) <= written


def _some(n):
    """The first, the last and those on both sides of every 2^20."""
    near = [i for b in range(0, n, 1 << 20) for i in (b - 1, b, b + 1)]
    return torch.tensor(sorted({i for i in near + [n - 1] if 0 <= i < n}))


def _normal(*shape):
    return torch.empty(shape, dtype=B, device="cuda").normal_()


@pytest.mark.parametrize("odd", [0, 1])
def test_many_elements(odd):
    """Matrices of more than 2^31 elements: rows of x, w in either order, and their gradients."""
    nn = _nn()
    torch.manual_seed(5)
    m, k, n = (1 << 20) + 100 + odd, 2048 + odd, 64 + odd
    x, w = _normal(m, k), (_normal(k, n) * k ** -0.5)
    assert x.numel() > 1 << 31
    rows = _some(m)
    out = nn.linear(x, w, None, "silu")
    _check(out[rows], x[rows].cpu(), w.cpu(), None, "silu", None, None, B)
    y, _ = nn.rms_norm(x, torch.ones(k, device="cuda"))
    want, _ = ref.norm(x[rows].cpu(), torch.ones(k))
    ref.close(y[rows], want, 112 * ref.u * want.abs(), B)
    q, s = nn.quantize_rows(x)
    ref.f8_close(q[rows], s[rows], x[rows].cpu().double(), 8 * ref.u)
    del q, s
    ndx, _ = nn.rms_norm_grad(y, x, torch.ones(k, device="cuda"))
    want, _ = ref.norm_grad(y[rows].cpu(), x[rows].cpu(), torch.ones(k))
    # the sums' share: at most (2 * 96 + 16) roundings of terms of r*(|g| + |xhat| mean|g xhat|), |g|, |xhat| being under 6
    ref.close(ndx[rows], want, torch.tensor(2 * 208 * ref.u * 6 * 8.0), B)
    del y, ndx
    dy, z = out, _normal(m, n)
    dx, dw, db = nn.linear_grad(dy, x, w, z, "gelu", bias_dtype=torch.float32)
    dz = dy[rows].cpu().double() * ref.slope(z[rows].cpu().double(), "gelu")
    off = 2e-6 * dy[rows].cpu().double().abs() + ref.U[B] * dz.abs() + ref.FLOOR[B]
    ref.close(dx[rows], dz @ w.cpu().double().t(), (off + (2 * n + 8) * ref.u * (dz.abs() + off)) @ w.cpu().double().abs().t(), B)
    want = torch.zeros(k, n, dtype=torch.float64, device="cuda")
    for i in range(0, m, 1 << 17):
        part = slice(i, i + (1 << 17))
        f = z[part].double()
        f = dy[part].double() * (torch.special.erfc(-f * 0.5 ** 0.5) / 2 + f * torch.exp(-f * f / 2) * 0.3989422804014327)
        want += (x[part].float().t().contiguous() @ f.float()).double()
    # dz's rounding (2^-9 of the terms in the mean square), the result's and the sums' in float
    assert float((dw.double() - want).norm() / want.norm()) < 2.0 ** -8


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("order", [0, 1])
def test_many_columns(order, odd):
    nn = _nn()
    torch.manual_seed(6)
    m, k, n = 70, 2048 + odd, (1 << 20) + 100 + odd
    x, w = _normal(m, k), _normal(k, n) if order == 0 else _normal(n, k).t()
    assert w.numel() > 1 << 31
    some = _some(n)
    for rows in (m, 3):
        out = nn.linear(x[:rows], w, None, "relu")
        _check(out[:, some], x[:rows].cpu(), w[:, some].cpu(), None, "relu", None, None, B)
    out = nn.linear(x, w)
    dx, dw, _ = nn.linear_grad(out, x, w)
    dys, ws = out[:, some].cpu().double(), x.cpu().double()
    ref.close(dw[:, some], ws.t() @ dys, (2 * m + 8) * ref.u * (ws.abs().t() @ dys.abs()), B)
    want = torch.zeros(m, k, dtype=torch.float64, device="cuda")
    for i in range(0, n, 1 << 17):
        part = slice(i, i + (1 << 17))
        want += (out[:, part].float() @ w[:, part].float().t().contiguous()).double()
    assert float((dx.double() - want).norm() / want.norm()) < 2.0 ** -8
