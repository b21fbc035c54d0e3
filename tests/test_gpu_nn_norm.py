"""rms_norm (with the residual, in the input's type and in 8 bits), quantize_rows
and rms_norm_grad against 64-bit references: every kernel by row length, one row
to many, odd lengths, strides, unaligned rows, special values."""

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# Row lengths on both sides of every kernel's range: 512, 1024, 2048, 4096, 8192, 16384.
LENGTHS = [1, 7, 8, 64, 333, 512, 513, 1024, 1111, 2048, 2056, 4096, 4100, 8192, 8193, 16384, 16387]
# A row's sum: at most 64 products a thread and 16 joining steps; its root halves the error.
TERMS = 96


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _data(rows, d, dtype, seed, **extra):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, d, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)
    return x, (1 + 0.2 * torch.randn(d, generator=g)), torch.randn(rows, d, generator=g).to(dtype), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", LENGTHS)
def test_norm(d, dtype):
    nn = _nn()
    for rows in (1, 5):
        x, w, r, _ = _data(rows, d, dtype, d)
        for wt in (dtype, torch.float32):
            wc = w.to(wt)
            for res in (None, r):
                y, h = nn.rms_norm(x.cuda(), wc.cuda(), residual=None if res is None else res.cuda())
                want, hw = ref.norm(x, wc, res)
                assert y.dtype == dtype
                ref.close(y, want, (TERMS + 16) * ref.u * want.abs(), dtype)
                if res is None:
                    assert h is None
                else:
                    ref.close(h, hw, ref.u * hw.abs(), dtype)
                q, s, h = nn.rms_norm(x.cuda(), wc.cuda(), residual=None if res is None else res.cuda(), quantize=True)
                assert q.dtype == ref.F8 and s.dtype == torch.float32 and s.shape == (rows,)
                ref.f8_close(q, s, want, (2 * TERMS + 32) * ref.u)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 9, 64, 1111, 4096, 20000])
def test_quantize_rows(d, dtype):
    nn = _nn()
    x, *_ = _data(6, d, dtype, d)
    x[3] = 0
    q, s = nn.quantize_rows(x.cuda())
    ref.f8_close(q, s, x.double(), 8 * ref.u)
    assert (q[3].float() == 0).all() and s[3].cpu() == torch.tensor(ref.TINY / ref.F8_MAX)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", LENGTHS)
def test_norm_grad(d, dtype):
    nn = _nn()
    for rows in (1, 5, 70):
        if rows * d > 600000:
            continue
        h, w, dy, g = _data(rows, d, dtype, d + rows)
        dh = torch.randn(rows, d, generator=g).to(dtype)
        for wt in (dtype, torch.float32):
            wc = w.to(wt)
            for more in (None, dh):
                dx, dw = nn.rms_norm_grad(dy.cuda(), h.cuda(), wc.cuda(), dh=None if more is None else more.cuda())
                want_x, want_w = ref.norm_grad(dy, h, wc, dh=more)
                r = (h.double().pow(2).mean(1, keepdim=True) + 1e-6).rsqrt()
                gw = (dy.double() * wc.double()).abs()
                xhat = (h.double() * r).abs()
                size = r * (gw + xhat * (gw * xhat).mean(1, keepdim=True)) + want_x.abs()
                ref.close(dx, want_x, 2 * (2 * TERMS + 16) * ref.u * size, dtype)
                # rows in up to 64 additions a share and 1024 shares, in 32 x 32 steps
                ref.close(dw, want_w, 2 * (TERMS + 160) * ref.u * (dy.double().abs() * xhat).sum(0), wt)


def test_norm_grad_many_rows():
    """More rows than workgroups: shares over several rows, and their sum."""
    nn = _nn()
    for rows, d in ((5000, 40), (4500, 700), (3000, 1500)):
        h, w, dy, _ = _data(rows, d, torch.float32, rows)
        dx, dw = nn.rms_norm_grad(dy.cuda(), h.cuda(), w.cuda())
        want_x, want_w = ref.norm_grad(dy, h, w)
        assert float((dx.cpu().double() - want_x).norm() / want_x.norm()) < 1e-6
        assert float((dw.cpu().double() - want_w).norm() / want_w.norm()) < 2e-6
        y, _ = nn.rms_norm(h.cuda(), w.cuda())
        want = ref.norm(h, w)[0]
        ref.close(y, want, (TERMS + 16) * ref.u * want.abs(), torch.float32)


def test_norm_grad_against_differences():
    """Along random directions: (f(+e) - f(-e)) / 2e in 64 bits against the kernel's inner product."""
    nn = _nn()
    h, w, dy, g = _data(9, 130, torch.float32, 3)
    dx, dw = (t.cpu().double() for t in nn.rms_norm_grad(dy.cuda(), h.cuda(), w.cuda()))
    f = lambda a, b: float((ref.norm(a, b)[0] * dy.double()).sum())  # noqa: E731
    for _ in range(4):
        vh, vw = torch.randn(9, 130, generator=g).double(), torch.randn(130, generator=g).double()
        e = 1e-6
        got = float((dx * vh).sum()), float((dw * vw).sum())
        want = ((f(h.double() + e * vh, w.double()) - f(h.double() - e * vh, w.double())) / (2 * e),
                (f(h.double(), w.double() + e * vw) - f(h.double(), w.double() - e * vw)) / (2 * e))
        for a, b, size in zip(got, want, ((dx * vh).abs().sum(), (dw * vw).abs().sum())):
            assert abs(a - b) <= 1e-5 * float(size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Rows of a wider matrix, one element past a 16-byte boundary, NaN all around."""
    nn = _nn()
    for d in (64, 1111, 4096):
        x, w, r, _ = _data(7, d, dtype, d)
        wide = lambda t: torch.cat([torch.full((7, 1), float("nan")).to(t), t, torch.full((7, 3), float("nan")).to(t)],  # noqa: E731
                                   1).cuda()[:, 1:1 + d]
        wu = torch.cat([w[:1], w]).to(dtype).cuda()[1:]
        y, h = nn.rms_norm(wide(x), wu, residual=wide(r))
        want, hw = ref.norm(x, w.to(dtype), r)
        ref.close(y, want, (TERMS + 16) * ref.u * want.abs(), dtype)
        ref.close(h, hw, ref.u * hw.abs(), dtype)
        dx, dw = nn.rms_norm_grad(wide(r), wide(x), wu, dh=wide(r))
        a, b = nn.rms_norm_grad(r.cuda(), x.cuda(), w.to(dtype).cuda(), dh=r.cuda())
        assert torch.equal(dx, a) and torch.equal(dw, b)


def test_special_rows():
    nn = _nn()
    x = torch.ones(5, 100)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 99] = float("nan")
    w = torch.ones(100)
    y, _ = nn.rms_norm(x.cuda(), w.cuda())
    want = ref.norm(x, w)[0]
    ref.close(y, want, 200 * ref.u * want.abs(), torch.float32)
    q, s, _ = nn.rms_norm(x.cuda(), w.cuda(), quantize=True)
    q = q.float().cpu()
    assert (q[0] == 0).all() and s[0].cpu() == torch.tensor(ref.TINY / ref.F8_MAX)
    assert q[2].isnan().all() and s[2].isnan() and q[1, 7].isnan()
    assert (q[3:] == 448).all()


def test_empty_and_leading_dimensions():
    nn = _nn()
    w = torch.ones(16, device="cuda")
    y, h = nn.rms_norm(torch.empty(0, 16, device="cuda"), w, residual=torch.empty(0, 16, device="cuda"))
    assert y.shape == h.shape == (0, 16)
    dx, dw = nn.rms_norm_grad(torch.empty(0, 16, device="cuda"), torch.empty(0, 16, device="cuda"), w)
    assert dx.shape == (0, 16) and (dw == 0).all()
    x = torch.randn(2, 3, 16, device="cuda")
    y, _ = nn.rms_norm(x, w)
    assert torch.equal(y.view(6, 16), nn.rms_norm(x.view(6, 16), w)[0])
    q, s = nn.quantize_rows(x)
    assert q.shape == x.shape and s.shape == (2, 3)


def test_autograd():
    nn = _nn()
    x, w, r, g = _data(6, 200, torch.float32, 9)
    leaves = [t.clone().cuda().requires_grad_() for t in (x, w, r)]
    y, h = nn.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    gy, gh = torch.randn(6, 200, generator=g), torch.randn(6, 200, generator=g)
    torch.autograd.backward([y, h], [gy.cuda(), gh.cuda()])
    same = [t.clone().double().requires_grad_() for t in (x, w, r)]
    hh = same[0] + same[2]
    yy = hh * (hh.pow(2).mean(1, keepdim=True) + 1e-6).rsqrt() * same[1]
    torch.autograd.backward([yy, hh], [gy.double(), gh.double()])
    for a, b in zip(leaves, same):
        assert float((a.grad.cpu().double() - b.grad).norm() / b.grad.norm()) < 1e-5
