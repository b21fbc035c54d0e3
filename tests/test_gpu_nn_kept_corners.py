"""Activations kept in 8 bits where their groups hold values that have no integer of their own."""

import numpy as np
import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
KIND = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
INF = float("inf")


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.where(a.isnan(), 0, a), torch.where(b.isnan(), 0, b))


def _masked_bytes(x, positive):
    """The definition with minus infinity as the integer -128, which counts for no unit; numpy, in 64 bits."""
    rows, d = x.shape
    groups = -(-d // 32)
    v = np.zeros((rows, groups * 32))
    v[:, :d] = x.double().numpy()
    v = v.reshape(rows, groups, 32)
    masked = v == -np.inf
    v = np.where(masked, 0, v)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(top)
    mantissa, exponent = np.frexp(np.where(bad, 1.0, top))
    e = np.where(top == 0, -126, np.maximum(np.where(mantissa * 128 < 127.5, exponent - 7, exponent - 6), -126))
    codes = np.rint(np.ldexp(np.where(bad[..., None], 0, v), -e[..., None]))
    if positive:
        codes = np.where((v > 0) & (codes < 1), 1, codes)
    codes = np.where(bad[..., None], 0, np.where(masked, -128, codes))
    values = np.where(bad[..., None], np.nan, np.where(masked, -np.inf, np.ldexp(codes, e[..., None])))
    return (torch.cat([torch.from_numpy(codes.astype(np.int8)).reshape(-1).view(torch.uint8),
                       torch.from_numpy(np.where(bad, 255, e + 127).astype(np.uint8)).reshape(-1)]),
            torch.from_numpy(values.reshape(rows, -1)[:, :d]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 5, 32, 96, 100])
def test_minus_infinity_is_kept(d, dtype):
    """Alone, beside finite values (whose unit it does not change), beside plus infinity and NaN, a row and a group of it."""
    nn = _nn()
    g = torch.Generator().manual_seed(d)
    x = torch.randn(9, d, generator=g) * torch.exp(2 * torch.randn(9, d, generator=g))
    x[0, 0], x[1, ::3], x[2], x[3, :32] = -INF, -INF, -INF, -INF
    x[4, -1] = -INF
    if d > 4:
        x[5, 1], x[5, 2] = -INF, INF
        x[6, 3], x[6, 4] = float("nan"), -INF
        x[7, 2] = INF
    x = x.to(dtype)
    for positive in (False, True):
        want, values = _masked_bytes(x, positive)
        kept = nn.keep8(x.cuda(), positive, masked=True)
        assert torch.equal(kept.data.cpu(), want)
        assert _same(kept.restore().cpu().double(), values.to(dtype).double())
        wide = torch.full((9, d + 3), 7.0, dtype=dtype, device="cuda")
        wide[:, 1:1 + d] = x.cuda()
        assert torch.equal(nn.keep8(wide[:, 1:1 + d], positive, masked=True).data.cpu(), want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (70, 96, 64), (64, 77, 33), (300, 520, 136), (512, 512, 512)])
def test_masked_units_have_a_gradient(m, n, k, activation, dtype):
    """Hidden units that the bias masks with minus infinity (or, in float16, a number past its largest): the units beside them have
    the gradient that they have from pre-activations kept in 16 bits, at the kept values; the masked ones none."""
    nn = _nn()
    g = torch.Generator().manual_seed(m + n)
    x = torch.randn(m, k, generator=g).to(dtype).cuda()
    w = (torch.randn(k, n, generator=g) * k ** -0.5).to(dtype).cuda()
    dy = torch.randn(m, n, generator=g).to(dtype).cuda()
    masked = torch.zeros(n, dtype=torch.bool)
    masked[[0, 5, n - 1]] = True
    b = torch.randn(n, generator=g)
    b[masked] = -INF
    if dtype == torch.float16:
        b[5] = -1e5
    leaves = [t.clone().requires_grad_() for t in (x, w, b.cuda())]
    out = nn.linear(*leaves, activation, keep8=True)
    got = torch.autograd.grad(out, leaves, dy)
    with torch.no_grad():
        plain, z = nn.linear(x, w, b.cuda(), activation, keep=True)
        assert torch.equal(out, plain) and (out[:, masked.cuda()] == 0).all()
        assert (z[:, masked.cuda()] == -INF).all() and z[:, ~masked.cuda()].isfinite().all()
        x8, z8 = nn.keep8(x), nn.keep8(z, activation == "relu", masked=True)
        back = z8.restore()
        assert torch.equal(back == -INF, z == -INF) and (activation != "relu" or torch.equal(back > 0, z > 0))
        groups = torch.nn.functional.pad(z.float().where(z > -INF, 0), (0, -n % 32)).view(m, -1, 32)
        unit = torch.exp2((torch.floor(torch.log2(groups.abs().amax(2) / 127.5)) + 1).clamp_min(-126))
        half = 0.5 * unit.repeat_interleave(32, 1)[:, :n]
        fine = ~masked.cuda()
        off = (back.float() - z.float()).abs()
        # relu's smallest codes move a value by up to a whole unit
        assert (off[:, fine] <= half[:, fine] * (2 if activation == "relu" else 1)).all()
        want = nn.linear_grad(dy, x8.restore(), w, back, activation, torch.float32)
    dx, dw, db = got
    assert (dw[:, masked.cuda()] == 0).all() and (db[masked.cuda()] == 0).all()
    xd, wd, zd, dyd = (t.cpu().double() for t in (x8.restore(), w, back, dy))
    slope = torch.where(zd == -INF, torch.zeros_like(zd), ref.slope(zd.clamp_min(-1e4), activation))
    dz = dyd * slope
    off = 2e-6 * dyd.abs() * (zd > -INF)
    rounded = off + (ref.U[dtype] * dz.abs() + ref.FLOOR[dtype])
    size = dz.abs() + rounded
    for one in (got, want):
        ref.close(one[0], dz @ wd.t(), (rounded + (2 * n + 8) * ref.u * size) @ wd.abs().t(), dtype)
        ref.close(one[1], xd.t() @ dz, xd.abs().t() @ (rounded + (2 * m + 8) * ref.u * size), dtype)
        ref.close(one[2], dz.sum(0), (off + (2 * m + 8) * ref.u * size).sum(0), torch.float32)


@pytest.mark.parametrize("dtype", HALF)
def test_minus_infinity_in_kept_inputs(dtype):
    """In a kept x or h it goes where it goes from 16 bits: into its own column of dw, its own row of the norm's gradient."""
    nn = _nn()
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(40, c, generator=g).to(dtype) for c in (64, 72))
    w = torch.randn(64, 72, generator=g).to(dtype).cuda()
    x[7, 9] = -INF
    x8 = nn.keep8(x.cuda(), masked=True)
    a, b = nn.linear_grad(dy.cuda(), x8, w), nn.linear_grad(dy.cuda(), x8.restore(), w)
    assert torch.equal(a[0], b[0]) and _same(a[1], b[1])
    rows = torch.ones(64, dtype=torch.bool, device="cuda")
    rows[9] = False
    assert a[1][rows].isfinite().all() and not a[1][9].isfinite().any()
    nw, dn = torch.ones(64, device="cuda"), torch.randn(40, 64, generator=g).to(dtype).cuda()
    a, b = nn.rms_norm_grad(dn, x8, nw), nn.rms_norm_grad(dn, x8.restore(), nw)
    assert _same(a[0], b[0]) and _same(a[1], b[1])
    assert torch.equal(a[0].isnan().any(1).nonzero().flatten().cpu(), torch.tensor([7]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 70])
def test_finite_values_stay_finite(d, dtype):
    """A group whose largest value rounds to 2^128 (or past 65504) comes back within half a unit, and not as an infinity."""
    nn = _nn()
    info = torch.finfo(dtype)
    x = torch.zeros(6, d, dtype=dtype)
    near = info.max * (1 - info.eps)
    x[0, ::3], x[1, 1::2], x[2, 0], x[3, 5] = info.max, -info.max, info.max, near
    x[4, 7], x[4, 8], x[4, 9] = -near, info.max / 2, -info.max / 3
    x[5, 3], x[5, 4] = info.max, -INF
    unit = 2.0 ** (122 if dtype != torch.float16 else 10)
    for masked in (False, True):
        back = nn.keep8(x.cuda(), masked=masked).restore().cpu()
        rows = slice(0, 6 if masked else 5)
        a, b = back[rows].double(), x[rows].double()
        fine = b > -INF
        assert a[fine].isfinite().all() and (a[fine] - b[fine]).abs().max() <= unit / 2
        assert (a[~fine] == -INF).all()
        assert back[0, 0] == info.max and back[1, 1] == -info.max
    assert nn.keep8(x.cuda()).restore()[5, :32].isnan().all()


@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("m", [40, 300])
def test_gradients_beside_the_largest_number(m, activation):
    """bfloat16's largest number in a kept x that meets a gradient of zero adds nothing to dw; in a kept z it has a slope of 0 or 1."""
    nn = _nn()
    g = torch.Generator().manual_seed(m)
    x, dy, z = (torch.randn(m, c, generator=g).bfloat16() for c in (64, 96, 96))
    w = torch.randn(64, 96, generator=g).bfloat16().cuda()
    top = torch.finfo(torch.bfloat16).max
    x[3, 5], x[3, 40], dy[3] = top, -top, 0
    z[7, 3], z[8, 40] = top, -top
    z[7, :32], z[8, 32:64] = z[7, :32].sign() * top, z[8, 32:64].sign() * top  # the unit is 2^122: only zeros and these are held
    x8, z8 = nn.keep8(x.cuda()), nn.keep8(z.cuda(), activation == "relu")
    got = nn.linear_grad(dy.cuda(), x8, w, z8, activation, torch.float32)
    want = nn.linear_grad(dy.cuda(), x8.restore(), w, z8.restore(), activation, torch.float32)
    slope = (z8.restore() > 0).float()[7, :32].cpu()
    assert torch.equal(slope, (z[7, :32] > 0).float())
    for a, b in zip(got, want):
        assert a.isfinite().all() and torch.equal(a, b)


def test_restored_in_another_type():
    """The C call: what was kept from float32 or bfloat16, in any of the three types."""
    from tensorforge_amd import _lib
    nn = _nn()
    top = torch.finfo(torch.float32).max
    x = torch.zeros(5, 64)
    x[0, 3], x[1, 4], x[2, 5], x[2, 6] = top, -top, -INF, 1.5
    x[3, 7], x[3, 8] = 1e6, -7e4
    x[4, 9], x[4, 40] = float("nan"), 3.0
    for kind in (torch.float32, torch.bfloat16):
        kept = nn.keep8(x.to(kind).cuda(), masked=True)
        values = kept.restore().cpu()
        for dtype in DTYPES:
            out = torch.empty(5, 64, dtype=dtype, device="cuda")
            assert _lib.lib().tf_restore8(kept.data.data_ptr(), 5, 64, KIND[dtype], out.data_ptr(), 64, torch.cuda.current_stream().cuda_stream) == 0
            most = torch.finfo(dtype).max
            want = torch.where(values > -INF, values.double().clamp(-most, most), values.double())
            got = out.cpu().double()
            # the largest of one type may be another's largest: both stand for 2^128
            got, want = (torch.where(t.abs() > 3e38, torch.where(t.isinf(), t, t.sign() * 3e38), t) for t in (got, want))
            assert _same(got, want), (kind, dtype)
            # (bfloat16 rounds float32's largest to plus infinity before it is kept, and its negative to minus infinity)
            assert out[2, 5] == -INF and out[4, :32].isnan().all()
            if kind == torch.float32:
                assert out[0, 3].isfinite() and out[1, 4].isfinite()
            else:
                assert out[0, :32].isnan().all() and out[1, 4] == -INF


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,n,k", [(0, 40, 64), (5, 0, 64), (5, 40, 0), (1, 1, 1), (7, 33, 65), (130, 96, 64)])
def test_autograd_of_every_size(m, n, k, activation):
    """keep8 with and without the kept z's own loss, without rows, columns or a depth, on rows of leading dimensions: the gradients are
    those of the gradient calls at the kept values."""
    nn = _nn()
    g = torch.Generator().manual_seed(m + n + k)
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
    x, w, b, r = make(1, m, k), make(k, n), make(n), make(m, n)
    dy, dz = make(1, m, n), make(1, m, n)
    for keep in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        got = nn.linear(leaves[0], leaves[1], leaves[2], activation, leaves[3], keep=keep, keep8=True)
        outs, ups = (list(got), [dy, dz]) if keep else ([got], [dy])
        grads = torch.autograd.grad(outs, leaves, ups)
        with torch.no_grad():
            out, z = nn.linear(x, w, b, activation, r, keep=True)
            assert torch.equal(outs[0], out) and (not keep or torch.equal(outs[1], z))
            x8, z8 = nn.keep8(x, masked=True), nn.keep8(z, activation == "relu", masked=True)
            want = nn.linear_grad(dy, x8, w, None if activation == "none" else z8, activation, torch.bfloat16)
            if keep:
                want = [p + q for p, q in zip(want, nn.linear_grad(dz, x8, w, bias_dtype=torch.bfloat16))]
        for p, q in zip(grads, (*want, dy.view(m, n))):
            assert torch.equal(p, q) and not p.isnan().any()
    nw = torch.ones(k, device="cuda", requires_grad=True)
    h = x.clone().requires_grad_()
    y, _ = nn.rms_norm(h, nw, keep8=True)
    a = torch.autograd.grad(y, [h, nw], make(1, m, k).mul_(0).add_(1))
    with torch.no_grad():
        c = nn.rms_norm_grad(torch.ones_like(x), nn.keep8(x), nw)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
