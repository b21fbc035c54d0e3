"""The loss over a vocabulary and its gradient against 64-bit references: every tile and
loader, both memory orders, one row to several tiles, several pieces, rows that do not count, odd
sizes and strides, special values, streams and graphs."""

import ctypes

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
IGNORE = -100


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _matrix(g, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=g) * scale).to(dtype)


def _ordered(w, order):
    return w.cuda() if order == 0 else w.t().contiguous().cuda().t()


def _data(m, n, k, dtype, ignored=0.2, scale=2.0, seed=0):
    g = torch.Generator().manual_seed(m + 3 * n + 7 * k + seed)
    x, w = _matrix(g, m, k, dtype), _matrix(g, k, n, dtype, scale * k ** -0.5)
    target = torch.randint(0, n, (m,), generator=g)
    if m > 1:
        target[torch.rand(m, generator=g) < ignored] = IGNORE
        target[0] = n - 1
        target[-1] = 0
    return x, w, target, g


def _loss_want(x, w, target):
    """loss, lse, and what float32 may lose: 2k+8 roundings of the logits' products; the exponentials' sum is off by a few
    roundings of its values (an ulp of the exponential, the argument's rounding, additions in a tree of at most 64 + 16 + n/4096
    steps), the logarithm and the subtraction by one each."""
    x, w = x.double(), w.double()
    z = x @ w
    size = x.abs() @ w.abs()
    off_z = ((2 * x.shape[1] + 8) * ref.u * size).amax(1)
    lse = torch.logsumexp(z, 1)
    spread = (z.amax(1) - z.amin(1)).clamp_min(0)
    off = off_z + ref.u * (spread * 2 + 128 + w.shape[1] / 4096 + 4 * lse.abs())
    counts = target != IGNORE
    at = target.clamp_min(0)
    loss = torch.where(counts, lse - z[torch.arange(len(target)), at], torch.zeros_like(lse))
    return z, loss, lse, off, off + off_z + 2 * ref.u * lse.abs()


def _check_loss(loss, lse, x, w, target):
    z, want, want_lse, off, off_loss = _loss_want(x, w, target)
    ref.close(lse, want_lse, off, torch.float32)
    ref.close(loss, want, off_loss, torch.float32)
    return z, want_lse


def _check_grad(dx, dw, dloss, x, w, target, z, lse, dtype):
    """dz = (p - [target]) * dloss off by its rounding to dtype (float16: 2^-39 of the largest dloss besides, half the spacing
    2^-24 of the smallest numbers where the largest is 2^14 at least) and the logits', lse's and exponential's errors (relative to p); sums as linear_grad's."""
    x, w, dloss = x.double(), w.double(), dloss.double().expand(len(target))
    m, k = x.shape
    n = w.shape[1]
    counts = (target != IGNORE)[:, None]
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p)
    hot[torch.arange(m), target.clamp_min(0)] = 1
    d = torch.where(counts, (p - hot) * dloss[:, None], torch.zeros_like(p))
    off_z = (2 * k + 8) * ref.u * (x.abs() @ w.abs())
    rel = 2 * off_z + ref.u * (2 * (z - lse[:, None]).abs() + 128 + n / 4096 + 6 * lse.abs()[:, None] + 16)
    small = 2.0 ** -39 * dloss.abs().max() if dtype == torch.float16 else 2.0 ** -133
    off = torch.where(counts, (p * rel + 4 * ref.u * (p - hot).abs()) * dloss.abs()[:, None], torch.zeros_like(p))
    off = off + (ref.U[dtype] * (d.abs() + off) + small) * counts
    size = d.abs() + off
    if dx is not None:
        ref.close(dx, d @ w.t(), (off + (2 * n + 8) * ref.u * size) @ w.abs().t(), dtype)
    if dw is not None:
        ref.close(dw, x.t() @ d, x.abs().t() @ (off + (2 * m + 8) * ref.u * size), dtype)


SHAPES = [(1, 1, 1), (1, 5, 64), (3, 64, 8), (2, 7, 5), (16, 130, 72), (64, 1000, 128), (65, 257, 200), (130, 64, 264), (61, 1001, 333),
          (300, 520, 96), (257, 1032, 520), (70, 3000, 64)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_loss_and_gradient(m, n, k, order, dtype):
    nn = _nn()
    x, w, target, g = _data(m, n, k, dtype)
    xc, wc, tc = x.cuda(), _ordered(w, order), target.cuda()
    loss, lse, none = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)
    assert none is None and loss.dtype == torch.float32 and lse.dtype == torch.float64
    z, want_lse = _check_loss(loss, lse, x, w, target)
    counts = int((target != IGNORE).sum())
    mean, _, count = nn.linear_cross_entropy(xc, wc, tc, keep=True)
    total = nn.linear_cross_entropy(xc, wc, tc, reduction="sum")
    rows = loss.double().sum()
    bound = 40 * ref.u * loss.double().abs().sum()  # additions in a tree, one after the other in a thread: up to 16 + 16 + m/1024
    assert abs(total.double() - rows) <= bound and count == counts and mean.shape == total.shape == ()
    assert abs(mean.double() * max(1, counts) - rows) <= 2 * bound
    dloss = torch.randn(m, generator=g)
    dx, dw = nn.linear_cross_entropy_grad(dloss.cuda(), xc, wc, tc, lse)
    assert dw.stride() == wc.stride() or 1 in w.shape
    _check_grad(dx, dw, dloss, x, w, target, z, want_lse, dtype)
    one = torch.tensor(0.7)
    dx, dw = nn.linear_cross_entropy_grad(one.cuda(), xc, wc, tc, lse, count)
    _check_grad(dx, dw, one / max(1, counts), x, w, target, z, want_lse, dtype)
    assert nn.linear_cross_entropy_grad(one.cuda(), xc, wc, tc, lse, count, want_dw=False)[1] is None
    a, b = nn.linear_cross_entropy_grad(one.cuda(), xc, wc, tc, lse, count, want_dx=False)
    assert a is None and torch.equal(b, dw)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("m,n,k", [(512, 17000, 128), (4100, 2056, 256), (2048, 4096, 1024), (40, 20001, 2048)])
def test_large(m, n, k, order, dtype):
    """Sizes that take the larger tiles, and splits of k in the gradient's products; against float64 on the GPU."""
    nn = _nn()
    x, w, target, g = _data(m, n, k, dtype)
    xc, wc, tc = x.cuda(), _ordered(w, order), target.cuda()
    loss, lse, count = nn.linear_cross_entropy(xc, wc, tc, keep=True)
    xd, wd = xc.double(), wc.double().contiguous()
    z = torch.matmul(xd, wd)
    want = torch.logsumexp(z, 1)
    assert float((lse.double() - want).abs().max()) < 1e-4
    counts = tc != IGNORE
    rows = torch.where(counts, want - z[torch.arange(m), tc.clamp_min(0)], torch.zeros_like(want))
    assert abs(float(loss) - float(rows.sum() / counts.sum())) < 1e-5
    dx, dw = nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), xc, wc, tc, lse, count)
    d = torch.exp(z - want[:, None])
    d[torch.arange(m), tc.clamp_min(0)] -= 1
    d *= (counts / counts.sum())[:, None]
    for got, full in ((dx, torch.matmul(d, wd.t().contiguous())), (dw, torch.matmul(xd.t().contiguous(), d))):
        # in the norm: the results' rounding and dz's, half a step each at most (uniform: 1/sqrt(3) of that), and what
        # float16 drops of results below its normal numbers
        err = float((got.double() - full).norm()) - (2.0 ** -25 * full.numel() ** 0.5 if dtype == torch.float16 else 0)
        assert err < 1.5 * ref.U[dtype] * float(full.norm())




@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("n", [50000, 33001])
def test_pieces_of_the_vocabulary(n, order, dtype):
    """Rows enough that the vocabulary goes in several pieces, the last one narrower: dx is added up over them."""
    nn = _nn()
    m, k = 16500, 72
    x, w, target, g = _data(m, n, k, dtype, scale=1.0)
    xc, wc, tc = x.cuda(), _ordered(w, order), target.cuda()
    lse = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)[1]
    dloss = torch.rand(m, generator=g).cuda() + 0.5
    dx, dw = nn.linear_cross_entropy_grad(dloss, xc, wc, tc, lse)
    xd, wd = xc.double(), wc.double().contiguous()
    want_dx, want_dw = torch.zeros(m, k, dtype=torch.float64, device="cuda"), torch.zeros(k, n, dtype=torch.float64, device="cuda")
    for i in range(0, m, 4125):
        z = torch.matmul(xd[i:i + 4125], wd)
        d = torch.exp(z - torch.logsumexp(z, 1)[:, None])
        at = tc[i:i + 4125]
        d[torch.arange(len(at)), at.clamp_min(0)] -= 1
        d *= (dloss[i:i + 4125] * (at != IGNORE))[:, None]
        want_dx[i:i + 4125] = torch.matmul(d, wd.t().contiguous())
        want_dw += torch.matmul(xd[i:i + 4125].t().contiguous(), d)
        del z, d
    for got, full in ((dx, want_dx), (dw, want_dw)):
        err = float((got.double() - full).norm()) - (2.0 ** -25 * full.numel() ** 0.5 if dtype == torch.float16 else 0)
        assert err < 1.5 * ref.U[dtype] * float(full.norm())
        rows = (got.double() - full).norm(dim=0 if got is dw else 1)
        size = full.norm(dim=0 if got is dw else 1)
        assert bool((rows <= 4 * ref.U[dtype] * size + 2.0 ** -20).all())  # no column or row of another piece
    assert (dx[tc == IGNORE] == 0).all()


def test_against_differences():
    """Along random directions, in 64 bits, against the inner product with the kernels' gradient."""
    nn = _nn()
    m, n, k = 30, 150, 40
    x, w, target, g = _data(m, n, k, torch.bfloat16)
    xc, wc, tc = x.cuda(), w.cuda(), target.cuda()
    loss, lse, count = nn.linear_cross_entropy(xc, wc, tc, keep=True)
    dx, dw = (t.cpu().double() for t in nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), xc, wc, tc, lse, count))

    def f(a, b):
        z = a @ b
        counts = target != IGNORE
        return float((torch.logsumexp(z, 1) - z[torch.arange(m), target.clamp_min(0)])[counts].mean())

    for _ in range(4):
        vx, vw = torch.randn(m, k, generator=g).double(), torch.randn(k, n, generator=g).double()
        e = 1e-5
        for got, v, want in ((dx, vx, (f(x.double() + e * vx, w.double()) - f(x.double() - e * vx, w.double())) / (2 * e)),
                             (dw, vw, (f(x.double(), w.double() + e * vw) - f(x.double(), w.double() - e * vw)) / (2 * e))):
            # two roundings of 2^-8 at most, of either sign: the root of the sum of squares, four of them
            assert abs(float((got * v).sum()) - want) <= 4 * 2 ** 0.5 * 2.0 ** -8 * float((got * v).norm())


@pytest.mark.parametrize("dtype", HALF)
def test_rows_that_do_not_count(dtype):
    """All of them, none, a class as the index to ignore; targets outside of the vocabulary."""
    nn = _nn()
    x, w, target, g = _data(70, 300, 64, dtype, ignored=0)
    xc, wc, tc = x.cuda(), w.cuda(), target.cuda()
    none = torch.full_like(tc, IGNORE)
    loss, lse, count = nn.linear_cross_entropy(xc, wc, none, keep=True)
    assert loss == 0 and count == 0 and nn.linear_cross_entropy(xc, wc, none, reduction="sum") == 0
    dx, dw = nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), xc, wc, none, lse, count)
    assert (dx == 0).all() and (dw == 0).all()
    ones = torch.where(torch.arange(70) % 3 == 0, torch.full_like(target, 17), target)
    rows = nn.linear_cross_entropy(xc, wc, ones.cuda(), ignore_index=17, reduction="none")
    want = nn.linear_cross_entropy(xc, wc, torch.where(ones == 17, torch.full_like(ones, IGNORE), ones).cuda(), reduction="none")
    assert torch.equal(rows, want) and (rows[::3] == 0).all()
    bad = target.clone()
    bad[3], bad[5], bad[9], bad[11] = 300, -1, 1 << 40, -(1 << 63)
    rows, lse, _ = nn.linear_cross_entropy(xc, wc, bad.cuda(), reduction="none", keep=True)
    wrong = torch.zeros(70, dtype=torch.bool)
    wrong[[3, 5, 9, 11]] = True
    assert torch.equal(rows.isnan().cpu(), wrong) and not lse.isnan().any()
    dx, dw = nn.linear_cross_entropy_grad(torch.ones(70, device="cuda"), xc, wc, bad.cuda(), lse)
    assert torch.equal(dx.isnan().any(1).cpu(), wrong) and dx[wrong.cuda()].isnan().all() and dw.isnan().all()


def test_special_values():
    """An infinity or a NaN stays in its row of the loss and of dx; a row that does not count gives zeros there."""
    nn = _nn()
    x, w, target, g = _data(80, 400, 64, torch.bfloat16, ignored=0)
    x[4, 3], x[7, 5], x[9, 0] = float("inf"), float("nan"), float("nan")
    target[9] = IGNORE
    xc, wc, tc = x.cuda(), w.cuda(), target.cuda()
    rows, lse, _ = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)
    bad = torch.zeros(80, dtype=torch.bool)
    bad[[4, 7]] = True
    assert torch.equal(rows.isnan().cpu(), bad) and rows[9] == 0
    dx, _ = nn.linear_cross_entropy_grad(torch.ones(80, device="cuda"), xc, wc, tc, lse, want_dw=False)
    assert torch.equal(dx.isnan().any(1).cpu(), bad) and (dx[9] == 0).all()
    # logits of minus infinity (a masked class): probability 0 and no gradient
    x = torch.ones(5, 8, dtype=torch.bfloat16)
    w = torch.zeros(8, 300, dtype=torch.bfloat16)
    w[0, ::2] = float("-inf")
    t = torch.tensor([1, 3, 5, 299, 7])
    rows, lse, _ = nn.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), reduction="none", keep=True)
    assert ((lse - torch.log(torch.tensor(150.0, device="cuda"))).abs() < 1e-5).all() and torch.allclose(rows.double(), lse, rtol=2 ** -23)
    _, dw = nn.linear_cross_entropy_grad(torch.ones(5, device="cuda"), x.cuda(), w.cuda(), t.cuda(), lse, want_dx=False)
    assert (dw[:, ::2] == 0).all() and not dw.isnan().any()
    # large logits: their difference counts
    w = torch.zeros(8, 70, dtype=torch.bfloat16)
    w[:, 0], w[:, 1] = 1e4, 1e4
    rows = nn.linear_cross_entropy(x[:2].cuda(), w.cuda(), torch.tensor([0, 2]).cuda(), reduction="none")
    top = 8 * 9984.0  # bfloat16 holds 1e4 as 9984; float32's spacing is 2^-7 there
    assert abs(float(rows[0]) - 0.6931472) < 1e-2 and abs(float(rows[1]) - top - 0.6931472) < 1e-2


@pytest.mark.parametrize("power", [-100, -8, 8, 100])
def test_dloss_of_any_size_in_float16(power):
    """dz's unit follows the largest dloss: with dloss times a power of two the results are the same numbers times it, where they
    are float16's normal numbers."""
    nn = _nn()
    x, w, target, g = _data(60, 200, 64, torch.float16)
    xc, wc, tc = x.cuda(), w.cuda(), target.cuda()
    lse = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)[1]
    dloss = torch.randn(60, generator=g).cuda()
    dx, dw = nn.linear_cross_entropy_grad(dloss * 2.0 ** power, xc, wc, tc, lse)
    a, b = nn.linear_cross_entropy_grad(dloss, xc, wc, tc, lse)
    for got, one in ((dx, a), (dw, b)):
        want = one.double() * 2.0 ** power
        normal = (one.abs() >= 2.0 ** -14) & (want.abs() >= 2.0 ** -14) & (want.abs() <= 65504)
        assert torch.equal(got.double()[normal], want[normal]) and not got.isnan().any()
        assert got[(one.abs() >= 2.0 ** -14) & (want.abs() > 65536)].isinf().all() and (got[want.abs() < 2.0 ** -26] == 0).all()
        assert abs(power) == 100 or normal.sum() > 1000


@pytest.mark.parametrize("order", [0, 1])
def test_strides_alignment_and_neighbours(order):
    """Operands off a boundary inside NaN; results inside a wider matrix (the C call)."""
    from tensorforge_amd import _lib
    nn = _nn()
    for m, n, k in ((5, 40, 64), (70, 333, 72), (130, 301, 77)):
        x, w, target, g = _data(m, n, k, torch.bfloat16)
        wc, tc = _ordered(w, order), target.cuda()
        nan = lambda r, c: torch.full((r, c), float("nan")).bfloat16()  # noqa: E731
        wide = torch.cat([nan(m, 1), x, nan(m, 3)], 1).cuda()[:, 1:1 + k]
        lines = w if order == 0 else w.t()
        w_wide = torch.cat([nan(lines.shape[0], 3), lines, nan(lines.shape[0], 2)], 1).cuda()[:, 3:3 + lines.shape[1]]
        w_wide = w_wide if order == 0 else w_wide.t()
        loss, lse, _ = nn.linear_cross_entropy(wide, w_wide, tc, reduction="none", keep=True)
        z, want_lse = _check_loss(loss, lse, x, w, target)
        dloss = torch.rand(m, generator=g)
        dx, dw = nn.linear_cross_entropy_grad(dloss.cuda(), wide, w_wide, tc, lse)
        _check_grad(dx, dw, dloss, x, w, target, z, want_lse, torch.bfloat16)
        outs = [torch.full((r, c + 9), 3.0, dtype=torch.bfloat16, device="cuda") for r, c in ((m, k), lines.shape)]
        d = dloss.cuda()
        a = _lib.LinearXentGradArgs(x=wide.data_ptr(), w=w_wide.data_ptr(), target=tc.data_ptr(), lse=lse.data_ptr(), dloss=d.data_ptr(),
                                    dx=outs[0][:, 1:].data_ptr(), dw=outs[1][:, 1:].data_ptr(), x_ld=k + 4, w_ld=lines.shape[1] + 5,
                                    dx_ld=k + 9, dw_ld=lines.shape[1] + 9, m=m, n=n, k=k, ignore=IGNORE, w_order=order, type=1, dloss_rows=1)
        size = ctypes.c_longlong()
        assert _lib.lib().tf_linear_xent_grad_workspace(ctypes.byref(a), ctypes.byref(size)) == 0
        space = torch.full((size.value + 64,), 0xff, dtype=torch.uint8, device="cuda")  # NaN
        a.workspace, a.workspace_bytes = space.data_ptr(), size.value
        assert _lib.lib().tf_linear_xent_grad(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        assert (space[size.value:] == 0xff).all()
        for out, want, c in ((outs[0], dx, k), (outs[1], dw if order == 0 else dw.t(), lines.shape[1])):
            assert torch.equal(out[:, 1:1 + c], want)
            assert (out[:, 0] == 3).all() and (out[:, 1 + c:] == 3).all()


def test_leading_dimensions_and_empty_sizes():
    nn = _nn()
    x, w, target, g = _data(24, 100, 32, torch.bfloat16)
    xc, wc, tc = x.cuda(), w.cuda(), target.cuda()
    rows, lse, _ = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)
    r3, l3, _ = nn.linear_cross_entropy(xc.view(2, 12, 32), wc, tc.view(2, 12), reduction="none", keep=True)
    assert torch.equal(r3.view(24), rows) and r3.shape == (2, 12)
    d = torch.rand(24, generator=g).cuda()
    dx, dw = nn.linear_cross_entropy_grad(d.view(2, 12), xc.view(2, 12, 32), wc, tc.view(2, 12), l3)
    a, b = nn.linear_cross_entropy_grad(d, xc, wc, tc, lse)
    assert torch.equal(dx.view(24, 32), a) and torch.equal(dw, b)
    one = nn.linear_cross_entropy(xc[0], wc, tc[0])
    assert one.shape == () and torch.equal(one, rows[0])
    for dtype in HALF:
        e, v = xc[:0].to(dtype), wc.to(dtype)
        loss, lse, count = nn.linear_cross_entropy(e, v, tc[:0], keep=True)
        assert loss == 0 and count == 0 and lse.shape == (0,)
        dx, dw = nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), e, v, tc[:0], lse, count)
        assert dx.shape == (0, 32) and (dw == 0).all() and dw.shape == (32, 100)
        flat, lse, count = nn.linear_cross_entropy(xc[:, :0].to(dtype), v[:0], tc, keep=True)
        assert abs(float(flat) - 4.6051702) < 1e-5
        dx, dw = nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), xc[:, :0].to(dtype), v[:0], tc, lse, count)
        assert dx.shape == (24, 0) and dw.shape == (0, 100)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(reduction):
    nn = _nn()
    x, w, target, g = _data(50, 200, 64, torch.bfloat16)
    weight = w.t().contiguous().cuda().requires_grad_()
    xc = x.cuda().requires_grad_()
    loss = nn.linear_cross_entropy(xc, weight.t(), target.cuda(), reduction=reduction)
    up = torch.rand(loss.shape, generator=g).cuda() if reduction == "none" else torch.tensor(0.5, device="cuda")
    loss.backward(up)
    with torch.no_grad():
        _, lse, count = nn.linear_cross_entropy(xc, weight.t(), target.cuda(), reduction=reduction, keep=True)
        dx, dw = nn.linear_cross_entropy_grad(up, xc, weight.t(), target.cuda(), lse, count)
    assert torch.equal(xc.grad, dx) and torch.equal(weight.grad, dw.t())
    frozen = nn.linear_cross_entropy(xc, w.cuda(), target.cuda())
    a, = torch.autograd.grad(frozen, xc)
    assert a.shape == xc.shape
    loss, lse, count = nn.linear_cross_entropy(xc, w.cuda(), target.cuda(), keep=True)
    assert loss.requires_grad and not lse.requires_grad and not count.requires_grad
    expanded, = torch.autograd.grad(nn.linear_cross_entropy(xc, w.cuda(), target.cuda(), reduction="none").sum(), xc)
    assert not expanded.isnan().any()
    g2, = torch.autograd.grad(nn.linear_cross_entropy(xc, w.cuda(), target.cuda()), xc, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g2.float().pow(2).sum().backward()


def test_streams_and_graphs():
    """The step on another stream, and in a graph replayed with other inputs; equal calls give equal bits."""
    nn = _nn()
    m, n, k = 200, 700, 136

    def step(x, w, t):
        loss, lse, count = nn.linear_cross_entropy(x, w, t, keep=True)
        return (loss, *nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), x, w, t, lse, count))

    inputs = [[v.cuda() for v in _data(m, n, k, torch.float16, seed=s)[:3]] for s in range(4)]
    want = [step(*i) for i in inputs]
    assert all(torch.equal(a, b) for a, b in zip(step(*inputs[0]), want[0]))
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


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,n,k", [(1, 70, 64), (2, 4000, 136), (30, 1001, 77), (64, 520, 264)])
def test_gradients_of_few_rows_round_once(m, n, k, dtype):
    """Up to 64 rows dz goes in two terms: its rounding (2^-8 or 2^-11) squared is left beside the results' own."""
    nn = _nn()
    x, w, target, g = _data(m, n, k, dtype, ignored=0)
    for order in (0, 1):
        xc, wc, tc = x.cuda(), _ordered(w, order), target.cuda()
        lse = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)[1]
        dloss = torch.randn(m, generator=g)
        dx, dw = nn.linear_cross_entropy_grad(dloss.cuda(), xc, wc, tc, lse)
        xd, wd = x.double(), w.double()
        z = xd @ wd
        p = torch.exp(z - torch.logsumexp(z, 1)[:, None])
        p[torch.arange(m), target] -= 1
        d = p * dloss.double()[:, None]
        # dz's error: its second rounding, and what float32 loses of the logits, lse and the exponential (as _check_grad)
        lost = 2 * (2 * k + 8) * ref.u * (xd.abs() @ wd.abs()) + ref.u * (2 * z.abs() + 144 + n / 4096 + 30)
        small = 2.0 ** -39 * dloss.abs().max().double() if dtype == torch.float16 else 2.0 ** -133
        off = (p.abs() + (p < 0)) * lost * dloss.double().abs()[:, None] + 2 * ref.U[dtype] ** 2 * d.abs() + small
        ref.close(dx, d @ wd.t(), (off + (2 * n + 8) * ref.u * d.abs()) @ wd.abs().t(), dtype)
        ref.close(dw, xd.t() @ d, xd.abs().t() @ (off + (2 * m + 8) * ref.u * d.abs()), dtype)


def test_a_captured_step():
    """Forward and backward through autograd in one graph, after a warm-up on another stream; replays with other inputs and eager
    steps of other leaves between them."""
    nn = _nn()
    m, n, k = 96, 300, 64

    def step(x, w, t):
        loss = nn.linear_cross_entropy(x, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    inputs = [[v.cuda() for v in _data(m, n, k, torch.bfloat16, seed=s)[:3]] for s in range(3)]
    eager = [step(x.clone().requires_grad_(), w.clone().requires_grad_(), t) for x, w, t in inputs]
    x, w, t = (v.clone() for v in inputs[0])
    x.requires_grad_(), w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, t)
    for (a, b, c), want in zip(inputs, eager):
        with torch.no_grad():
            x.copy_(a), w.copy_(b), t.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        step(a.clone().requires_grad_(), b.clone().requires_grad_(), c)


@pytest.mark.parametrize("order", [0, 1])
def test_far_offsets(order):
    """Weights of more than 2^31 elements: classes at both ends and around 2^31, in the loss and in dw."""
    nn = _nn()
    n, k = (1 << 20) + 40, 2056
    w = torch.zeros((n, k) if order else (k, n), dtype=torch.bfloat16, device="cuda")
    at = [0, 1, (1 << 31) // k - 1, (1 << 31) // k, (1 << 31) // k + 1, n // 2, n - 2, n - 1]
    g = torch.Generator().manual_seed(1)
    x = _matrix(g, 8, k, torch.bfloat16).cuda()
    rows = _matrix(g, 8, k, torch.bfloat16, k ** -0.5).cuda()
    for i, c in enumerate(at):
        (w if order else w.t())[c] = rows[i]
    wc = w.t() if order else w
    target = torch.tensor(at, device="cuda")
    loss, lse, _ = nn.linear_cross_entropy(x, wc, target, reduction="none", keep=True)
    z = x.double() @ rows.double().t().contiguous()  # the other classes' logits are 0
    want = torch.log(torch.exp(z).sum(1) + (n - 8))
    assert ((lse.double() - want).abs() < 2e-5).all()
    assert ((loss.double() - (want - z.diagonal())).abs() < 4e-5).all()
    one = torch.ones(8, device="cuda")
    dx, dw = nn.linear_cross_entropy_grad(one, x, wc, target, lse)
    p = torch.exp(z - want[:, None]) - torch.eye(8, dtype=torch.float64, device="cuda")
    full = p @ rows.double()
    assert float((dx.double() - full).norm() / full.norm()) < 2.0 ** -8
    part = p.t().contiguous() @ x.double()
    cols = dw.t()[target].double()
    assert float((cols - part).norm() / part.norm()) < 2.0 ** -8
    other = torch.exp(-want) @ x.double()
    for c in (2, (1 << 31) // k + 2, n - 3):
        assert float((dw.t()[c].double() - other).norm() / other.norm()) < 2.0 ** -8
    del w, wc, dw, dx
    torch.cuda.empty_cache()


def test_a_large_gradient_of_the_logits():
    """A piece whose gradient of the logits holds more than 2^31 elements: the ends of the rows, and what they add to dw."""
    nn = _nn()
    m, n, k = 270000, 16384, 64  # two pieces of 8192 classes
    g = torch.Generator().manual_seed(2)
    w = _matrix(g, k, n, torch.bfloat16, k ** -0.5).cuda()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, (1 << 31) // 8192 - 1, (1 << 31) // 8192, (1 << 31) // 8192 + 1, m - 2, m - 1])
    x[rows] = _matrix(g, len(rows), k, torch.bfloat16).cuda()
    target = torch.full((m,), IGNORE, device="cuda")
    target[rows] = torch.tensor([0, 5, 100, 8000, 16000, 16382, 16383], device="cuda")
    loss, lse, _ = nn.linear_cross_entropy(x, w, target, reduction="none", keep=True)
    dx, dw = nn.linear_cross_entropy_grad(torch.ones(m, device="cuda"), x, w, target, lse)
    z = x[rows].double() @ w.double()
    d = torch.exp(z - torch.logsumexp(z, 1)[:, None])
    d[torch.arange(len(rows)), target[rows]] -= 1
    full = d @ w.double().t().contiguous()
    assert float((dx[rows].double() - full).norm() / full.norm()) < 2.0 ** -8
    full = x[rows].double().t().contiguous() @ d
    assert float((dw.double() - full).norm() / full.norm()) < 2.0 ** -8
    dead = torch.ones(m, dtype=torch.bool, device="cuda")
    dead[rows] = False
    assert (dx[dead] == 0).all() and (loss[dead] == 0).all()
    del dx, dw
    torch.cuda.empty_cache()


@pytest.mark.parametrize("order", [0, 1])
def test_operands_far_apart(order):
    """Rows whose distance puts the last ones past 2^31 elements."""
    nn = _nn()
    m, n, k = (70, 300, 66) if order == 0 else (70, 69, 130)
    x, w, target, g = _data(m, n, k, torch.bfloat16)
    lines = w if order == 0 else w.t()
    ld = (1 << 25) + 8
    memory = torch.empty(70 * ld, dtype=torch.bfloat16, device="cuda")
    xf = memory.as_strided((m, k), (ld, 1), 0)
    wf = memory.as_strided(tuple(lines.shape), (ld, 1), 1024)
    xf.copy_(x), wf.copy_(lines)
    wc, tc = wf if order == 0 else wf.t(), target.cuda()
    loss, lse, _ = nn.linear_cross_entropy(xf, wc, tc, reduction="none", keep=True)
    z, want_lse = _check_loss(loss, lse, x, w, target)
    dloss = torch.rand(m, generator=g)
    dx, dw = nn.linear_cross_entropy_grad(dloss.cuda(), xf, wc, tc, lse)
    _check_grad(dx, dw, dloss, x, w, target, z, want_lse, torch.bfloat16)
    x8 = nn.keep8(xf)
    assert torch.equal(x8.data, nn.keep8(x.cuda()).data)
    dy = _matrix(g, m, n, torch.bfloat16).cuda()
    got = nn.linear_grad(dy, x8, wc, None)
    near = nn.linear_grad(dy, x8.restore(), _ordered(w, order), None)
    for a, b in zip(got[:2], near[:2]):
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2.0 ** -8
    del memory, xf, wf
    torch.cuda.empty_cache()


@pytest.mark.parametrize("size", [1, 8, 60])
def test_small_losses_of_large_logits(size):
    """A row that is sure of its class: the loss is the sum of the others' exponentials, however large the logits are."""
    nn = _nn()
    m, n, k = 40, 300, 64
    g = torch.Generator().manual_seed(size)
    x, w = torch.zeros(m, k), torch.zeros(k, n)
    x[:, 0], w[0] = size, 8.0  # exact logits of 8 * size for every class, beside
    x[:, 1] = torch.arange(m) * 0.5
    w[1, 7] = 1.0  # 0 to 19.5 more for the seventh
    x[:, 2], w[2] = 0.25, torch.randint(-4, 5, (n,), generator=g).float()
    x, w = x.bfloat16(), w.bfloat16()
    z = x.double() @ w.double()
    target = torch.full((m,), 7)
    others = z - z[:, 7:8]
    others[:, 7] = float("-inf")
    want = torch.log1p(torch.exp(others).sum(1))
    loss, lse, _ = nn.linear_cross_entropy(x.cuda(), w.cuda(), target.cuda(), reduction="none", keep=True)
    # sums of 300 exponentials in a tree, then a logarithm and a product: a few roundings of a value of 1 to 400
    off = (loss.cpu().double() - want).abs()
    assert (off <= 16 * ref.u * (1 + want)).all(), off.max()
    # and the gradient: the target's -(1 - p) is off by its rounding and a few roundings of 1, the others' by relative ones
    dx, _ = nn.linear_cross_entropy_grad(torch.ones(m, device="cuda"), x.cuda(), w.cuda(), target.cuda(), lse)
    p = torch.softmax(z, 1)
    d = p.clone()
    d[:, 7] = -(torch.exp(others).sum(1) / (1 + torch.exp(others).sum(1)))
    lost = 64 * ref.u * p + 2 * 2.0 ** -16 * d.abs()
    full = d @ w.double().t()
    ref.close(dx, full, (lost + (2 * n + 8) * ref.u * d.abs()) @ w.double().abs().t(), torch.bfloat16)


def test_totals_of_many_rows():
    """Sums over rows that a float sum would lose parts of."""
    nn = _nn()
    m = 3_000_001
    x = torch.zeros(m, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(8, 3, dtype=torch.bfloat16, device="cuda")
    target = torch.zeros(m, dtype=torch.int64, device="cuda")
    target[1::2] = IGNORE
    mean, _, count = nn.linear_cross_entropy(x, w, target, keep=True)
    total = nn.linear_cross_entropy(x, w, target, reduction="sum")
    row = float(nn.linear_cross_entropy(x[0], w, target[0]))
    assert float(count) == 1_500_001 and abs(float(mean) - row) <= 2 * ref.u * row and abs(float(total) - 1_500_001 * row) <= 4 * ref.u * 1_500_001 * row


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    nn = _nn()
    x, w, target, g = _data(6, 40, 16, torch.bfloat16)
    with fwd.dual_level():
        for at in (0, 1):
            a = [x.cuda(), w.cuda()]
            a[at] = fwd.make_dual(a[at], torch.ones_like(a[at]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError)):
                    nn.linear_cross_entropy(*a, target.cuda())
