"""The loss over a vocabulary where its logits are at the ends of float32, and its gradient in two terms over several pieces."""

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
IGNORE = -100
INF = float("inf")


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("classes", [40, 1000])
def test_logits_at_the_ends_of_float32(classes, rows):
    """Masked classes of minus infinity or bfloat16's lowest value add nothing; a row of nothing else has no loss."""
    nn = _nn()
    low = torch.finfo(torch.bfloat16).min
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[1:, 1] = 1, 1
    target = torch.full((rows,), 7, device="cuda")
    for lowest in (low, -INF):
        w = torch.zeros(8, classes, dtype=torch.bfloat16, device="cuda")
        w[0, ::2] = lowest
        loss, lse, _ = nn.linear_cross_entropy(x, w, target, reduction="none", keep=True)
        want = torch.log(torch.tensor(classes / 2, dtype=torch.float64))
        assert ((loss.cpu().double() - want).abs() <= 16 * ref.u * want).all() and ((lse.cpu() - want).abs() <= 16 * ref.u * want).all()
        dx, dw = nn.linear_cross_entropy_grad(torch.ones(rows, device="cuda"), x, w, target, lse, want_dx=False)
        assert dw.isfinite().all() and (dw[:, ::2] == 0).all()
        w[0] = lowest
        for order in (0, 1):
            wc = w if order == 0 else w.t().contiguous().t()
            loss, lse, _ = nn.linear_cross_entropy(x, wc, target, reduction="none", keep=True)
            assert loss.isnan().all() and (lse == -INF).all()
            target[0] = IGNORE
            loss = nn.linear_cross_entropy(x, wc, target, reduction="none")
            assert loss[0] == 0 and loss[1:].isnan().all()
            target[0] = 7
    for highest in (-low, INF):
        w = torch.zeros(8, classes, dtype=torch.bfloat16, device="cuda")
        w[1, 5] = highest
        loss, lse, _ = nn.linear_cross_entropy(x, w, target, reduction="none", keep=True)
        # row 0 meets the highest with a zero: 0 * infinity is NaN too
        assert loss[0].isfinite() == (highest < INF) and loss[1:].isnan().all() and lse[1:].isnan().all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("m,n", [(64, 1_100_041), (33, 2_200_000)])
def test_two_terms_over_several_pieces(m, n, order, dtype):
    """Rows few enough for dz's second term and classes enough for two pieces, the last one narrower: dx's halves added up over the
    pieces, dw from a column's offset.  Against float64; every result is rounded once (half a step at most), what dz's second
    rounding and the float32 sums leave is a tenth of that in the norm."""
    nn = _nn()
    k = 64
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn((k, n) if order == 0 else (n, k), generator=g, device="cuda") * k ** -0.5).to(dtype)
    wc = w if order == 0 else w.t()
    width = -(-(-(-n // 2)) // 256) * 256  # of the first piece
    target = torch.randint(0, n, (m,), generator=g, device="cuda")
    target[:6] = torch.tensor([0, width - 1, width, width + 1, n - 1, IGNORE], device="cuda")
    z = torch.matmul(x.double(), wc.double().contiguous())
    lse = torch.logsumexp(z, 1)
    loss, got_lse, _ = nn.linear_cross_entropy(x, wc, target, reduction="none", keep=True)
    counts = target != IGNORE
    at = target.clamp_min(0)
    want = torch.where(counts, lse - z[torch.arange(m), at], torch.zeros_like(lse))
    # k of 64: logits off by 2k + 8 roundings of their products at most; exponentials and their sum by 128 + n/4096 of them
    off = ((2 * k + 8) * (x.double().abs() @ wc.double().abs().contiguous()).amax(1) + 150 + n / 4096 + 8 * lse.abs()) * ref.u
    assert ((got_lse - lse).abs() <= off).all() and ((loss.double() - want).abs() <= 2 * off).all()
    d = torch.exp(z - lse[:, None])
    del z
    d[torch.arange(m), at] -= 1
    d *= counts[:, None]
    for rows in (True, False):
        # dloss large enough that float16 holds the other classes' gradients (1e-6 of it) as normal numbers
        dloss = (torch.rand(m, generator=g, device="cuda") + 0.5) * 1024 if rows else torch.full((), 1024.0, device="cuda")
        dz = d * dloss.double().reshape(-1, 1)
        dx, dw = nn.linear_cross_entropy_grad(dloss, x, wc, target, got_lse)
        full = torch.matmul(dz, wc.t().double().contiguous())
        assert float((dx.double() - full).norm()) < 1.1 * ref.U[dtype] * float(full.norm())
        assert (dx[5] == 0).all()
        full = torch.matmul(x.t().double().contiguous(), dz)
        off = dw.double() - full
        assert float(off.norm()) < 1.1 * ref.U[dtype] * float(full.norm())
        # and column by column: no column of another piece, none left out (float16: half a spacing of small numbers besides)
        size = full.norm(dim=0)
        assert bool((off.norm(dim=0) <= 2 * ref.U[dtype] * size + 2.0 ** -25 * k ** 0.5).all())
        del full, off, dw, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("m,n,k", [(0, 5, 8), (5, 1, 8), (5, 7, 0), (1, 1, 1), (65, 3, 2)])
def test_autograd_of_every_size(m, n, k, reduction):
    """No rows, one class, no depth: as the gradient call; every row ignored gives zeros."""
    nn = _nn()
    g = torch.Generator().manual_seed(m + n + k)
    x, w = torch.randn(m, k, generator=g).bfloat16().cuda(), torch.randn(n, k, generator=g).bfloat16().cuda()
    for target in (torch.randint(0, n, (m,), generator=g).cuda(), torch.full((m,), IGNORE, device="cuda")):
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        loss = nn.linear_cross_entropy(leaves[0], leaves[1].t(), target, reduction=reduction)
        up = torch.rand(loss.shape, generator=g).cuda()
        got = torch.autograd.grad(loss, leaves, up)
        with torch.no_grad():
            again, lse, count = nn.linear_cross_entropy(x, w.t(), target, reduction=reduction, keep=True)
            dx, dw = nn.linear_cross_entropy_grad(up, x, w.t(), target, lse, count)
        assert torch.equal(loss, again) and torch.equal(got[0], dx) and torch.equal(got[1], dw.t())
        want = torch.nn.functional.cross_entropy((x.double().cpu() @ w.double().cpu().t()), target.cpu(), reduction="none")
        if reduction == "none":
            assert ((loss.cpu().double() - want).abs() <= 1e-5 * (1 + want)).all()
        assert all(t.isfinite().all() for t in got)
        if m and target[0] == IGNORE:
            assert (got[0] == 0).all() and (got[1] == 0).all() and (loss == 0).all()
        if n == 1:
            # The one class's pair is t, logit * log2(e) rounded, and exp2(logit * log2(e) - t): an exponent of at most u * |t| / 2
            # (|t| < 16 here), an ulp of the exponential, one of the logarithm: 8u * ln 2 + 4u of 1, in p - 1 too; a row of dw
            # adds m of them.
            off = 12 * ref.u * (up.abs().sum().item() + 1)
            assert (loss.abs() <= 12 * ref.u * max(1, m)).all() and (got[0].abs() <= off * w.float().abs().max()).all()
            assert (got[1].abs() <= off * x.float().abs().max()).all()


def test_calls_at_once_from_threads_and_streams():
    """Steps through autograd from four threads on streams of their own give the bits of steps alone."""
    import threading
    nn = _nn()
    shapes = [(33, 700, 64), (200, 520, 136), (65, 1001, 77), (16, 4000, 256)]
    data = []
    for i, (m, n, k) in enumerate(shapes):
        g = torch.Generator().manual_seed(i)
        data.append((torch.randn(m, k, generator=g).half().cuda(), (torch.randn(n, k, generator=g) * k ** -0.5).half().cuda(),
                     torch.randint(0, n, (m,), generator=g).cuda(), torch.randn(k, generator=g).cuda()))

    def step(x, w, t, nw):
        a, b, c = (v.clone().requires_grad_() for v in (x, w, nw))
        y, _ = nn.rms_norm(a, c, keep8=True)
        loss = nn.linear_cross_entropy(nn.linear(y, b.t(), None, "gelu", keep8=True), torch.eye(w.shape[0], dtype=w.dtype, device="cuda"), t)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b, c)))

    alone = [step(*d) for d in data]
    torch.cuda.synchronize()
    bad, streams = [], [torch.cuda.Stream() for _ in data]

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(8):
                got = step(*data[i])
                streams[i].synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, alone[i])):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
