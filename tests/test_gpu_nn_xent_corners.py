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
