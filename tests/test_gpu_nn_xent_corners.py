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
