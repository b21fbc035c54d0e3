"""The operators together: examples/residual_mlp.py trains the pre-norm residual
block and serves it in 8 bits; its gradients against the same steps in float64."""

import importlib.util
import pathlib

import pytest
import torch

import nn_reference as ref

pytestmark = pytest.mark.gpu

PATH = pathlib.Path(__file__).resolve().parent.parent / "examples" / "residual_mlp.py"


def _example():
    spec = importlib.util.spec_from_file_location("residual_mlp", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_block_learns_and_serves():
    ex = _example()
    p, losses = ex.train(512, 128, 512, 30)
    assert losses[-1] < 0.5 * losses[0] and all(b < a * 1.05 for a, b in zip(losses, losses[1:])), losses
    served, trained = ex.Served(p), ex.half(p)
    for rows in (1, 3, 64, 300):
        g = torch.Generator(device="cuda").manual_seed(rows)
        x, r = (torch.randn((rows, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
        with torch.no_grad():
            want = ex.block(trained, x, r).float()
        # e4m3 keeps 4 bits (a rounding of 2^-4 at most, 2^-5.4 in the mean square); four roundings on the way to a sum
        # that the residual (most of the output) enters unrounded
        assert float((ex.Served.__call__(served, x, r).float() - want).norm() / want.norm()) < 0.05


def test_block_gradients():
    """Against the same steps in float64 with the same roundings between them: what is kept (h, y, z, a) and what goes from
    call to call (da, dy) in bfloat16.  What is left are float32 sums, whose errors move few values across a rounding: of
    1% of the values one unit, 2^-8 of them, is 0.1 * 2^-8 in the norm."""
    ex = _example()
    p = {k: v.requires_grad_() for k, v in ex.weights(136, 264, 3).items()}
    g = torch.Generator(device="cuda").manual_seed(4)
    x, r, dy = (torch.randn((77, 136), generator=g, device="cuda").bfloat16() for _ in range(3))
    x.requires_grad_()
    out = ex.block(ex.half(p), x, r)
    out.backward(dy)

    def kept(t):
        return t.bfloat16().double()

    q = {k: kept(v.detach().cpu()) if v.dim() == 2 else v.detach().cpu().double() for k, v in p.items()}
    g = dy.cpu().double()
    full = x.detach().cpu().double() + r.cpu().double()
    h = kept(full)
    y = kept(ref.norm(full, q["norm"])[0])
    z = y @ q["w1"] + q["b1"]
    a = kept(ref.act(z, "gelu"))
    da = kept(g @ q["w2"].t())
    dz = da * ref.slope(kept(z), "gelu")
    dx, dn = ref.norm_grad(kept(dz @ q["w1"].t()), h, q["norm"], dh=g)
    want = {"norm": dn, "w1": kept(y.t() @ dz), "b1": dz.sum(0), "w2": kept(a.t() @ g), "b2": g.sum(0)}
    pairs = [(out.detach(), kept(a @ q["w2"] + q["b2"] + h)), (x.grad, kept(dx))] + [(p[k].grad, want[k]) for k in p]
    for got, w in pairs:
        assert float((got.double().cpu() - w).norm() / w.norm()) < 0.1 * 2.0 ** -8
