"""The operators together, as examples/residual_mlp.py uses them: a block whose activations are kept in
8 bits under the cross entropy of a head over its outputs, and the block served in 8-bit integers."""

import numpy as np
import pytest
import torch

import nn_reference as ref
from test_gpu_nn_block import _example
from test_gpu_nn_keep8 import _bytes, _values

pytestmark = pytest.mark.gpu


def _kept8(t):
    return _values(*_bytes(t), t.shape[1]).double()


def _round(t):
    return t.bfloat16().double()


def test_gradients_of_a_step():
    """Against the same step in float64 with the same roundings between the calls, and the activations as they are kept.  What is left
    are float32 sums and dz's rounding in the products: up to half a step of 2^-8 of each value, some sqrt(1/3) of that in the mean
    square, in dx of the head (once), of the block's second layer (its dz is rounded already) and of its first (again), beside
    bfloat16 results' own: in the norm under 2 * 2^-8."""
    ex = _example()
    rows, width, hidden, classes = 90, 136, 264, 1000
    p = {k: v.requires_grad_() for k, v in ex.weights(width, hidden, 3).items()}
    g = torch.Generator(device="cuda").manual_seed(4)
    p["head"] = (torch.randn((classes, width), generator=g, device="cuda") * width ** -0.5).requires_grad_()
    x, r = (torch.randn((rows, width), generator=g, device="cuda").bfloat16() for _ in range(2))
    x.requires_grad_()
    target = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    target[::7] = -100
    loss = ex.classify(ex.half(p), x, r, target)
    loss.backward()

    q = {k: _round(v.detach().cpu()) if v.dim() == 2 else v.detach().cpu().double() for k, v in p.items()}
    t = target.cpu()
    full = x.detach().cpu().double() + r.cpu().double()
    h = _round(full)
    y = _round(ref.norm(full, q["norm"])[0])
    z = y @ q["w1"] + q["b1"]
    a = _round(ref.act(z, "gelu"))
    out = _round(a @ q["w2"] + q["b2"] + h)
    logits = out @ q["head"].t()
    counts = t != -100
    lse = torch.logsumexp(logits, 1)
    rows_loss = (lse - logits[torch.arange(rows), t.clamp_min(0)])[counts]
    assert abs(float(loss.detach()) - float(rows_loss.mean())) < 1e-3 * float(rows_loss.mean())
    d = torch.exp(logits - lse[:, None])
    d[torch.arange(rows), t.clamp_min(0)] -= 1
    d *= (counts / counts.sum())[:, None]
    dout = _round(d @ q["head"])
    kz, ka, ky, kh = (_kept8(v.bfloat16()) for v in (_round(z), a, y, h))
    da = _round(dout @ q["w2"].t())
    dz = da * ref.slope(kz, "gelu")
    dx, dn = ref.norm_grad(_round(dz @ q["w1"].t()), kh, q["norm"], dh=dout)
    want = {"norm": dn, "w1": ky.t() @ dz, "b1": dz.sum(0), "w2": ka.t() @ dout, "b2": dout.sum(0), "head": d.t() @ out}
    for got, w in [(x.grad, dx)] + [(p[k].grad, want[k]) for k in want]:
        off = float((got.double().cpu() - w).norm() / w.norm())
        assert off < 2 * 2.0 ** -8, off
    # and what is kept in 8 bits costs: 127 steps to a group's largest value, a few of its values; the gradients point the same way
    plain = {"w1": y.t() @ (da * ref.slope(z, "gelu")), "w2": a.t() @ dout}
    for k, w in plain.items():
        got = p[k].grad.double().cpu()
        assert float((got * w).sum() / (got.norm() * w.norm())) > 0.999


def test_classes_are_trained_and_served():
    """It runs; every parameter gets a finite gradient; the block in 8-bit integers is near the bfloat16 one."""
    ex = _example()
    p, losses = ex.train_classes(256, 128, 512, 777, 3)
    assert len(losses) == 3 and np.isfinite(losses).all() and all(v.isfinite().all() for v in p.values())
    before = {**ex.weights(128, 512, 0)}
    assert all(not torch.equal(p[k], before[k]) for k in before)
    served, trained = ex.Served(p, torch.int8), ex.half(p)
    for rows in (1, 3, 64, 300):
        g = torch.Generator(device="cuda").manual_seed(rows)
        x, r = (torch.randn((rows, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
        with torch.no_grad():
            want = ex.block(trained, x, r).float()
        # integers keep 1/254 of a row's largest value, which is three to four of its root mean square: a rounding of 0.5 to 1% in four
        # places on the way to a sum that the residual enters unrounded
        assert float((served(x, r).float() - want).norm() / want.norm()) < 0.02
