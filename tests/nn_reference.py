"""The residual block's operators in 64 bits on the CPU, from their definitions,
and the error bounds the kernels' results are held to.

Bounds: U[t] is the unit roundoff of the output's type; inner arithmetic is
float32 (unit roundoff u = 2^-24) with sums of at most `terms` additions, each
partial sum off by at most u, so a sum of products is off by at most
2 * terms * u * sum|products| (one u a product, one an addition).  relu, gelu and
silu have slopes of at most 1.13; the polynomial inside gelu's tail is off by at
most 7e-7 of the tail, exponentials and reciprocals by a few u.
"""

import math

import torch

F8 = torch.float8_e4m3fn
u = 2.0 ** -24
U = {torch.float32: u, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the spacing of the smallest numbers
FLOOR = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
F8_MAX, TINY = 448.0, 2.0 ** -100


def act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return z * torch.special.erfc(-z * math.sqrt(0.5)) / 2
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return torch.special.erfc(-z * math.sqrt(0.5)) / 2 + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def norm(x, w, r=None, eps=1e-6):
    h = x.double() + (r.double() if r is not None else 0)
    return h / (h.pow(2).mean(1, keepdim=True) + eps).sqrt() * w.double(), h


def norm_grad(dy, h, w, eps=1e-6, dh=None):
    dy, h, w = dy.double(), h.double(), w.double()
    r = (h.pow(2).mean(1, keepdim=True) + eps).rsqrt()
    g, xhat = dy * w, h * r
    dx = r * (g - xhat * (g * xhat).mean(1, keepdim=True)) + (dh.double() if dh is not None else 0)
    return dx, (dy * xhat).sum(0)


def close(got, want, bound, dtype):
    """Every element within bound + one rounding to dtype; NaN exactly where NaN is wanted."""
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), "NaN in other places"
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    limit = (bound + U[dtype] * (want.abs() + bound) + FLOOR[dtype]).expand_as(want)
    off = (got - want).abs()
    bad = fine & ~(off <= limit)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / limit)[fine].max()):.3g} of its bound"


def f8_close(q, scale, y, slack):
    """Codes within half a spacing (and `slack` of the value) of y/scale, scales within `slack`."""
    want = y.abs().amax(1).clamp_min(TINY) / F8_MAX
    s = scale.double().cpu()
    assert ((s - want).abs() <= slack * want).all()
    v = (y / want[:, None])
    q = q.cpu().float().double()
    spacing = torch.exp2(torch.floor(torch.log2(torch.maximum(v.abs(), q.abs()).clamp_min(2.0 ** -6))) - 3)
    assert ((q - v).abs() <= spacing / 2 + 4 * slack * v.abs()).all()
