"""A pre-norm residual MLP block, trained in bfloat16 and served in 8 bits (e4m3 or integers).

    h   = x + r                              the residual stream
    y   = rms_norm(h)
    out = h + gelu(y @ w1 + b1) @ w2 + b2

Training runs the block through tforge_nn under autograd: the norm and both
products with their epilogues forward, their gradient calls backward, plain SGD on
float32 copies of the weights.  The data is synthetic: the targets come from a
block with other weights.  Then the trained weights are laid out once in 8 bits
(one scale a column) and the block serves one token, and a batch: the norm writes
8 bits with a scale a row, the first layer reads them, its output is quantised
row by row and the second layer adds the residual.

With --classes the block learns to classify instead: its outputs go through a head of
that many classes into the cross entropy, whose logits are never in memory, and what the
backward pass needs of the activations is kept in 8 bits.

    python examples/residual_mlp.py [--rows 4096] [--width 2048] [--hidden 8192] [--steps 20] [--classes 32000] [--integers]
"""

import argparse
import pathlib
import sys
import time

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))
from tensorforge_amd import tforge_nn as nn  # noqa: E402


def weights(width, hidden, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = lambda *s, scale: torch.randn(s, generator=g, device="cuda") * scale  # noqa: E731
    return {"norm": torch.ones(width, device="cuda"), "w1": t(width, hidden, scale=width ** -0.5),
            "b1": t(hidden, scale=0.02), "w2": t(hidden, width, scale=hidden ** -0.5), "b2": t(width, scale=0.02)}


def block(p, x, r, keep8=False):
    y, h = nn.rms_norm(x, p["norm"], residual=r, keep8=keep8)
    return nn.linear(nn.linear(y, p["w1"], p["b1"], "gelu", keep8=keep8), p["w2"], p["b2"], "none", h, keep8=keep8)


def half(p):
    """The weights as the kernels take them in training: matrices in bfloat16, vectors in float32."""
    return {k: v.bfloat16() if v.dim() == 2 else v for k, v in p.items()}


class Served:
    """The block in 8 bits: weights laid out once, column by column with one scale each."""

    @torch.no_grad()
    def __init__(self, p, dtype=torch.float8_e4m3fn):
        self.norm, self.b1, self.b2, self.dtype = p["norm"], p["b1"], p["b2"], dtype
        self.w1, self.s1 = nn.quantize_rows(p["w1"].t().contiguous(), dtype)
        self.w2, self.s2 = nn.quantize_rows(p["w2"].t().contiguous(), dtype)

    @torch.no_grad()
    def __call__(self, x, r):
        q, s, h = nn.rms_norm(x, self.norm, residual=r, quantize=self.dtype)
        a = nn.linear(q, self.w1.t(), self.b1, "gelu", x_scale=s, w_scale=self.s1, out_dtype=x.dtype)
        q, s = nn.quantize_rows(a, self.dtype)
        return nn.linear(q, self.w2.t(), self.b2, "none", h, x_scale=s, w_scale=self.s2, out_dtype=x.dtype)


def train(rows, width, hidden, steps, rate=2.0, seed=0):
    """(weights, loss of each step): a block that learns another's outputs."""
    target = half(weights(width, hidden, seed + 1))
    p = {k: v.requires_grad_() for k, v in weights(width, hidden, seed).items()}
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    x, r = (torch.randn((rows, width), generator=g, device="cuda").bfloat16() for _ in range(2))
    with torch.no_grad():
        want = block(target, x, r)
    losses = []
    for _ in range(steps):
        out = block(half(p), x, r)
        loss = (out.float() - want.float()).square().mean()
        loss.backward()
        with torch.no_grad():
            for v in p.values():
                v -= rate * v.grad
                v.grad = None
        losses.append(float(loss.detach()))
    return {k: v.detach() for k, v in p.items()}, losses


def classify(p, x, r, target):
    """The loss of a block with a head over its outputs."""
    return nn.linear_cross_entropy(block(p, x, r, keep8=True), p["head"].t(), target)


def train_classes(rows, width, hidden, classes, steps, rate=2.0, seed=0):
    """(weights, loss of each step): a block and a head that learn the classes that others give."""
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    head = lambda: torch.randn((classes, width), generator=g, device="cuda") * width ** -0.5  # noqa: E731
    x, r = (torch.randn((rows, width), generator=g, device="cuda").bfloat16() for _ in range(2))
    with torch.no_grad():
        target = nn.linear(block(half(weights(width, hidden, seed + 1)), x, r), head().bfloat16().t()).argmax(1)
    target[::17] = -100  # rows that do not count
    p = {k: v.requires_grad_() for k, v in {**weights(width, hidden, seed), "head": head()}.items()}
    losses = []
    for _ in range(steps):
        loss = classify(half(p), x, r, target)
        loss.backward()
        with torch.no_grad():
            for v in p.values():
                v -= rate * v.grad
                v.grad = None
        losses.append(float(loss.detach()))
    return {k: v.detach() for k, v in p.items()}, losses


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--width", type=int, default=2048)
    ap.add_argument("--hidden", type=int, default=8192)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--classes", type=int, default=0)
    ap.add_argument("--integers", action="store_true", help="serve in 8-bit integers")
    a = ap.parse_args(argv)
    if a.classes:
        p, losses = train_classes(a.rows, a.width, a.hidden, a.classes, a.steps)
    else:
        p, losses = train(a.rows, a.width, a.hidden, a.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps", flush=True)
    served, trained = Served(p, torch.int8 if a.integers else torch.float8_e4m3fn), half(p)
    g = torch.Generator(device="cuda").manual_seed(7)
    for rows in (1, a.rows):
        x, r = (torch.randn((rows, a.width), generator=g, device="cuda").bfloat16() for _ in range(2))
        with torch.no_grad():
            want = block(trained, x, r)
        got = served(x, r)
        off = float((got.float() - want.float()).norm() / want.float().norm())
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(50):
            served(x, r)
        torch.cuda.synchronize()
        print(f"{rows} rows in 8 bits: {(time.perf_counter() - t) / 50 * 1e6:.1f} us, {off:.4f} off the bfloat16 block", flush=True)
    return losses


if __name__ == "__main__":
    main()
