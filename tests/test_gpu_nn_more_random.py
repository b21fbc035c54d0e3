"""Seeded draws over the integers' products, the gradients from kept activations and the loss over a
vocabulary: sizes, types, orders, row distances and alignments together, against 64-bit references; and
calls of all three at once on several streams."""

import random

import pytest
import torch

import nn_reference as ref
import test_gpu_nn_int8 as integers
import test_gpu_nn_keep8 as kept
import test_gpu_nn_xent as xent

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def _nn():
    from tensorforge_amd import tforge_nn
    return tforge_nn


def _size(rng, most):
    return rng.choice([1, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, rng.randint(1, most), rng.randint(1, most)])


def _laid(rng, t):
    """t on the GPU: as it is, in a wider matrix, or off a 16-byte boundary."""
    pad, off = rng.choice([(0, 0), (0, 0), (8, 0), (16, 8), (5, 3), (1, 1)])
    if not pad:
        return t.cuda()
    wide = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype)
    wide[:, off:off + t.shape[1]] = t
    return wide.cuda()[:, off:off + t.shape[1]]


@pytest.mark.parametrize("seed", range(40))
def test_integers(seed):
    nn, rng = _nn(), random.Random(seed)
    m, n, k = _size(rng, 400), _size(rng, 700), _size(rng, 2000)
    g = torch.Generator().manual_seed(seed)
    q, wq = integers._codes(g, m, k), integers._codes(g, n, k)
    s, ws = torch.rand(m, generator=g) * 0.01, torch.rand(n, generator=g) * 0.01
    out_dtype, activation = rng.choice(HALF), rng.choice(["none", "relu", "gelu", "silu"])
    b = torch.randn(n, generator=g).to(rng.choice([out_dtype, torch.float32])) if rng.random() < 0.6 else None
    r = torch.randn(m, n, generator=g).to(out_dtype) if rng.random() < 0.5 else None
    call = lambda **how: nn.linear(_laid(rng, q), _laid(rng, wq).t(), None if b is None else b.cuda(), activation,  # noqa: E731
                                   None if r is None else _laid(rng, r), keep=True, x_scale=s.cuda(), w_scale=ws.cuda(),
                                   out_dtype=out_dtype, **how)
    out, z = call()
    zw, ow, off, off_out = integers._want(q, wq, s, ws, b, activation, r)
    ref.close(z, zw, off, out_dtype)
    ref.close(out, ow, off_out, out_dtype)
    again = call(tile=rng.choice([1, 2, 3, 4, 5]), splits=rng.choice([1, 2, 5]))
    assert torch.equal(again[0], out) and torch.equal(again[1], z)


@pytest.mark.parametrize("seed", range(40))
def test_gradients_from_what_was_kept(seed):
    nn, rng = _nn(), random.Random(seed)
    m, n, k = _size(rng, 500), _size(rng, 500), _size(rng, 500)
    dtype, activation, order = rng.choice(HALF), rng.choice(["none", "relu", "gelu", "silu"]), rng.choice([0, 1])
    g = torch.Generator().manual_seed(seed)
    dy, x, z = kept._matrix(g, m, n, dtype), kept._matrix(g, m, k, dtype), kept._matrix(g, m, n, dtype, 1.5)
    w = kept._matrix(g, k, n, dtype, k ** -0.5)
    wc = _laid(rng, w) if order == 0 else _laid(rng, w.t().contiguous()).t()
    x8 = nn.keep8(_laid(rng, x))
    z8 = nn.keep8(_laid(rng, z), activation == "relu") if activation != "none" else None
    bias = rng.choice([None, dtype, torch.float32])
    got = nn.linear_grad(_laid(rng, dy), x8, wc, z8, activation, bias, rng.random() < 0.8, rng.random() < 0.8)
    kept._check_grad(got, dy, x8.restore().cpu(), w, None if z8 is None else z8.restore().cpu(), activation, dtype, bias)
    h8 = nn.keep8(_laid(rng, z))
    weight = (1 + 0.1 * torch.randn(n, generator=g)).cuda()
    for a, b in zip(nn.rms_norm_grad(_laid(rng, dy), h8, weight), nn.rms_norm_grad(dy.cuda(), h8.restore(), weight)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("seed", range(60))
def test_the_loss(seed):
    nn, rng = _nn(), random.Random(seed)
    m, n, k = _size(rng, 500), _size(rng, 2500), _size(rng, 400)
    dtype, order = rng.choice(HALF), rng.choice([0, 1])
    x, w, target, g = xent._data(m, n, k, dtype, ignored=rng.choice([0.0, 0.3, 0.9]), scale=rng.choice([0.1, 2.0, 6.0]), seed=seed)
    xc, tc = _laid(rng, x), target.cuda()
    wc = _laid(rng, w) if order == 0 else _laid(rng, w.t().contiguous()).t()
    loss, lse, _ = nn.linear_cross_entropy(xc, wc, tc, reduction="none", keep=True)
    z, want_lse = xent._check_loss(loss, lse, x, w, target)
    dloss = torch.randn(m, generator=g) if rng.random() < 0.5 else torch.tensor(rng.uniform(-2, 2))
    dx, dw = nn.linear_cross_entropy_grad(dloss.cuda(), xc, wc, tc, lse, want_dx=rng.random() < 0.8, want_dw=rng.random() < 0.8)
    xent._check_grad(dx, dw, dloss, x, w, target, z, want_lse, dtype)


def test_calls_at_once():
    """Six streams, each with its own calls of all three, without waiting for each other: the bits each gives alone."""
    nn = _nn()

    def work(seed):
        g = torch.Generator().manual_seed(seed)
        m, n, k = 100 + 40 * seed, 520 + 8 * seed, 264
        x, w, target, _ = (v.cuda() if isinstance(v, torch.Tensor) else v for v in xent._data(m, n, k, torch.bfloat16, seed=seed))
        wq, ws = nn.quantize_rows(w.t().contiguous(), torch.int8)
        dy = kept._matrix(g, m, n, torch.bfloat16).cuda()

        def run():
            loss, lse, count = nn.linear_cross_entropy(x, w, target, keep=True)
            grads = nn.linear_cross_entropy_grad(torch.ones((), device="cuda"), x, w, target, lse, count)
            q, s = nn.quantize_rows(x, torch.int8)
            out, z = nn.linear(q, wq.t(), None, "gelu", keep=True, x_scale=s, w_scale=ws)
            more = nn.linear_grad(dy, nn.keep8(x), w, nn.keep8(z), "gelu")
            return (loss, *grads, out, *more[:2])

        return run

    runs = [work(i) for i in range(6)]
    want = [r() for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for r, s in zip(runs, streams):
            with torch.cuda.stream(s):
                got.append(r())
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
