"""How rms_norm and linear stand in autograd, without a GPU: the native layer is replaced by plain torch steps of
the same contract (None where an input wants a gradient, results that record nothing)."""

import pytest
import torch

import nn_reference as ref
from tensorforge_amd import tforge_nn as nn

NAMES = {v: k for k, v in nn.ACTIVATIONS.items()}


class Plain:
    """The native layer's calls in float64, in torch's operators."""

    def rms_norm(self, x, weight, residual, eps, quantize):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
            return None
        h = x if residual is None else x + residual.view_as(x)
        y = h * (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * weight
        return y.detach(), (None if residual is None else h.detach())

    def rms_norm_grad(self, dy, h, weight, eps, dh):
        n = h.shape[-1]
        dx, dw = ref.norm_grad(dy.reshape(-1, n), h.reshape(-1, n), weight, eps, None if dh is None else dh.reshape(-1, n))
        return dx.view_as(h).detach(), dw.detach()

    def linear(self, x, w, bias, act, residual, keep, x_scale, w_scale, out_dtype, tile, splits):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias, residual)):
            return None
        z = x @ w + (0 if bias is None else bias)
        out = ref.act(z, NAMES[act])
        out = (out if residual is None else out + residual.view_as(out)).detach()
        return (out, z.detach()) if keep else out

    def linear_grad(self, dy, x, w, z, act, bias_dtype, want_dx, want_dw, tile, splits, terms):
        k, n = w.shape
        dz = (dy * ref.slope(z.view_as(dy), NAMES[act]) if act else dy).reshape(-1, n).detach()
        return ((dz @ w.t()).view_as(x).detach() if want_dx else None, (x.reshape(-1, k).t() @ dz).detach() if want_dw else None,
                dz.sum(0) if bias_dtype is not None else None)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(nn, "_C", Plain())


def _leaves(*shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g, dtype=torch.float64).requires_grad_() for s in shapes]


def _norm(x, w, r=None):
    return ref.norm(x, w, r)[0]


def test_first_order(plain):
    x, w, r, w1, b = _leaves((6, 8), (8,), (6, 8), (8, 5), (5,))
    f = lambda norm, linear: (linear(norm(x, w, r), w1, b).sin()).sum()  # noqa: E731
    got = torch.autograd.grad(f(lambda *a: nn.rms_norm(*a)[0], lambda *a: nn.linear(*a, "gelu")), (x, w, r, w1, b))
    want = torch.autograd.grad(f(_norm, lambda a, c, d: ref.act(a @ c + d, "gelu")), (x, w, r, w1, b))
    for a, c in zip(got, want):
        assert torch.allclose(a, c, rtol=1e-10)


def test_second_order_is_refused(plain):
    """A penalty on a gradient needs the gradient calls' own: an error, not a penalty without effect."""
    x, w, w1, b = _leaves((6, 8), (8,), (8, 5), (5,))
    for loss, of in ((nn.rms_norm(x, w)[0].sin().sum(), w), (nn.linear(x, w1, b, "silu").sin().sum(), w1),
                     (nn.linear(x, w1, b).sin().sum(), w1)):
        g, = torch.autograd.grad(loss, of, create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.pow(2).sum().backward()


def test_tangents_are_seen():
    """The native layer hands a dual tensor to autograd, under no_grad too."""
    import torch.autograd.forward_ad as fwd
    x, w, v = (torch.ones(s, dtype=torch.bfloat16) for s in ((4, 8), (8, 8), (8,)))
    with fwd.dual_level():
        for at in (0, 1):
            a, b = [x, w], [x, v]
            a[at], b[at] = (fwd.make_dual(t[at], torch.ones_like(t[at])) for t in (a, b))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode():
                    assert nn._C.linear(*a, None, 0, None, False, None, None, None, 0, 0) is None
                    assert nn._C.rms_norm(*b, None, 1e-6, False) is None
        with pytest.raises(ValueError, match="no gradient"):
            nn.rms_norm(*b, quantize=True)


def test_calls_without_a_gradient_refuse():
    """What cannot pass a gradient on says so where an input wants one, and takes it under no_grad (up to the missing GPU)."""
    h, w, v, s = (torch.ones(n, dtype=torch.bfloat16) for n in ((4, 8), (8, 16), (8,), (4, 16)))
    f8, w8 = h.to(ref.F8), w.t().contiguous().to(ref.F8).t()
    one = torch.ones(4), torch.ones(16)
    calls = [(lambda a: nn.quantize_rows(a), [h]), (lambda a, b, c: nn.rms_norm_grad(a, b, c), [h, h, v]),
             (lambda a, b, c, d: nn.rms_norm_grad(a, b, c, dh=d), [h, h, v, h]),
             (lambda a, b, c, d: nn.linear_grad(a, b, c, d, "gelu"), [s, h, w, s]),
             (lambda a, b, c, d: nn.linear(f8, w8, a, "none", b, x_scale=c, w_scale=d), [one[1], s, *one]),
             (lambda a, b, c: nn.rms_norm(a, b, c, quantize=True), [h, v, h])]
    for call, tensors in calls:
        for i in range(len(tensors)):
            args = [t.clone().requires_grad_() if q == i else t for q, t in enumerate(tensors)]
            with pytest.raises(ValueError, match="no gradient"):
                call(*args)
            with torch.no_grad(), pytest.raises(ValueError, match="not on a GPU"):
                call(*args)


def test_refusals_with_a_gradient_wanted():
    """The checks of the tensors hold for calls that go through autograd too."""
    h, w, v = (torch.zeros(n, dtype=torch.bfloat16) for n in ((4, 8), (8, 16), (8,)))
    one = torch.zeros(16)
    for call, error, words in [
            (lambda a: nn.linear(a, w, x_scale=one[:4]), ValueError, "scales belong"),
            (lambda a: nn.linear(a, w, w_scale=one), ValueError, "scales belong"),
            (lambda a: nn.linear(a, w, x_scale=one[:4], w_scale=one), ValueError, "scales belong"),
            (lambda a: nn.linear(a, w, out_dtype=torch.float16), TypeError, "keep x's type"),
            (lambda a: nn.linear(a, w.half()), TypeError, "w is Half"),
            (lambda a: nn.linear(a, h), ValueError, "not 8 x n"),
            (lambda a: nn.linear(a, w, v), ValueError, "bias is not"),
            (lambda a: nn.linear(a, w, residual=h), ValueError, "residual is 4 x 8, not 4 x 16"),
            (lambda a: nn.linear(a, w, activation="tanh"), ValueError, "not one of none, relu, gelu, silu"),
            (lambda a: nn.linear(a, w, tile=9), ValueError, "not on a GPU"),
            (lambda a: nn.rms_norm(a, v.half()), TypeError, "weight is Half"),
            (lambda a: nn.rms_norm(a, one), ValueError, "not a contiguous vector of 8"),
            (lambda a: nn.rms_norm(a, v, residual=w), ValueError, "residual is 8 x 16, not 4 x 8")]:
        for a in (h, h.clone().requires_grad_()):
            with pytest.raises(error, match=words):
                call(a)


@pytest.mark.parametrize("activation", ["none", "gelu"])
@pytest.mark.parametrize("of", ["both", "out", "z"])
def test_the_kept_pre_activation_is_differentiable(activation, of, plain):
    """A loss on the kept z, alone or beside the output's, reaches x, w and the bias."""
    leaves = _leaves((6, 8), (8, 5), (5,), (6, 5))

    def loss(out, z):
        return (out.sin().sum() if of != "z" else 0) + (z.pow(3).sum() if of != "out" else 0)

    x, w, b, r = leaves
    got = torch.autograd.grad(loss(*nn.linear(x, w, b, activation, r, keep=True)), leaves, allow_unused=True)
    z = x @ w + b
    want = torch.autograd.grad(loss(ref.act(z, activation) + r, z), leaves, allow_unused=True)
    for a, c in zip(got, want):
        assert (a is None) == (c is None) and (a is None or torch.allclose(a, c, rtol=1e-10))


@pytest.mark.parametrize("shape,other", [((2, 3, 8), (6, 8)), ((6, 8), (2, 3, 8)), ((8,), (1, 8)), ((1, 1, 8), (8,))])
def test_a_residual_of_other_leading_dimensions(shape, other, plain):
    """Leading dimensions are rows: the residual's gradient has the residual's own, and memory of its own."""
    x, r, w, w1 = _leaves(shape, other, (8,), (8, 8))
    for f, want in ((lambda: sum(t.sin().sum() for t in nn.rms_norm(x, w, r)),
                     lambda: sum(t.sin().sum() for t in ref.norm(x.view(-1, 8), w, r.view(-1, 8)))),
                    (lambda: nn.linear(x, w1, None, "gelu", r).sin().sum(),
                     lambda: (ref.act(x.view(-1, 8) @ w1, "gelu") + r.view(-1, 8)).sin().sum())):
        grads = []
        for g in (f, want):
            x.grad = r.grad = None
            g().backward()
            grads.append((x.grad, r.grad))
            assert x.grad.shape == x.shape and r.grad.shape == r.shape
            assert g is want or x.grad.data_ptr() != r.grad.data_ptr()
        for a, c in zip(*grads):
            assert torch.allclose(a, c, rtol=1e-10)


def test_a_loss_on_h_alone(plain):
    """The norm is not part of it: the gradients are h's, also where h holds an infinity."""
    x, w, r = _leaves((4, 8), (8,), (4, 8))
    with torch.no_grad():
        x[1, 2] = float("inf")
    _, h = nn.rms_norm(x, w, r)
    gh = torch.arange(32.0, dtype=torch.float64).view(4, 8)
    gx, gw, gr = torch.autograd.grad(h, (x, w, r), gh, allow_unused=True)
    assert torch.equal(gx, gh) and torch.equal(gr, gh) and gw is None
