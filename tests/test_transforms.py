"""torch.func and forward-mode derivatives of LayerNorm and the sigmoid gate (no GPU): the package's own autograd
functions with torch operations in the kernels' place, and refusals that come before any device work."""
import sys

import pytest
import torch
from torch.autograd import forward_ad


class PlainOps:
    """The extension's calls that the autograd functions make, in torch operations. Like the extension they take plain
    tensors alone."""

    @staticmethod
    def _plain(*ts):
        for t in ts:
            assert t is None or not torch._C._functorch.is_functorch_wrapped_tensor(t)

    @classmethod
    def norm_forward(cls, x, w, b, eps, keep8, stats):
        cls._plain(x, w, b)
        mean = x.mean(-1, keepdim=True)
        rstd = torch.rsqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
        h = (x - mean) * rstd
        y = (h if w is None else h * cls._over(w, h)) + (0 if b is None else cls._over(b, h))
        return (y, rstd, None, h, torch.zeros(1)) if keep8 else (y, rstd, mean, None, None)

    @classmethod
    def norm_backward(cls, x, rstd, mean, codes, exps, w, b, dy, want):
        cls._plain(x, rstd, mean, codes, exps, w, b, dy)
        h = codes if x is None else (x - mean) * rstd
        gw = dy if w is None else dy * cls._over(w, dy)
        dx = rstd * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))

        def rows(t, like):
            return t.reshape(*((like.shape[0], -1) if like.ndim == 2 else (-1,)), t.shape[-1]).sum(-2)

        return dx, None if w is None else rows(dy * h, w), None if b is None else rows(dy, b)

    @staticmethod
    def _over(w, x):
        return w if w.ndim == 1 else w.reshape(w.shape[0], *(1,) * (x.ndim - 2), w.shape[1])

    @classmethod
    def gate_forward(cls, x, z, keep8):
        cls._plain(x, z)
        return [x * torch.sigmoid(z)] + ([x.clone(), torch.zeros(1), z.clone(), torch.zeros(1)] if keep8 else [])

    @classmethod
    def gate_backward(cls, kept, dy):
        cls._plain(*kept, dy)
        x, z = kept[::2] if len(kept) == 4 else kept
        s = torch.sigmoid(z)
        return dy * s, dy * x * s * (1 - s)


@pytest.fixture
def plain_ops(monkeypatch):
    import kernels  # noqa: F401
    for name in ("kernels.layer_norm", "kernels.kept8"):
        monkeypatch.setattr(sys.modules[name], "flb_ops", PlainOps)


X = torch.randn(3, 20, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
W, B = 1 + 0.1 * X[0], 0.1 * X[1]


def norm(keep8):
    import kernels
    return lambda t: kernels.layer_norm(t, W, B, keep8=keep8), lambda t: torch.nn.functional.layer_norm(t, (20,), W, B)


def gate(keep8):
    import kernels
    return lambda t: kernels.sigmoid_gate(t, t + 1, keep8=keep8), lambda t: t * torch.sigmoid(t + 1)


BOTH = pytest.mark.parametrize("op,keep8", [(norm, False), (norm, True), (gate, False), (gate, True)])


@BOTH
def test_first_derivatives(plain_ops, op, keep8):
    """grad, vjp (its pull called after the transform has ended, and inside it) and vmap give the formula's gradient."""
    f, want_f = op(keep8)
    ours, want = (lambda t, g=g: (g(t) ** 2).sum() for g in (f, want_f))
    want = torch.func.grad(want)(X)
    assert torch.allclose(torch.func.grad(ours)(X), want)
    out, pull = torch.func.vjp(f, X)
    assert torch.allclose(pull(2 * out)[0], want)
    with torch.no_grad():
        assert torch.allclose(pull(2 * out)[0], want)
    assert torch.allclose(torch.func.grad(lambda t: (torch.vmap(f)(t) ** 2).sum())(X), want)
    # a pull inside another transform that it does not depend on
    scale = torch.func.grad(lambda s: s * (pull(2 * out)[0] * X).sum())(torch.tensor(1.0, dtype=torch.float64))
    assert torch.allclose(scale, (want * X).sum())
    # a leaf of plain autograd: the gradient is right, and has a graph that refuses its use
    leaf = X.clone().requires_grad_(True)
    got = torch.func.grad(ours)(leaf)
    assert torch.allclose(got, want) and got.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        got.sum().backward()


@BOTH
def test_second_derivatives_are_refused(plain_ops, op, keep8):
    f, _ = op(keep8)
    for loss in (lambda t: (f(t) ** 2).sum(), lambda t: f(t).sum()):
        inner = torch.func.grad(loss)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.func.grad(lambda t: (inner(t) ** 3).sum())(X)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.func.vjp(inner, X)[1](torch.ones_like(X))
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.func.grad(lambda t: (torch.func.vjp(f, t)[1](torch.ones_like(X))[0] * X).sum())(X)
    # a graph of the gradient that is not used is no error
    assert torch.func.grad(lambda t: (t * torch.func.grad(lambda u: f(u).sum())(X).detach()).sum())(X).shape == X.shape


@BOTH
def test_forward_mode_under_transforms_is_refused(plain_ops, op, keep8):
    f, _ = op(keep8)
    for call in (f, torch.vmap(f), torch.func.grad(lambda t: f(t).sum())):
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            torch.func.jvp(call, (X,), (torch.ones_like(X),))


@BOTH
def test_vmap_over_the_backward_is_refused(plain_ops, op, keep8):
    f, _ = op(keep8)
    with pytest.raises(RuntimeError, match="vmap over this operator's backward"):
        torch.vmap(torch.func.grad(lambda t: f(t).sum()))(X)
    with pytest.raises(RuntimeError, match="vmap over this operator's backward"):
        torch.func.jacrev(f)(X)
    _, pull = torch.func.vjp(f, X)
    with pytest.raises(RuntimeError, match="vmap over this operator's backward"):
        torch.vmap(pull)(X.expand(2, 3, 20))
    with torch.no_grad(), pytest.raises(RuntimeError, match="vmap over this operator's backward"):
        torch.vmap(pull)(X.expand(2, 3, 20))


def test_a_norm_with_groups_under_transforms(plain_ops):
    """A mapped weight: the gradient through vmap and vjp, and its second derivative refused."""
    import kernels
    x, w = X.reshape(3, 2, 10), torch.stack([W[:10], W[10:], W[5:15]])
    f = torch.vmap(lambda p, q: kernels.layer_norm(p, q))
    plain = torch.vmap(lambda p, q: torch.nn.functional.layer_norm(p, (10,), q))
    for k in (0, 1):
        want = torch.func.grad(lambda p, q: (plain(p, q) ** 3).sum(), argnums=k)(x, w)
        ours = torch.func.grad(lambda p, q: (f(p, q) ** 3).sum(), argnums=k)
        assert torch.allclose(ours(x, w), want)
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.func.grad(lambda p, q: ours(p, q).sum(), argnums=k)(x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("keep8", [False, True])
def test_with_the_kernels(keep8):
    """The same with the extension's calls: first derivatives through every transform alike, second ones refused."""
    import kernels
    x = torch.randn(4, 6, 96, device="cuda")
    w = torch.rand(96, device="cuda") + 0.5
    for f in (lambda t: kernels.layer_norm(t, w, keep8=keep8), lambda t: kernels.sigmoid_gate(t, t + 1, keep8=keep8)):
        leaf = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad((f(leaf) ** 2).sum(), leaf)
        loss = lambda t: (f(t) ** 2).sum()  # noqa: E731
        assert torch.equal(torch.func.grad(loss)(x), want)
        assert torch.equal(torch.func.grad(lambda t: (torch.vmap(f)(t) ** 2).sum())(x), want)
        got = torch.func.grad(loss)(leaf)
        assert torch.equal(got, want) and got.requires_grad
        for call in (lambda: got.sum().backward(), lambda: torch.func.grad(lambda t: torch.func.grad(loss)(t).sum())(x)):
            with pytest.raises(RuntimeError, match="differentiable once"):
                call()
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            torch.func.jvp(f, (x,), (x,))
