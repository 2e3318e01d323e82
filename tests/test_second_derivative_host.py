"""smel._lib.once: a backward's results keep their values and refuse to be differentiated again (no GPU)."""
import pytest
import torch

from smel import _lib


def _backward(ctx, d):
    x, = ctx.saved_tensors
    dx = 2 * x * d
    return dx, None, dx


class _Squares(torch.autograd.Function):
    """x x + b, with a gradient of b that is x's (one tensor twice)."""

    @staticmethod
    def forward(ctx, x, n, b):
        ctx.save_for_backward(x)
        return x * x

    backward = staticmethod(_lib.once(_backward))


@pytest.mark.parametrize("constant", [True, False])
def test_refused(constant):
    x, b = torch.randn(5).requires_grad_(True), torch.randn(5).requires_grad_(True)

    def loss():
        y = _Squares.apply(x, 3, b)
        return y.sum() if constant else (y * y).sum()
    plain = torch.autograd.grad(loss(), (x, b))
    both = torch.autograd.grad(loss(), (x, b), create_graph=True)
    assert all(torch.equal(p, q.detach()) and not p.requires_grad and q.requires_grad for p, q in zip(plain, both))
    for g in both:
        with pytest.raises(RuntimeError, match="once"):
            (g.square().sum() + x.sum()).backward(retain_graph=True)
    x.grad = None     # of the other term, which came first
    loss().backward()
    assert torch.equal(x.grad, plain[0]) and not x.grad.requires_grad


def test_frozen_inputs():
    """Without a leaf that asks for it, and with a single result that is missing."""
    b = torch.randn(5).requires_grad_(True)
    g, = torch.autograd.grad(_Squares.apply(torch.ones(5), 0, b).sum(), b, create_graph=True)
    assert torch.equal(g.detach(), torch.full((5,), 2.0))

    class Nothing(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 1

        backward = staticmethod(_lib.once(lambda ctx, d: None))
    x = torch.ones(3, requires_grad=True)
    assert torch.autograd.grad(Nothing.apply(x).sum(), x, create_graph=True, allow_unused=True) == (None,)
