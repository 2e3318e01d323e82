"""A second derivative through this package's functions is refused, not dropped: also where the first one's incoming gradient is a
constant (a sum's), so that nothing but the function itself could tell."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(f, *shape, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(*shape, generator=g).to(DEV, dtype).requires_grad_(True)

    def loss():
        outs = f(x)
        outs = outs if isinstance(outs, tuple) else (outs,)
        return sum(t.float().sum() for t in outs if t.requires_grad)
    plain, = torch.autograd.grad(loss(), x)
    dx, = torch.autograd.grad(loss(), x, create_graph=True)
    assert torch.equal(dx.detach(), plain) and not plain.requires_grad and dx.requires_grad
    penalty = dx.float().square().sum() + x.float().sum()
    with pytest.raises(RuntimeError, match="once"):
        penalty.backward()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_select(score):
    from smel.moe import select_experts
    check(lambda x: select_experts(x, 4, score, groups=4, top_groups=2, renorm=False), 40, 64)


def test_sandwich():
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    w, h = torch.rand(96, device=DEV), torch.randn(9, 96, device=DEV).bfloat16()
    check(lambda x: sandwich_rmsnorm(h, x, w, w, 1e-6), 9, 96)
    check(lambda x: post_rmsnorm(h, x, w, 1e-6), 9, 96)
    check(lambda x: post_rmsnorm(x, h, w, 1e-6), 9, 96)      # the gradient goes through as it is
    check(lambda x: post_rmsnorm(h, h, w, 1e-6, gate=x), 9, 96)


def test_layernorm_and_balance():
    from smel.loss import balance_loss
    from smel.norm import add_layernorm, layernorm
    w, h = torch.rand(96, device=DEV), torch.randn(9, 96, device=DEV).bfloat16()
    check(lambda x: layernorm(x, w, w, 1e-5), 9, 96)
    check(lambda x: add_layernorm(h, x, w, w, 1e-5), 9, 96)
    check(lambda x: add_layernorm(x, x, w, w, 1e-5), 9, 96)
    check(lambda x: balance_loss(x, torch.arange(18, device=DEV).view(9, 2) % 64), 9, 64)
