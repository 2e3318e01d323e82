"""The training step's operators as they are used together: residual add and layer norm with trained weights, the router with
its balance loss, the MoE layer, backward, and the orthogonalised update of every LoRA factor."""
import pytest
import torch

from helpers import to_device_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _step(x, h, w, b, W, ex, lora, mask, coef):
    from smel.loss import balance_loss
    from smel.moe import moe_forward, route
    from smel.norm import add_layernorm
    s, n = add_layernorm(h, x, w, b, 1e-5)
    _, _, topi, logits = route(n, W["mlp.gate.weight"], 4, with_logits=True)
    aux, counts = balance_loss(logits, topi, mask=mask, coef=coef)
    y = s + moe_forward(n, W, ex, 4, lora)
    return y, aux, counts


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_step_together(dt):
    """Each operator's results inside the step are those of its own call on the same values, and the step's gradients are the
    sum of the parts: the layer alone (coef 0) and the balance loss alone, to a few roundings of the type (the dx of either part
    and their sum: 4 half steps of the parts' magnitudes)."""
    from oracle import moe_ref as R
    from smel.lora import orthogonalize
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[dt]
    x, ol = R.make_layer(T=150, H=256, E=16, I=128, K=4, n_sel=3, r=8, alpha=16.0, shared_inter=128, group=64, down_group=64,
                         int4=True, seed=5, lora_b_std=0.02, dtype=torch.float32)
    W, ex, lora = to_device_layer(ol, DEV, dtype)
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g)
    x, h = x.to(DEV, dtype), r(150, 256).to(DEV, dtype)
    mask = (torch.rand(150, generator=g) > 0.2).to(DEV)
    gy = (r(150, 256) * 1e-2).to(DEV, dtype)
    params = list(lora.parameters())

    def grads(gy, coef):
        ts = [t.detach().requires_grad_(True) for t in (x, h, (1 + 0.1 * torch.ones(256)).to(DEV), torch.zeros(256, device=DEV))]
        y, aux, counts = _step(*ts, W, ex, lora, mask, coef)
        loss_terms, cots = (y, aux), (gy, torch.ones((), device=DEV))
        out = torch.autograd.grad(loss_terms, ts + params, cots, allow_unused=True)
        return y, aux, counts, out

    y, aux, counts, both = grads(gy, 0.5)
    assert torch.isfinite(y).all() and torch.isfinite(aux) and counts.sum().item() == 4 * int(mask.sum())
    _, _, _, layer = grads(gy, 0.0)
    _, _, _, aux_only = grads(torch.zeros_like(gy), 0.5)
    half = torch.finfo(dtype).eps / 2
    for i, name in enumerate(("dx", "dh", "dw", "db")):
        a, p, q = (t[i].double() for t in (both, layer, aux_only))
        scale = (p.abs() + q.abs()) if i < 2 else (p.abs() + q.abs()).max()
        row = (p.abs() + q.abs()).amax(-1, keepdim=True) if i < 2 else 0     # the norm's backward mixes a row
        assert ((a - p - q).abs() <= 16 * half * (scale + row)).all(), name
    for p, a in zip(layer[4:], both[4:]):     # the balance loss does not reach the factors
        assert torch.equal(p, a)
    updates = orthogonalize(both[4:])
    for p, grad, u in zip(params, both[4:], updates):
        assert u.shape == p.shape and torch.isfinite(u).all()
        assert torch.equal(u, orthogonalize(grad))
        with torch.no_grad():
            p.add_(u, alpha=-1e-3)
    y2, _, _, _ = grads(gy, 0.5)
    assert not torch.equal(y2, y)
