"""The end of one block and the beginning of the next as a training step uses them: the norms around the residual add, experts chosen
by scores, bias and groups, the routed experts and the shared one, backward, and all gradients clipped together."""
import pytest
import torch

from helpers import to_device_layer

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _step(h, a, w1, w2, w3, gate, scale, W, ex, lora, bias):
    from smel.moe import route_grouped, routed_experts, shared_mlp
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    s, n = sandwich_rmsnorm(h, a, w1, w2, 1e-6, gate=gate, gate_act="sigmoid", scale=scale)
    scores, topv, topi = route_grouped(n, W["mlp.gate.weight"], 4, bias=bias, groups=4, top_groups=2, scale=2.0)
    y = routed_experts(n, topv, topi, ex, lora.experts) + shared_mlp(n, W, lora.shared)
    return post_rmsnorm(s, y, w3, 1e-6), topi


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_block_step(dt):
    """Every gradient is there, finite and the same on a second run; the experts' part is what the picks say (a step with the picks
    forced by the bias alone uses only them); the clipped gradients have the norm asked for."""
    from oracle import moe_ref as R
    from smel.lora import clip_grads, clip_grads_, grad_norm
    dtype = {"bf16": torch.bfloat16, "fp32": torch.float32}[dt]
    x, ol = R.make_layer(T=150, H=256, E=16, I=128, K=4, n_sel=3, r=8, alpha=16.0, shared_inter=128, group=64, down_group=64,
                         int4=True, seed=5, lora_b_std=0.02, dtype=torch.float32)
    W, ex, lora = to_device_layer(ol, DEV, dtype)
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    params = list(lora.parameters())
    bias = 0.1 * r(16)
    start = [x.to(DEV, dtype), r(150, 256).to(dtype), 1 + 0.1 * r(256), 1 + 0.1 * r(256), 1 + 0.1 * r(256), 0.1 * r(256), torch.full((1,), 0.8, device=DEV)]
    gy = (r(150, 256) * 1e-2).to(dtype)

    def grads(bias=bias):
        ts = [t.detach().requires_grad_(True) for t in start]
        y, topi = _step(*ts, W, ex, lora, bias)
        return y, topi, torch.autograd.grad(y, ts + params, gy)
    y, topi, gr = grads()
    assert torch.isfinite(y).all() and all(torch.isfinite(t).all() and t.any() for t in gr[:7])
    y2, topi2, gr2 = grads()
    assert torch.equal(y, y2) and torch.equal(topi, topi2) and all(torch.equal(a, b) for a, b in zip(gr, gr2))
    forced = torch.full((16,), -10.0, device=DEV)
    forced[[1, 2, 8, 11]] = 10.0
    _, topi3, _ = grads(forced)
    assert (topi3.sort(1).values == torch.tensor([1, 2, 8, 11], device=DEV)).all()
    out, norm = clip_grads(gr, 0.01)
    ref = torch.sqrt(sum(t.double().square().sum() for t in gr))
    assert abs(float(norm) - float(ref)) <= 2 ** -23 * float(ref) and float(norm) > 0.01
    assert float(grad_norm(out)) == pytest.approx(0.01, rel=2 ** -8)
    assert torch.equal(clip_grads_(list(gr), 0.01), norm) and all(torch.equal(a, b) for a, b in zip(gr, out))
