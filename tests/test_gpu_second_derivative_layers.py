"""A second derivative through the router's and the layer's functions is refused, not dropped (test_gpu_second_derivative.py has the
training step's operators)."""
import pytest
import torch

from helpers import to_device_layer
from test_gpu_second_derivative import DEV, check

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.mark.parametrize("H,dt", [(128, "bf16"), (72, "bf16"), (128, "fp32")])
def test_route(H, dt):
    from smel.moe import route, route_gemma4
    w = torch.randn(16, H, device=DEV).to(DT[dt])
    W = {"router.scale": torch.ones(H, device=DEV).to(DT[dt]), "router.proj.weight": w,
         "router.per_expert_scale": torch.rand(16, device=DEV).to(DT[dt])}
    for logits in (False, True):
        check(lambda x: route(x, w, 2, with_logits=logits), 9, H, dtype=DT[dt])
        check(lambda x: route_gemma4(x, W, 2, 1e-6, with_logits=logits), 9, H, dtype=DT[dt])


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_layer(dt):
    from oracle import moe_ref as R
    from smel.moe import FrozenExpertsFn, moe_forward, route, routed_experts, shared_mlp
    _, ol = R.make_layer(T=4, H=256, E=16, I=128, K=4, n_sel=3, r=8, alpha=16.0, shared_inter=128, group=64, down_group=64, int4=True,
                         seed=5, lora_b_std=0.02, dtype=torch.float32)
    W, ex, lora = to_device_layer(ol, DEV, DT[dt])
    _, topv, topi = route(torch.randn(20, 256, device=DEV).to(DT[dt]), W["mlp.gate.weight"], 4)
    check(lambda x: routed_experts(x, topv, topi, ex, lora.experts), 20, 256, dtype=DT[dt])
    check(lambda x: shared_mlp(x, W, lora.shared), 20, 256, dtype=DT[dt])
    check(lambda x: moe_forward(x, W, ex, 4, lora), 20, 256, dtype=DT[dt])
    check(lambda x: FrozenExpertsFn.apply(x, [2] * 16, ex.frozen, 32, "silu"), 32, 256, dtype=DT[dt])


def test_norms_and_loss():
    from smel.loss import LMHead, chunked_ce
    from smel.norm import add_rmsnorm, gated_rmsnorm, rmsnorm
    w, h = torch.rand(96, device=DEV).bfloat16(), torch.randn(9, 96, device=DEV).bfloat16()
    check(lambda x: rmsnorm(x, w, 1e-6, False), 9, 96)
    check(lambda x: add_rmsnorm(h, x, w, 1e-6, True), 9, 96)
    check(lambda x: add_rmsnorm(h, x, w, 1e-6, True)[0], 9, 96)      # the gradient goes through as it is
    check(lambda x: gated_rmsnorm(x, h, w, 1e-6), 9, 96)
    head = LMHead(weight=torch.randn(300, 128, device=DEV).bfloat16(), vocab_chunk=128)
    check(lambda x: chunked_ce(x, head, torch.arange(40, device=DEV), denom=40.0), 40, 128)
