"""route_grouped (smel.moe) where the router's product and the choice behind it meet their edges."""
import pytest
import torch

from test_gpu_second_derivative import DEV, check

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.mark.parametrize("H,dt", [(128, "bf16"), (72, "bf16"), (128, "fp32")])
def test_second_derivative_refused(H, dt):
    from smel.moe import route_grouped
    w = torch.randn(16, H, device=DEV).to(DT[dt])
    check(lambda x: route_grouped(x, w, 2, groups=4, top_groups=2, renorm=False), 9, H, dtype=DT[dt])
    check(lambda x: route_grouped(x, w, 2, with_logits=True)[3], 9, H, dtype=DT[dt])
