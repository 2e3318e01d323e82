"""The router's entry points refuse rows and weights of different widths, or on different devices, on the host before any launch: the
kernels would read past the weight (no GPU: tensors without memory stand for the operands)."""
import pytest
import torch

from smel import _lib, moe

M = dict(device="meta")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [128, 72])
def test_widths(monkeypatch, H, dt):
    monkeypatch.setattr(_lib, "require_device", lambda *ts: None)
    monkeypatch.setattr(_lib, "one_device", lambda *ts: None)
    x = torch.empty(4, H, dtype=dt, **M)
    for w in (torch.empty(16, H // 2, dtype=dt, **M), torch.empty(16, 2 * H, dtype=dt, **M), torch.empty(H, dtype=dt, **M),
              torch.empty(1, 16, H, dtype=dt, **M)):
        W = {"router.proj.weight": w, "router.scale": torch.empty(H, dtype=dt, **M), "router.per_expert_scale": torch.empty(16, dtype=dt, **M)}
        for f in (lambda: moe.route(x, w, 2), lambda: moe.route_grouped(x, w, 2), lambda: moe.route_gemma4(x, W, 2, 1e-6)):
            with pytest.raises(ValueError, match="router weight"):
                f()
    w = torch.empty(16, H, dtype=dt, **M)
    for f in (lambda: moe.route(x[0], w, 2), lambda: moe.route_grouped(x.view(2, 2, H), w, 2)):
        with pytest.raises(ValueError, match="router weight"):
            f()
    good = {"router.proj.weight": w, "router.scale": torch.empty(H, dtype=dt, **M), "router.per_expert_scale": torch.empty(16, dtype=dt, **M)}
    for name, n in (("router.scale", H - 1), ("router.per_expert_scale", 15)):
        with pytest.raises(ValueError, match=name):
            moe.route_gemma4(x, {**good, name: torch.empty(n, dtype=dt, **M)}, 2, 1e-6)


class _On:
    """A GPU's tensor as far as the device check looks."""

    def __init__(self, device):
        self.device, self.is_cuda, self.dtype, self.shape = torch.device(device), True, torch.bfloat16, (4, 128)


def test_devices():
    for f in (moe.route, moe.route_grouped):
        with pytest.raises(ValueError, match="one call on cuda:0 and cuda:1"):
            f(_On("cuda:0"), _On("cuda:1"), 2)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layer(monkeypatch, dt):
    monkeypatch.setattr(_lib, "require_device", lambda *ts: None)
    monkeypatch.setattr(_lib, "one_device", lambda *ts: None)
    for H in (64, 256):
        with pytest.raises(ValueError, match="router weight"):
            moe.moe_forward(torch.empty(4, 128, dtype=dt, **M), {"mlp.gate.weight": torch.empty(16, H, dtype=dt, **M)}, None, 2)
