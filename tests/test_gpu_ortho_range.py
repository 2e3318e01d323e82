"""smel.lora.orthogonalize at the ends of its types' ranges, and at sizes where a block takes several slices of columns; the
tolerances are those of test_gpu_ortho."""
import pytest
import torch

from test_gpu_ortho import DT, close, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("steps", [5, 9])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [16, 24, 48, 100])
def test_largest_values(rows, dt, steps):
    """Values up to the type's largest: |G|_F passes 2^128, and 1 / |G|_F lies under the smallest normal value."""
    from smel.lora import orthogonalize
    G = make((rows, 300), "fp32", rows, 1.0)
    G = (G / G.abs().max() * 3.3e38).to(DT[dt])
    assert torch.isfinite(G).all()
    close(orthogonalize(G.to(DEV), steps), G, dt, steps=steps)
