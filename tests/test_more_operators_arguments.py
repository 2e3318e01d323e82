"""Arguments of clipping that are no numbers (no GPU): refused, not taken for another call."""
import pytest
import torch

from smel.lora import clip_grads, clip_grads_


def test_no_max_norm():
    for ts in ([], [torch.ones(3)]):
        for f in (clip_grads, clip_grads_):
            with pytest.raises(TypeError):
                f(ts, None)
