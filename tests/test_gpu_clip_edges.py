"""Clipping by the global norm (smel.lora): forward-mode tangents, and the norm's sums over several launches."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_tangents_are_refused():
    """None of the three has a rule for forward mode: a tangent raises before anything is written, values without one go through."""
    from smel.lora import clip_grads, clip_grads_, grad_norm
    x, other = torch.full((40,), 2.0, device=DEV), torch.full((8,), 3.0, device=DEV)
    want, norm = clip_grads([other, x], 1.0)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for bad in (lambda: grad_norm([other, d]), lambda: grad_norm(d), lambda: clip_grads([other, None, d], 1.0), lambda: clip_grads_([other, d], 1.0),
                    lambda: clip_grads_(d, 1.0)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward mode"):
                    bad()
        assert torch.equal(x, torch.full((40,), 2.0, device=DEV)) and torch.equal(other, torch.full((8,), 3.0, device=DEV))
        out, n2 = clip_grads([other, x], 1.0)
        assert torch.equal(n2, norm) and all(torch.equal(a, b) for a, b in zip(out, want))
    assert torch.equal(clip_grads_([other, x], 1.0), norm) and torch.equal(x, want[1]) and torch.equal(other, want[0])


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_same_bits_as_one_launch(kind):
    """500 tensors of a chunk each take five launches, their concatenation one: the same parts, added in the same order."""
    from smel.lora import clip_grads, grad_norm
    g = torch.Generator().manual_seed(6)
    flat = torch.randn(500 * 8192, generator=g).to(DEV)
    ts = list(flat.split(8192))
    out, norm = clip_grads(ts, 1.0, kind)
    one, n1 = clip_grads([flat], 1.0, kind)
    assert torch.equal(norm, n1) and torch.equal(torch.cat(out), one[0]) and torch.equal(grad_norm(ts, kind), n1)


def test_within_the_norm():
    """In place, a strided tensor goes through a copy, also with a factor of 1: its values, and those beside it, stay."""
    from smel.lora import clip_grads_
    base = torch.randn(30, 40, device=DEV)
    want = base.clone()
    norm = clip_grads_([base[:, ::3], base[1::2, 1]], 1e9)
    assert torch.equal(base, want) and float(norm) < 1e9
    assert clip_grads_([None], 1.0).device.type == "cpu"      # no tensor says where
