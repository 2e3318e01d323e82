"""The norms around a residual add on one row without leading dimensions: a gate [n] is one per channel where its dtype is the weights',
else one per element, of the row's dtype."""
import pytest
import torch

from test_gpu_sandwich import DEV, DT, EPS, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "sigmoid"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_full_gate_beside_wide_weights(dt, act):
    """As the same row with a leading dimension, bit for bit."""
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    t, ds, dy = make(1, 200, DT[dt], torch.float32, 5, "full", "tensor")
    go = (ds.to(DEV), dy.to(DEV))

    def run(lead, only=None, w2=True):
        ls = {k: (v[0] if k in ("h", "x", "gate") and not lead else v).to(DEV).requires_grad_(True) for k, v in t.items()}
        kw = dict(gate=ls["gate"], gate_act=act, scale=ls["scale"])
        if only is None:
            out = sandwich_rmsnorm(ls["h"], ls["x"], ls["w1"], ls["w2"] if w2 else None, EPS, **kw)
        else:
            out = (post_rmsnorm(ls["h"], ls["x"], ls["w1"], EPS, **kw),)
        need = [ls[k] for k in ("h", "x", "w1", "gate", "scale")]
        gr = torch.autograd.grad(out, need, [d if lead else d[0] for d in go[:len(out)]])
        return [v.detach().reshape(-1) for v in (*out, *gr)]
    for kw in ({}, {"w2": False}, {"only": "post"}):
        assert all(torch.equal(a, b) for a, b in zip(run(False, **kw), run(True, **kw)))


def test_channel_gate_of_the_weights_dtype_stays():
    from smel.norm import post_rmsnorm
    t, ds, _ = make(1, 64, torch.bfloat16, torch.float32, 7, "channel")
    h, x, w, gate = (t[k].to(DEV) for k in ("h", "x", "w1", "gate"))
    assert gate.dtype == torch.float32
    assert torch.equal(post_rmsnorm(h[0], x[0], w, EPS, gate=gate), post_rmsnorm(h, x, w, EPS, gate=gate)[0])
    assert torch.equal(post_rmsnorm(h[0], x[0], None, EPS, gate=gate), post_rmsnorm(h, x, None, EPS, gate=gate)[0])
    with pytest.raises(ValueError):      # neither the weights' dtype nor the row's
        post_rmsnorm(h[0], x[0], w, EPS, gate=gate.half())
    with pytest.raises(ValueError):
        post_rmsnorm(h[0], x[0], w.bfloat16(), EPS, gate=gate)


def test_one_row_of_one_column():
    """[1] of fp32 beside 16-bit weights is the row's gate."""
    from smel.norm import post_rmsnorm
    t, _, _ = make(1, 1, torch.bfloat16, torch.bfloat16, 7, "token", gate_dt=torch.float32)
    h, x, w, gate = (t[k].to(DEV) for k in ("h", "x", "w1", "gate"))
    assert torch.equal(post_rmsnorm(h[0], x[0], w, EPS, gate=gate[0]), post_rmsnorm(h, x, w, EPS, gate=gate)[0])
