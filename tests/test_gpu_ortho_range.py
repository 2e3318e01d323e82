"""smel.lora.orthogonalize at the ends of its types' ranges, and at sizes where a block takes several slices of columns; the
tolerances are those of test_gpu_ortho."""
import math

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


def plan(shapes, dt):
    """(columns of an apply block, columns of a gram block, columns of a gram slice) of a launch over these matrices of one rank's
    tiles: the sizes say which code of the kernels runs."""
    cols = sum(math.prod(s[:-2]) * max(s[-2:]) for s in shapes)
    nt = {1: 1, 2: 2, 3: 4, 4: 4}[(min(shapes[0][-2:]) + 15) // 16]
    apply = {1: 1024, 2: 256 if dt == "fp32" else 512, 4: 256}[nt]
    while apply > 128 and cols // apply < 192:
        apply //= 2
    gram = {1: 512, 2: 256, 4: 128}[nt]
    while gram > 128 and cols // gram < 512:
        gram //= 2
    return apply, max(gram, cols // 512 // 16 * 16), gram


CASES = [   # lead, short, long, its apply block's columns (fp32, 16 bits), whether a gram block takes more than a slice
    (12, 16, 2049, 128, False), (25, 16, 2051, 256, False), (50, 13, 2049, 512, True), (100, 16, 2049, 1024, True),
    (110, 9, 2819, 1024, True), (50, 24, 2049, 256, True), (75, 31, 2819, 256, True), (18, 60, 2819, 256, False),
    (72, 60, 2819, 256, True), (72, 33, 2049, 256, True)]


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("lead,r,n,apply,several", CASES)
def test_many_columns(lead, r, n, apply, several, tall, dt):
    """Blocks of every size: each width of an apply block, gram blocks of several slices with a part of one at the end."""
    from smel.lora import orthogonalize
    shape = (lead, n, r) if tall else (lead, r, n)
    a, block, piece = plan([shape], dt)
    assert a == apply or dt != "fp32" and r > 16 and r <= 32 and a == 512
    assert (block > piece) == several
    G = make(shape, dt, r + n)
    close(orthogonalize(G.to(DEV)), G, shape)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_layer_of_updates(dt):
    """Every factor of a layer, twelve experts and the shared one, in one call: apply blocks of 512 columns, gram blocks of a slice and
    a half."""
    from smel.lora import orthogonalize
    r, H, I = 16, 2048, 512
    one = lambda lead: [(*lead, r, H), (*lead, I, r), (*lead, r, H), (*lead, I, r), (*lead, r, I), (*lead, H, r)]
    shapes = one((12,)) + one(())
    assert plan(shapes, dt) == (512, 192, 128)
    ts = [make(s, dt, i) for i, s in enumerate(shapes)]
    for t, y in zip(ts, orthogonalize([t.to(DEV) for t in ts])):
        close(y, t, tuple(t.shape))


def test_columns_of_several_launches():
    """2^32 columns in one call, from one row read 65536 times."""
    from smel.lora import orthogonalize
    row = make((1, 1, 65536), "bf16", 3)
    y = orthogonalize(row.to(DEV).expand(65536, 1, 65536))
    for k in (0, 4095, 4096, 32767, 32768, 65535):
        close(y[k], row[0], k)
    assert torch.equal(y[1:].amin(0), y[0]) and torch.equal(y[1:].amax(0), y[0])
