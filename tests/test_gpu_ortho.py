"""Orthogonalised updates (smel.lora.orthogonalize over include/smel_ortho.h) against the formula in 64 bits.

Tolerance, from the arithmetic: the products run in 64 bits, whose 2^-53 grows by at most a^2 = 11.9 a step (the square of a
small singular value's growth), 2.3e5 in five steps, times a few hundred terms: under 1e-8 of a result whose singular values
are about 1; then one rounding to fp32. 16-bit results come from fp32 sums of r products of Q's 24-bit values: off by at most
3 r + 8 roundings (three parts of Q, r terms each) of sum |Q| |G|, X = Q G, before their own rounding."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
COEFFS = (3.4445, -4.7750, 2.0315)
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def formula(G, steps=5, coeffs=COEFFS, eps=1e-7):
    X = G.double()
    X = X / (torch.sqrt((X * X).sum(dim=(-2, -1), keepdim=True)) + eps)
    a, b, c = coeffs
    flip = X.shape[-2] > X.shape[-1]
    X = X.transpose(-2, -1) if flip else X
    size = X.abs()
    Q = torch.eye(X.shape[-2], dtype=torch.float64).expand(*X.shape[:-2], -1, -1)
    for _ in range(steps):
        S = X @ X.transpose(-2, -1)
        P = b * S + c * (S @ S)
        X, Q = a * X + P @ X, a * Q + P @ Q
    size = Q.abs() @ size
    return (X.transpose(-2, -1), size.transpose(-2, -1)) if flip else (X, size)


def close(got, G, what, **kw):
    want, size = formula(G.cpu(), **kw)
    g = got.cpu().double()
    assert got.dtype == G.dtype and g.shape == want.shape and got.is_contiguous(), what
    bar = (torch.finfo(got.dtype).eps / 2 * (1 + 2 ** -8) + 2.0 ** -24) * want.abs() + TINY[got.dtype] + 1e-8
    if got.dtype != torch.float32:
        bar = bar + (3 * min(G.shape[-2:]) + 8) * 2.0 ** -24 * size
    bad = ~((g - want).abs() <= bar)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {((g - want).abs() / bar).max()}"


def make(shape, dt, seed, decades=2.0):
    g = torch.Generator().manual_seed(seed)
    *lead, m, n = shape
    r = min(m, n)
    scale = torch.pow(10.0, -decades * torch.arange(r) / max(1, r - 1))
    x = (torch.randn(*lead, r, r, generator=g) * scale) @ torch.randn(*lead, r, max(m, n), generator=g) * 1e-2
    return (x if m <= n else x.transpose(-2, -1)).to(DT[dt]).contiguous()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 5), (5, 1), (2, 3), (4, 4), (16, 16), (17, 17), (3, 16, 2048), (3, 2048, 16),
                                   (6, 700), (16, 1), (5, 33, 129), (2, 129, 33), (48, 1000), (2, 64, 127), (127, 64),
                                   (2, 128, 128), (2, 100, 2816), (128, 1030), (1500, 128), (2, 2, 8, 2049), (7, 15, 31)])
def test_orthogonalize(shape, dt):
    from smel.lora import orthogonalize
    G = make(shape, dt, sum(shape))
    got = orthogonalize(G.to(DEV))
    close(got, G, shape)
    assert torch.equal(got, orthogonalize(G.to(DEV)))


@pytest.mark.parametrize("decades", [0.0, 4.0, 6.0])
@pytest.mark.parametrize("r", [16, 40, 128])
def test_orthogonalize_spread(r, decades):
    """Singular values far under the largest keep their directions."""
    from smel.lora import orthogonalize
    G = make((2, r, 600), "fp32", r, decades)
    close(orthogonalize(G.to(DEV)), G, r)


@pytest.mark.parametrize("steps,coeffs,eps", [(0, COEFFS, 1e-7), (1, COEFFS, 1e-7), (2, (1.5, -0.5, 0.0), 0.0), (12, (1.875, -1.25, 0.375), 1e-7),
                                              (5, COEFFS, 0.5)])
@pytest.mark.parametrize("r", [8, 24, 60, 120])
def test_orthogonalize_steps(r, steps, coeffs, eps):
    from smel.lora import orthogonalize
    G = make((r, 300), "fp32", r, 1.0)
    close(orthogonalize(G.to(DEV), steps, coeffs, eps), G, r, steps=steps, coeffs=coeffs, eps=eps)


def test_orthogonalize_moves_singular_values_to_one():
    from smel.lora import orthogonalize
    G = make((24, 500), "fp32", 3, 1.0)
    s = torch.linalg.svdvals(orthogonalize(G.to(DEV), 20, (1.875, -1.25, 0.375)).double().cpu())
    assert (s - 1).abs().max() <= 24 * 500 * 2.0 ** -24


def test_orthogonalize_list():
    """A layer's factors, more than one launch's worth of jobs, mixed types, shapes and ranks, an empty one, the same tensor
    twice: each result is that of its own call."""
    from smel.lora import orthogonalize
    shapes = [(4, 16, 256), (4, 64, 16), (16, 256), (64, 16), (3, 40, 90), (2, 100, 300), (0, 16, 64), (5, 0, 7), (1, 1)]
    ts = [make(s, ("fp32", "bf16", "fp16")[i % 3], i) if 0 not in s else torch.zeros(s) for i, s in enumerate(shapes * 11)]
    dev = [t.to(DEV) for t in ts]
    dev.append(dev[0])
    out = orthogonalize(dev)
    assert isinstance(out, list) and len(out) == len(dev)
    for t, y in zip(dev, out):
        assert y.shape == t.shape and y.dtype == t.dtype
        assert torch.equal(y, orthogonalize(t))
    for t, y in list(zip(dev, out))[:9]:
        if t.numel():
            close(y, t, tuple(t.shape))
    assert orthogonalize([]) == [] and len(orthogonalize((dev[0],))) == 1


def test_orthogonalize_views():
    from smel.lora import orthogonalize
    base = make((4, 48, 400), "fp32", 5)
    b = base.to(DEV)
    views = {"transposed": lambda t: t.transpose(1, 2), "columns": lambda t: t[:, :, 3:203], "rows": lambda t: t[:, ::3],
             "columns apart": lambda t: t[:, :, ::2], "batch apart": lambda t: t[::2], "swapped": lambda t: t.transpose(0, 1),
             "one row": lambda t: t[:, 7:8, ::3], "one column": lambda t: t[:, :, 11:12], "expanded": lambda t: t[:1].expand(3, 48, 400),
             "lead": lambda t: t.view(2, 2, 48, 400).transpose(0, 1), "4d slice": lambda t: t.view(2, 2, 48, 400)[:, 1:]}
    before = b.clone()
    for name, view in views.items():
        v = view(b)
        close(orthogonalize(v), v, name)
    assert torch.equal(b, before)


def test_orthogonalize_special_values():
    """A zero matrix stays zero; NaN or inf spoils its own matrix alone; tiny and huge scales do not matter."""
    from smel.lora import orthogonalize
    G = make((5, 16, 300), "fp32", 6)
    G[1] = 0
    G[2, 3, 299] = float("nan")
    G[3, 0, 0] = float("inf")
    y = orthogonalize(G.to(DEV)).cpu()
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    close(y[[0, 4]], G[[0, 4]], "others")
    for scale in (1e30, 1e-30):
        for rows in (16, 48, 100):
            H = make((rows, 300), "fp32", rows) * scale
            close(orthogonalize(H.to(DEV), eps=0.0), H, scale, eps=0.0)
            H = H.bfloat16()
            close(orthogonalize(H.to(DEV), eps=0.0), H, scale, eps=0.0)


def test_orthogonalize_parameters_carry_no_graph():
    from smel.lora import ExpertsLoRA, orthogonalize
    lora = ExpertsLoRA([0, 3, 5], 128, 64, r=6).to(DEV)
    for p in lora.parameters():
        p.grad = torch.randn_like(p)
    out = orthogonalize([p.grad for p in lora.parameters()])
    for p, o in zip(lora.parameters(), out):
        close(o, p.grad, tuple(p.shape))
    w = torch.randn(4, 8, device=DEV, requires_grad=True)
    assert not orthogonalize(w).requires_grad


def test_orthogonalize_graph_and_streams():
    from smel.lora import orthogonalize
    a = [make(s, "fp32", i).to(DEV) for i, s in enumerate([(6, 16, 512), (40, 300), (2, 128, 200)])]
    b = [t * 0.5 + 1e-3 for t in a]
    ref, ref2 = [t.clone() for t in orthogonalize(a)], [t.clone() for t in orthogonalize(b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(a)
    for _ in range(3):
        for t in out:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, ref))
        assert all(torch.equal(x, y) for x, y in zip(orthogonalize(b), ref2))
    for _ in range(3):
        with torch.cuda.stream(side):
            two = orthogonalize(b)
        one = orthogonalize(a)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(one, ref)) and all(torch.equal(x, y) for x, y in zip(two, ref2))


def test_orthogonalize_refusals():
    from smel.lora import orthogonalize
    x = torch.zeros(4, 8, device=DEV)
    for bad in (lambda: orthogonalize(torch.zeros(129, 200, device=DEV)), lambda: orthogonalize(x.double()),
                lambda: orthogonalize(x[0]), lambda: orthogonalize([x, x.cpu()]), lambda: orthogonalize(x, coeffs=(1.0, 2.0)),
                lambda: orthogonalize([x, x.long()])):
        with pytest.raises(ValueError):
            bad()


def test_orthogonalize_far_offsets():
    """Matrices, rows and columns whose offsets pass 2^31 elements: the same bits as packed ones."""
    from smel.lora import orthogonalize
    big = torch.zeros(1100 << 21, dtype=torch.bfloat16, device=DEV)
    G = make((3, 16, 700), "bf16", 4).to(DEV)
    far = big.as_strided((3, 16, 700), (1 << 30, 1 << 21, 1))
    far.copy_(G)
    assert torch.equal(orthogonalize(far), orthogonalize(G))
    H = make((16, 1000), "bf16", 5).to(DEV)
    lines = big.as_strided((16, 1000), (1, 1 << 21))
    lines.copy_(H)
    assert torch.equal(orthogonalize(lines), orthogonalize(H))


def test_orthogonalize_many_matrices():
    """More matrices than a launch takes above rank 64, and many small ones: each as alone."""
    from smel.lora import orthogonalize
    G = make((300, 72, 80), "fp32", 6).to(DEV)
    y = orthogonalize(G)
    for k in (0, 255, 256, 299):
        assert torch.equal(y[k], orthogonalize(G[k]))
    close(y[[0, 255, 256, 299]], G[[0, 255, 256, 299]], "ends")
    S = make((70000, 2, 5), "fp32", 7).to(DEV)
    y = orthogonalize(S)
    close(y[[0, 65535, 65536, 69999]], S[[0, 65535, 65536, 69999]], "ends")
