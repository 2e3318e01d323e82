"""smel.lora.orthogonalize over its whole range of steps, ranks that the updates do not fill, and scales, against the formula in
64 bits.

Tolerance, from the arithmetic (u = 2^-53): up to K steps, a^(2 K) <= 2^24, run on the r x r matrices, whose rounding grows by a^2 a
step; up to 2 K in two such passes; more as the formula itself, step by step in 64 bits. A sum over n columns and the r x r products
leave (n + r) u of X's size at every step, on either side. What lies in a direction of singular value s (of X0) grows by a at most a
step until it is about 1 and stays there: by min(a^steps, 1 / s). So both sides are off by 2 (n + r) u (min(a^steps, 1 / s_min) + a^(2 k)),
k the steps of a pass on the r x r matrices, then by the result's rounding. 16-bit results of a single
pass come from fp32 sums: (3 r + 8) 2^-24 of sum |Q| |G| more, X = Q G (derived in test_gpu_ortho); of more passes from 64-bit sums."""
import pytest
import torch

from test_gpu_ortho import COEFFS, DT, TINY, formula, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def limit(a):
    """Steps that one pass on the r x r matrices takes."""
    k = 1
    while k < 64 and max(1.0, a * a) ** (k + 1) <= 2.0 ** 24:
        k += 1
    return k


def close(got, G, steps, coeffs=COEFFS, eps=1e-7, smallest=None, what=""):
    G = G.cpu()
    want, size = formula(G, steps, coeffs, eps)
    g = got.cpu().double()
    assert got.dtype == G.dtype and g.shape == want.shape and got.is_contiguous(), what
    m, n = G.shape[-2:]
    a, K = abs(coeffs[0]), limit(coeffs[0])
    X = G.double()
    X = X / (torch.sqrt((X * X).sum(dim=(-2, -1), keepdim=True)) + eps)
    s = torch.linalg.svdvals(X).min().item() if smallest is None else smallest
    k = steps if steps <= K else (steps + 1) // 2 if steps <= 2 * K else 0
    noise = 2 * (m + n) * 2.0 ** -53 * (min(max(a, 1.0) ** steps, 1 / max(s, 1e-300)) + max(a, 1.0) ** (2 * k))
    if noise > 1e-2:      # entries are of 0.03 to 0.3: null directions grown from either side's rounding; of the formula's size
        assert torch.linalg.svdvals(g).max() <= max(torch.linalg.svdvals(want).max(), 1.0) + 0.3, what
        return
    bar = (torch.finfo(got.dtype).eps / 2 * (1 + 2 ** -8) + 2.0 ** -24) * want.abs() + TINY[got.dtype] + noise
    if steps <= K and got.dtype != torch.float32:
        bar = bar + (3 * min(m, n) + 8) * 2.0 ** -24 * size
    bad = ~((g - want).abs() <= bar)
    assert not bad.any(), f"{what} {tuple(G.shape)} {steps}: {int(bad.sum())} of {bad.numel()}, worst {((g - want).abs() / bar).max()}"


def outer(tokens, r, n, seed, lead=()):
    """A factor's gradient from a few tokens, as it is kept in fp32: of that rank but for its rounding."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*lead, r, tokens, generator=g) @ torch.randn(*lead, tokens, n, generator=g)


@pytest.mark.parametrize("steps", [5, 6, 7, 8, 12, 13, 20, 64])
@pytest.mark.parametrize("r", [16, 24, 40, 128])
@pytest.mark.parametrize("tokens", [1, 3])
def test_few_tokens(tokens, r, steps):
    """The gradients of an expert that saw one or three tokens."""
    from smel.lora import orthogonalize
    G = outer(tokens, r, 500, r + tokens, (2,))
    assert torch.linalg.matrix_rank(G[0].double(), rtol=1e-5).item() == tokens
    got = orthogonalize(G.to(DEV), steps)
    close(got, G, steps)
    H = G.transpose(1, 2).contiguous()
    close(orthogonalize(H.to(DEV), steps), H, steps)
    assert torch.equal(got, orthogonalize(G.to(DEV), steps))


@pytest.mark.parametrize("steps", [7, 12, 20])
@pytest.mark.parametrize("r", [16, 24, 60, 120])
def test_half_rank(r, steps):
    """Of whole numbers, exactly of rank r / 2: the null directions hold rounding alone, which grows by a a step on either side."""
    from smel.lora import orthogonalize
    g = torch.Generator().manual_seed(r)
    G = torch.randint(-8, 9, (r, r // 2), generator=g).float() @ torch.randint(-8, 9, (r // 2, 400), generator=g).float()
    close(orthogonalize(G.to(DEV), steps), G, steps)


@pytest.mark.parametrize("steps", [5, 12, 20, 64])
@pytest.mark.parametrize("r", [16, 24, 60, 120])
def test_equal_rows(r, steps):
    """Equal rows stay equal in every step of the formula, so their differences hold nothing that could grow."""
    from smel.lora import orthogonalize
    G = make((r, 500), "fp32", r, 1.0)
    G[1] = G[0]
    G[r - 1] = G[3]
    y = orthogonalize(G.to(DEV), steps)
    X = G.double() / G.double().norm()
    s = torch.linalg.svdvals(X)
    assert s[r - 3] > 1e-4 and s[r - 2] < 1e-12
    close(y, G, steps, smallest=s[r - 3].item())
    if steps > 12:
        assert torch.equal(y[0], y[1]) and torch.equal(y[3], y[r - 1])


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("steps", [7, 10, 12, 16])
@pytest.mark.parametrize("shape", [(3, 16, 300), (40, 301), (2, 333, 100), (29, 25)])
def test_sixteen_bits(shape, steps, dt):
    """Rank 3, in whole numbers that the type holds: the results carry their own rounding alone."""
    from smel.lora import orthogonalize
    g = torch.Generator().manual_seed(steps)
    *lead, m, n = shape
    G = (torch.randint(-4, 5, (*lead, m, 3), generator=g).float() @ torch.randint(-4, 5, (*lead, 3, n), generator=g).float()).to(DT[dt])
    assert torch.equal(G.float(), G.float().round()) and G.abs().max() <= 48
    close(orthogonalize(G.to(DEV), steps), G, steps)


@pytest.mark.parametrize("coeffs", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5), (0.5, 0.25, 0.0)])
@pytest.mark.parametrize("steps", [13, 14, 21, 41, 64])
@pytest.mark.parametrize("r", [6, 30, 64, 128])
def test_coefficients(r, steps, coeffs):
    from smel.lora import orthogonalize
    G = make((r, 200), "fp32", r, 1.5)
    close(orthogonalize(G.to(DEV), steps, coeffs), G, steps, coeffs)


@pytest.mark.parametrize("steps", [10, 17])
def test_list_and_views(steps):
    """Mixed shapes, types and ranks, an empty one, more jobs than a launch takes, strided and expanded inputs: each as alone."""
    from smel.lora import orthogonalize
    shapes = [(4, 16, 256), (64, 16), (3, 40, 90), (2, 100, 300), (0, 16, 64), (1, 1), (129, 20), (5, 1)]
    ts = [make(s, ("fp32", "bf16", "fp16")[i % 3], i, 1.0) if 0 not in s else torch.zeros(s) for i, s in enumerate(shapes * 14)]
    out = orthogonalize([t.to(DEV) for t in ts], steps)
    for i, (t, y) in enumerate(zip(ts, out)):
        assert y.shape == t.shape and y.dtype == t.dtype
        if t.numel() and i < 24:
            close(y, t, steps, what=str(i))
        assert torch.equal(y, orthogonalize(t.to(DEV), steps))
    base = make((4, 48, 400), "fp32", 5)
    b = base.to(DEV)
    for name, view in {"transposed": lambda t: t.transpose(1, 2), "columns": lambda t: t[:, :, 3:203], "rows": lambda t: t[:, ::3],
                       "columns apart": lambda t: t[:, :, ::2], "batch apart": lambda t: t[::2], "one row": lambda t: t[:, 7:8, ::3],
                       "one column": lambda t: t[:, :, 11:12], "4d slice": lambda t: t.view(2, 2, 48, 400)[:, 1:]}.items():
        v = view(b)
        close(orthogonalize(v, steps), v, steps, what=name)
    assert torch.equal(b.cpu(), base)
    same = orthogonalize(b[:1].expand(3, 48, 400), steps)
    assert torch.equal(same[0], same[2])


@pytest.mark.parametrize("steps", [9, 30])
def test_special_values(steps):
    """A zero matrix and zero rows stay zero; NaN or inf spoils its own matrix alone."""
    from smel.lora import orthogonalize
    for r in (16, 28, 50, 90):
        G = make((5, r, 300), "fp32", r, 1.0)
        G[1] = 0
        G[2, 3, 299] = float("nan")
        G[3, 0, 0] = float("inf")
        G[4, 5] = 0
        y = orthogonalize(G.to(DEV), steps).cpu()
        assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and not y[4, 5].any()
        close(y[0], G[0], steps)
        s = torch.linalg.svdvals(G[4].double() / G[4].double().norm())
        close(y[4], G[4], steps, smallest=s[-2].item())


@pytest.mark.parametrize("steps", [11, 15])
def test_graph_and_streams(steps):
    from smel.lora import orthogonalize
    a = [make(s, "fp32", i, 1.0).to(DEV) for i, s in enumerate([(6, 16, 512), (40, 300), (2, 128, 200)])]
    b = [t * 0.5 + 1e-3 for t in a]
    ref, ref2 = [t.clone() for t in orthogonalize(a, steps)], [t.clone() for t in orthogonalize(b, steps)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(a, steps)
    for _ in range(3):
        for t in out:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, ref))
        assert all(torch.equal(x, y) for x, y in zip(orthogonalize(b, steps), ref2))
    with torch.cuda.stream(side):
        two = orthogonalize(b, steps)
    one = orthogonalize(a, steps)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(one, ref)) and all(torch.equal(x, y) for x, y in zip(two, ref2))


@pytest.mark.parametrize("steps", [5, 9, 14])
def test_far_offsets(steps):
    """Strides and sizes that pass 2^31 elements. Columns repeated 2^18 times, whose results are those of one copy over 2^9."""
    from smel.lora import orthogonalize
    big = torch.zeros(1100 << 21, dtype=torch.bfloat16, device=DEV)
    G = make((3, 16, 700), "bf16", 4).to(DEV)
    far = big.as_strided((3, 16, 700), (1 << 30, 1 << 21, 1))
    far.copy_(G)
    assert torch.equal(orthogonalize(far, steps), orthogonalize(G, steps))
    H = make((16, 1000), "bf16", 5).to(DEV)
    lines = big.as_strided((16, 1000), (1, 1 << 21))
    lines.copy_(H)
    assert torch.equal(orthogonalize(lines, steps), orthogonalize(H, steps))
    del big, far, lines
    one = make((32, 260), "bf16", 6, 1.0)
    y = orthogonalize(one.to(DEV).repeat(1, 1 << 18), steps, eps=0.0)
    assert y.numel() > 1 << 31
    for part in (y[:, :260], y[:, 260 * 131072:260 * 131073], y[:, -260:]):
        assert torch.equal(part, y[:, :260])
        close(part.contiguous() * 512, one, steps, eps=0.0)
