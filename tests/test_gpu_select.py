"""The choice of experts by scores, bias and groups (smel.moe.select_experts, route_grouped over include/smel_moe.h) against the
definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, s = eps(dtype) / 2): a sigmoid is an exponential, a sum and a quotient, off by at most
10 u of itself; a softmax score by (24 + 2 r) u, r the row's range of logits (the argument z - m is rounded, and so is its product
with log2 e). The sum of 16 positive scores adds 16 u, quotient and scale 4 u. Gradients: each ds_k is off by 64 (1 + r / 8) u of the size
of its terms, the products behind it by as much again; then one rounding to the logits' type (fp16: half its smallest step).
Ids are compared where the choices lie apart by more than 1e-5 (|c| + the row's largest score), three times what two scores' errors
make, or are exactly equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def scores64(z, score):
    z = z.double()
    if score == "sigmoid":
        return torch.sigmoid(z)
    dead = torch.isneginf(z).all(1, keepdim=True)
    return torch.softmax(torch.where(dead, 0.0, z), 1) * ~dead


def picks64(s, bias, K, groups=1, top_groups=1, best=2):
    """(ids, whether the choice hangs on no rounding) of the scores s in 64 bits."""
    T, E = s.shape
    c = s if bias is None else s + bias.double()
    most = s.amax(1, keepdim=True)
    apart = lambda hi, lo: (hi == lo) | (hi - lo > 1e-5 * (hi.abs() + (most if hi.dim() == 2 else most[:, 0])))  # noqa: E731
    ok = torch.ones(T, dtype=torch.bool)
    if top_groups < groups:
        cg = c.view(T, groups, -1)
        v = cg.sort(dim=2, descending=True).values[:, :, :best].sum(2)
        order = v.sort(dim=1, descending=True, stable=True)
        ok &= apart(order.values[:, top_groups - 1], order.values[:, top_groups])
        keep = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, order.indices[:, :top_groups], True)
        c = torch.where(keep[:, :, None], cg, float("nan")).view(T, E)
    order = torch.where(c.isnan(), -math.inf, c).sort(dim=1, descending=True, stable=True)
    ids = order.indices[:, :K]
    top = order.values[:, :K + 1]
    ok &= apart(top[:, :-1], top[:, 1:]).all(1)
    return ids, ok


def close(got, ref, tol, what):
    g = got.detach().cpu().double()
    assert g.shape == ref.shape, what
    bad = ~((g - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {((g - ref).abs() / tol).max()}"


def formula(z, topi, d, score, renorm, scale):
    """topv, dz in 64 bits for these picks, and their bounds."""
    s = scores64(z, score)
    sk = s.gather(1, topi)
    S = sk.sum(1, keepdim=True) + 1e-20 if renorm else torch.ones(z.shape[0], 1, dtype=torch.float64)
    zd = z.double()
    live = torch.where(torch.isneginf(zd), math.inf, zd).amin(1, keepdim=True)
    r = torch.zeros(1, 1, dtype=torch.float64) if score == "sigmoid" else (zd.amax(1, keepdim=True) - live).clamp(0, 1e3)
    topv = scale * sk / S
    es = (10 if score == "sigmoid" else 24 + 2 * r) * U
    out = {"topv": (topv, topv * (2 * es + 24 * U) + 2.0 ** -126)}
    if d is None:
        return out
    d = d.double()
    ds, size = scale * d, scale * d.abs()
    if renorm:
        dot = (d * sk).sum(1, keepdim=True) / S
        ds, size = scale * (d - dot) / S, scale * (d.abs() + (d.abs() * sk).sum(1, keepdim=True) / S) / S
    es = 64 * (1 + r / 8) * U
    if score == "sigmoid":
        slope = torch.exp(-zd.abs()) / (1 + torch.exp(-zd.abs())) ** 2
        at = slope.gather(1, topi)
        dz = torch.zeros_like(s).scatter(1, topi, ds * at)
        tol = torch.zeros_like(s).scatter(1, topi, 2 * es * size * at)
    else:
        dot, dsize = (ds * sk).sum(1, keepdim=True), (size * sk).sum(1, keepdim=True)
        dz = s * (torch.zeros_like(s).scatter(1, topi, ds) - dot)
        tol = 2 * es * s * (torch.zeros_like(s).scatter(1, topi, size) + dsize)
    out["dz"] = dz, tol + half(z.dtype) * (1 + 2 ** -8) * dz.abs() + TINY[z.dtype]
    return out


def logits_of(T, E, dt, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)).to(dt), 0.1 * torch.randn(E, generator=g), \
        torch.randn(T, 16, generator=g)


def run(z, bias, d, K, **kw):
    from smel.moe import select_experts
    zg = z.to(DEV).requires_grad_(True)
    topv, topi, *rest = select_experts(zg, K, bias=None if bias is None else bias.to(DEV), **kw)
    dz, = torch.autograd.grad(topv, zg, d.to(DEV))
    return topv, topi, dz, *rest


SHAPES = [  # T, E, K, groups, kept
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (3, 2, 1, 2, 1), (5, 7, 3, 1, 1), (23, 64, 4, 1, 1), (70, 96, 6, 3, 2), (33, 100, 5, 4, 2),
    (129, 128, 8, 1, 1), (40, 160, 8, 8, 3), (517, 256, 8, 8, 4), (66, 256, 16, 1, 1), (31, 300, 9, 12, 5), (20, 511, 16, 1, 1),
    (57, 512, 10, 16, 4), (19, 495, 7, 33, 9), (9, 64, 5, 64, 20), (17, 510, 3, 2, 1), (14, 512, 16, 64, 2), (301, 63, 2, 9, 9),
    (1, 512, 16, 1, 1), (2050, 24, 2, 2, 1),
    (4096, 64, 6, 1, 1), (4097, 64, 16, 8, 3), (4098, 37, 3, 1, 1), (4099, 128, 8, 1, 1), (5003, 100, 9, 4, 3), (4100, 120, 7, 15, 5),
    (4111, 16, 4, 16, 9), (4103, 34, 2, 17, 3), (4102, 102, 16, 17, 7), (4101, 2, 1, 1, 1)]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,E,K,groups,kept", SHAPES)
def test_select(T, E, K, groups, kept, dt, score):
    for with_bias, renorm, best in ((True, True, 2), (False, False, 1)):
        z, bias, d = logits_of(T, E, DT[dt], T * 7 + E + K)
        bias = bias if with_bias else None
        topv, topi, dz, s = run(z, bias, d[:, :K], K, score=score, groups=groups, top_groups=kept, group_best=best, renorm=renorm,
                                scale=2.5, with_scores=True)
        assert topv.dtype == torch.float32 and topi.dtype == torch.int64 and dz.dtype == z.dtype
        s64 = scores64(z, score)
        r = 0 if score == "sigmoid" else (z.double().amax(1, keepdim=True) - z.double().amin(1, keepdim=True))
        close(s, s64, s64 * ((10 if score == "sigmoid" else 24 + 2 * r) * U) + 2.0 ** -126, "scores")
        ids, ok = picks64(s64, bias, K, groups, kept, best)
        assert ok.sum() >= 0.6 * T or T < 5
        assert torch.equal(topi.cpu()[ok], ids[ok])
        want = formula(z, topi.cpu(), d[:, :K], score, renorm, 2.5)
        close(topv, *want["topv"], "topv")
        close(dz, *want["dz"], "dz")
        again = run(z, bias, d[:, :K], K, score=score, groups=groups, top_groups=kept, group_best=best, renorm=renorm, scale=2.5)
        assert all(torch.equal(a, b) for a, b in zip((topv, topi, dz), again))


def test_select_without_gradient_same_bits():
    from smel.moe import select_experts
    z, bias, d = logits_of(64, 256, torch.bfloat16, 3)
    topv, topi, _ = run(z, bias, d[:, :8], 8, groups=8, top_groups=4)
    a, b = select_experts(z.to(DEV), 8, bias=bias.to(DEV), groups=8, top_groups=4)
    assert torch.equal(a, topv) and torch.equal(b, topi) and not a.requires_grad


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_index(score):
    from smel.moe import select_experts
    z = torch.zeros(3, 40)
    z[1, 7::5] = 1.0
    z[2] = torch.arange(40).div(4, rounding_mode="floor").float().flip(0)
    topi = select_experts(z.to(DEV), 9, score=score)[1].cpu()
    for t in range(3):
        assert topi[t].tolist() == z[t].sort(dim=0, descending=True, stable=True).indices[:9].tolist()
    # equal groups: the first ones stay
    topi = select_experts(z[:1].to(DEV), 6, score=score, groups=10, top_groups=2)[1].cpu()
    assert topi[0].tolist() == [0, 1, 2, 3, 4, 5]
    # -0 and +0 are one choice
    zero = torch.zeros(1, 8, device=DEV)
    assert select_experts(zero, 3, bias=torch.tensor([-0.5, -0.5, -0.5, 0, -0.0, 0, 0, 0], device=DEV))[1].tolist() == [[3, 4, 5]]


def test_groups_count_with_their_best():
    """One strong expert alone wins a group with group_best 1, two middling ones with 2; the bias steers groups too."""
    from smel.moe import select_experts
    z = torch.full((1, 8), -4.0)
    z[0, 1], z[0, 4], z[0, 5] = 2.0, 1.0, 1.0
    kw = dict(groups=2, top_groups=1)
    assert select_experts(z.to(DEV), 2, group_best=1, **kw)[1].tolist() == [[1, 0]]
    assert select_experts(z.to(DEV), 2, group_best=2, **kw)[1].tolist() == [[4, 5]]
    bias = torch.zeros(8, device=DEV)
    bias[2] = 5.0
    topv, topi = select_experts(z.to(DEV), 2, bias=bias, **kw)
    assert topi.tolist() == [[2, 1]]
    s = torch.sigmoid(torch.tensor([-4.0, 2.0], dtype=torch.float64))
    close(topv[0], s / s.sum(), 64 * U * torch.ones(2), "topv without the bias")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_rows_of_anything(score, groups, kept):
    """NaN, infinities, the type's lowest value, whole rows switched off: ids stay K different ones of [0, E), other rows are as alone,
    and a row without a score has weight 0 and a zero gradient."""
    for dt in DT.values():
        z, _, d = logits_of(12, 64, dt, 5)
        clean = z.clone()
        lowest = torch.finfo(dt).min
        z[1] = float("nan")
        z[2, ::3] = float("nan")
        z[3] = -math.inf
        z[4, 5:] = -math.inf
        z[5, 9] = math.inf
        z[6] = lowest
        z[7, 3:] = lowest
        z[8, 20] = torch.finfo(dt).max
        topv, topi, dz, s = run(z, None, d[:, :8], 8, score=score, groups=groups, top_groups=kept, with_scores=True)
        ids = topi.cpu().sort(1).values
        assert ((ids >= 0) & (ids < 64)).all() and (ids[:, 1:] > ids[:, :-1]).all()
        one = run(clean, None, d[:, :8], 8, score=score, groups=groups, top_groups=kept, with_scores=True)
        same = [0, 9, 10, 11]
        assert all(torch.equal(a[same], b[same]) for a, b in zip((topv, topi, dz, s), one))
        for t in (3,):      # nothing left
            assert not topv[t].any() and not s[t].any() and not dz[t].any()
        off = [4, 6, 7]
        want = formula(z[off], topi.cpu()[off], d[off, :8], score, True, 1.0)
        close(topv[off], *want["topv"], "topv")
        close(dz[off], *want["dz"], "dz")
        if groups == 1:
            assert topi[4, :5].sort().values.tolist() == [0, 1, 2, 3, 4] and topi[8, 0] == 20
            assert topi[5, 0] == 9 or score == "softmax"      # whose row is NaN then
            assert topi[4, 5:].tolist() == [5, 6, 7] and not topv[4, 5:].any()
        dead = torch.full((64,), -math.inf)
        dead[40:] = 0       # a bias that leaves 24 experts
        _, topi, _ = run(clean, dead, d[:, :8], 8, score=score)
        assert (topi >= 40).all()
        dead[44:] = -math.inf     # and four, fewer than K: those first, then the lowest others
        _, topi, _ = run(clean, dead, d[:, :8], 8, score=score)
        assert (topi[:, :4].sort(1).values.cpu() == torch.arange(40, 44)).all() and (topi[:, 4:].cpu() == torch.arange(4)).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_views(dt):
    """Column slices at odd offsets, rows far apart, transposed and expanded logits, a strided gradient, a bias of other types."""
    from smel.moe import select_experts
    g = torch.Generator().manual_seed(4)
    base = torch.randn(200, 301, generator=g).to(DT[dt])
    bd = base.to(DEV)
    views = {"slice": lambda t: t[:90, 3:103], "rows": lambda t: t[::3, 101:201], "transposed": lambda t: t[:100, :60].t(),
             "expanded": lambda t: t[:1, :100].expand(6, 100)}
    bias = torch.randn(200, generator=g).bfloat16()
    for name, view in views.items():
        z = view(base)
        d = torch.randn(z.shape[0], 12, generator=g)
        zg = view(bd).detach().requires_grad_(True)
        topv, topi = select_experts(zg, 6, bias=bias.to(DEV)[::2], groups=5, top_groups=2)
        dz, = torch.autograd.grad(topv, zg, d.to(DEV)[:, ::2])
        a, b, c = run(z.contiguous(), bias[::2].float(), d[:, ::2].contiguous(), 6, groups=5, top_groups=2)
        assert torch.equal(topv, a) and torch.equal(topi, b) and torch.equal(dz, c), name


def test_empty_and_one():
    from smel.moe import select_experts
    z = torch.empty(0, 32, device=DEV, requires_grad=True)
    topv, topi, s = select_experts(z, 4, with_scores=True)
    assert topv.shape == topi.shape == (0, 4) and s.shape == (0, 32)
    assert torch.autograd.grad(topv, z, torch.empty(0, 4, device=DEV))[0].shape == (0, 32)


def test_against_differences():
    """dz against the difference quotient of the kernel's own topv at fixed picks. The quotient is off by its own error (measured in
    64 bits) and by the two values' rounding over the step."""
    from smel.moe import select_experts
    step = 2.0 ** -8
    for score in ("sigmoid", "softmax"):
        for renorm in (True, False):
            z, _, d = logits_of(400, 48, torch.float32, 9)
            order = scores64(z, score).sort(dim=1, descending=True).values
            z = z[(order[:, 5] - order[:, 6]) > 0.06 * order[:, 5]]      # the picks stay over the steps
            n = z.shape[0]
            assert n >= 4
            d = d[:n, :6]
            g = torch.Generator().manual_seed(2)
            v = torch.randn(n, 48, generator=g)
            kw = dict(score=score, renorm=renorm)
            topv, topi, dz = run(z, None, d, 6, **kw)

            def at(k, f64):
                zz = z + k * step * v
                if f64:
                    return (formula(zz, topi.cpu(), None, score, renorm, 1.0)["topv"][0] * d.double()).sum(1)
                a, b = select_experts(zz.to(DEV), 6, **kw)
                ours = torch.zeros(n, 48, dtype=torch.float64).scatter(1, b.cpu(), a.cpu().double())
                assert (b.cpu().sort(1).values == topi.cpu().sort(1).values).all()
                return (ours.gather(1, topi.cpu()) * d.double()).sum(1)
            quotient = (at(1, False) - at(-1, False)) / (2 * step)
            ref = (formula(z, topi.cpu(), d, score, renorm, 1.0)["dz"][0] * v.double()).sum(1)
            own = ((at(1, True) - at(-1, True)) / (2 * step) - ref).abs()
            rounding = 100 * U * (topv.cpu().double() * d.double().abs()).sum(1) / step
            got = (dz.cpu().double() * v.double()).sum(1)
            assert ((quotient - got).abs() <= own + rounding + 1e-6).all()


def test_graph_and_streams():
    from smel.moe import select_experts
    z, bias, d = (t.to(DEV) for t in logits_of(300, 256, torch.bfloat16, 6))

    def step(z=z, score="sigmoid"):
        zg = z.detach().requires_grad_(True)
        topv, topi, s = select_experts(zg, 8, score=score, bias=bias, groups=8, top_groups=4, with_scores=True)
        return [topv, topi, s, torch.autograd.grad(topv, zg, d[:, :8])[0]]
    for score in ("sigmoid", "softmax"):
        ref = [t.clone() for t in step(score=score)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(score=score)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(score=score)
        for _ in range(3):
            for t in out:
                t.detach().fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, ref))
            assert all(torch.equal(a, c) for a, c in zip(step(score=score), ref))
    other = step(z=z.flip(0))
    torch.cuda.synchronize()
    s2 = torch.cuda.Stream()
    one = step()
    for _ in range(3):
        with torch.cuda.stream(s2):
            two = step(z=z.flip(0))
        now = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(now, one)) and all(torch.equal(a, c) for a, c in zip(two, other))


def test_refusals():
    from smel.moe import select_experts
    z, b = torch.zeros(4, 32, device=DEV), torch.zeros(32, device=DEV)
    for bad in (lambda: select_experts(z.double(), 2), lambda: select_experts(z[0], 2), lambda: select_experts(z, 2, score="relu"),
                lambda: select_experts(z, 2, bias=b[:8]), lambda: select_experts(z, 2, bias=b.long()), lambda: select_experts(z, 2, bias=b.cpu()),
                lambda: select_experts(z, 2, groups=5), lambda: select_experts(z, 2, groups=4, top_groups=5), lambda: select_experts(z, 0),
                lambda: select_experts(z, 9, groups=4, top_groups=1), lambda: select_experts(z, 33), lambda: select_experts(z, 2, groups=0),
                lambda: select_experts(z, 2, group_best=3), lambda: select_experts(z.cpu(), 2)):
        with pytest.raises(ValueError):
            bad()
    from smel._lib import SmelError
    for bad in (lambda: select_experts(torch.zeros(2, 513, device=DEV), 2), lambda: select_experts(z, 17),
                lambda: select_experts(torch.zeros(2, 130, device=DEV), 2, groups=65, top_groups=2)):
        with pytest.raises(SmelError):
            bad()
    zg = z.clone().requires_grad_(True)
    topv, _ = select_experts(zg, 2)
    gz, = torch.autograd.grad(topv, zg, torch.ones_like(topv).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):      # once differentiable
        gz.sum().backward()
    topv, topi = select_experts(zg, 2)
    topi.add_(1)
    with pytest.raises(RuntimeError):      # picks changed in place before the backward
        topv.sum().backward()


def test_saved_tensors_moved_and_transforms():
    import torch.autograd.forward_ad as fw
    from smel.moe import select_experts
    z, bias, d = (t.to(DEV) for t in logits_of(30, 64, torch.bfloat16, 8))
    base = torch.cat((z, z), 1)
    for zz in (z, base[:, 5:69]):
        for score in ("sigmoid", "softmax"):
            zg = zz.detach().requires_grad_(True)
            ref, = torch.autograd.grad(select_experts(zg, 4, score, bias)[0], zg, d[:, :4])
            with torch.autograd.graph.save_on_cpu():
                topv, _ = select_experts(zg, 4, score, bias)
            assert torch.equal(ref, torch.autograd.grad(topv, zg, d[:, :4])[0])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: select_experts(t, 4)[0].sum())(z)
    with fw.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                select_experts(fw.make_dual(z, torch.ones_like(z)), 4)


def test_far_offsets():
    """Logits past 2^31 elements, packed and with rows far apart: the same bits as alone."""
    T, E = (1 << 25) - 5, 72
    z, bias, d = (t.to(DEV) for t in logits_of(100, E, torch.bfloat16, 12))
    few = run(z, bias, d[:, :2], 2, groups=4, top_groups=2)
    from smel.moe import select_experts
    big = torch.zeros(T, E, dtype=torch.bfloat16, device=DEV)
    big[:100] = big[-100:] = z
    dt = torch.zeros(T, 2, device=DEV)
    dt[:100] = dt[-100:] = d[:, :2]
    zg = big.requires_grad_(True)
    topv, topi = select_experts(zg, 2, bias=bias, groups=4, top_groups=2)
    dz, = torch.autograd.grad(topv, zg, dt)
    for at in (slice(0, 100), slice(T - 100, T)):
        assert torch.equal(topv[at], few[0]) and torch.equal(topi[at], few[1]) and torch.equal(dz[at], few[2])
    assert not dz[100:300].any() and not dz[-300:-100].any()
    del big, zg, dz, dt, topv, topi
    far = torch.zeros(100, 1 << 25, dtype=torch.bfloat16, device=DEV)[:, 7:7 + E]
    far.copy_(z)
    zg = far.requires_grad_(True)
    topv, topi = select_experts(zg, 2, bias=bias, groups=4, top_groups=2)
    assert torch.equal(topv, few[0]) and torch.equal(topi, few[1])
    assert torch.equal(torch.autograd.grad(topv, zg, d[:, :2])[0], few[2])


def test_backward_of_foreign_ids():
    """The C entry counts ids outside [0, E) nowhere, and clears the columns between E and the row stride."""
    from smel import _lib as L
    z, _, d = (t.to(DEV) for t in logits_of(6, 30, torch.float32, 1))
    topi = torch.tensor([[0, -1], [29, 30], [5, 1 << 40], [-7, 99], [1, 2], [3, 4]], device=DEV)
    d = d[:, :2].contiguous()
    dz = torch.full((6, 40), 9.0, device=DEV)
    L.call("smel_select_experts_bwd", z.data_ptr(), 30, 2, 6, 30, 2, 0, 0, 1.0, topi.data_ptr(), d.data_ptr(), None, dz.data_ptr(), 40,
           L.stream())
    assert not dz[:, 30:].any()
    ok = (topi >= 0) & (topi < 30)
    s = torch.sigmoid(z.double())
    want = torch.zeros(6, 30, dtype=torch.float64, device=DEV)
    for t in range(6):
        for k in range(2):
            if ok[t, k]:
                want[t, topi[t, k]] += (d.double()[t, k] * s[t, topi[t, k]] * (1 - s[t, topi[t, k]]))
    close(dz[:, :30], want.cpu(), 100 * U * want.abs().cpu() + 1e-30, "dz")


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("H,E", [(256, 64), (128, 40), (72, 24)])
def test_route_grouped(H, E, dt):
    """The router's product with the choice behind it: logits are route's, the choice select_experts' of them, and dx is the
    logits' gradient times the weight (bf16: the gradient's and the products' roundings)."""
    from smel.moe import route, route_grouped, select_experts
    dtype = DT[dt]
    g = torch.Generator().manual_seed(H + E)
    x, w = torch.randn(90, H, generator=g).to(DEV, dtype), (0.2 * torch.randn(E, H, generator=g)).to(DEV, dtype)
    bias, d = 0.1 * torch.randn(E, generator=g).to(DEV), torch.randn(90, 4, generator=g).to(DEV)
    xg = x.clone().requires_grad_(True)
    scores, topv, topi, logits = route_grouped(xg, w, 4, bias=bias, groups=4, top_groups=2, scale=2.0, with_logits=True)
    assert torch.equal(logits.to(dtype), route(x, w, 4, with_logits=True)[3])
    lg = logits.detach().requires_grad_(True)
    a, b, c = select_experts(lg, 4, bias=bias, groups=4, top_groups=2, scale=2.0, with_scores=True)
    assert torch.equal(a, topv) and torch.equal(b, topi) and torch.equal(c, scores)
    dl, = torch.autograd.grad(a, lg, d)
    dx, = torch.autograd.grad(topv, xg, d, retain_graph=True)
    ref = dl.double() @ w.double()
    size = dl.double().abs() @ w.double().abs()
    close(dx, ref.cpu(), ((half(dtype) + E * U) * size + half(dtype) * ref.abs()).cpu() + 1e-12, "dx")
    both, = torch.autograd.grad((topv, logits), xg, (d, dl.to(logits.dtype)))
    close(both, 2 * ref.cpu(), ((4 * half(dtype) + 2 * E * U) * size).cpu() + 1e-12, "dx of both")
    assert len(route_grouped(x, w, 4)) == 3


def test_route_grouped_edges():
    from smel.moe import route_grouped
    x, w = torch.randn(1, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True), torch.randn(16, 64, device=DEV, dtype=torch.bfloat16)
    scores, topv, topi = route_grouped(x, w, 2, score="softmax", groups=4, top_groups=1)
    assert scores.shape == (1, 16) and topi.shape == (1, 2) and torch.autograd.grad(topv.sum() + scores.sum() * 0, x)[0].shape == (1, 64)
    with pytest.raises(ValueError):
        route_grouped(x.cpu(), w, 2)


@pytest.mark.parametrize("E,K", [(16, 1), (64, 1), (128, 3), (256, 8)])
def test_rows_do_not_depend_on_the_batch(E, K):
    """A token's results are the same bits alone and among many (powers of two of experts, whatever lanes a token gets)."""
    z, bias, d = logits_of(4500, E, torch.float32, E)
    for score in ("sigmoid", "softmax"):
        for groups, kept in ((1, 1), (4, 2)):
            many = run(z, bias, d[:, :K], K, score=score, groups=groups, top_groups=kept)
            few = run(z[:70], bias, d[:70, :K], K, score=score, groups=groups, top_groups=kept)
            assert all(torch.equal(a[:70], b) for a, b in zip(many, few))


def test_one_renormalised_pick():
    """K = 1 with renormalised weights: the weight is the scale, its gradient zero but for the rounding of d s / s."""
    for score in ("sigmoid", "softmax"):
        z, bias, d = logits_of(300, 64, torch.float32, 2)
        topv, topi, dz = run(z, bias, d[:, :1], 1, score=score, scale=2.5)
        close(topv, *(t.expand(300, 1) for t in (torch.tensor([[2.5]], dtype=torch.float64), torch.tensor([[8 * U]], dtype=torch.float64))), "topv")
        s = scores64(z, score).gather(1, topi.cpu())
        assert (dz.cpu().double().abs() <= 4 * U * 2.5 * d[:, :1].double().abs() / s * s.clamp(max=1)).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_route_grouped_without_tokens(dt):
    from smel.moe import route_grouped
    x = torch.empty(0, 128, device=DEV, dtype=DT[dt], requires_grad=True)
    w = torch.randn(64, 128, device=DEV).to(DT[dt])
    scores, topv, topi = route_grouped(x, w, 4, groups=4, top_groups=2)
    assert scores.shape == (0, 64) and topv.shape == topi.shape == (0, 4)
    assert torch.autograd.grad(topv, x, torch.empty_like(topv))[0].shape == (0, 128)
