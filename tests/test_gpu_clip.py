"""The global gradient norm and clipping by it (smel.lora.grad_norm, clip_grads, clip_grads_ over include/smel_clip.h) against the
definition in 64 bits.

Tolerances (u = 2^-24): squares are summed in 64 bits (terms off by 2^-53 of themselves, adding many of them by far less than u), so the
norm is off by its rounding to fp32, u; the factor by its own, u; a scaled value by 2 u of itself before its one rounding to the
tensor's type (half of its step, fp16 also half of the smallest one)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts if t is not None))


def check(ts, out, norm, most, kind=2.0, eps=1e-6):
    n = norm64(ts) if kind == 2.0 else max((float(t.double().abs().max()) for t in ts if t is not None and t.numel()), default=0.0)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - n) <= 1.01 * U * n
    c = min(1.0, most / (n + eps))
    for t, o in zip(ts, out):
        if t is None:
            assert o is None
            continue
        assert o.shape == t.shape and o.dtype == t.dtype and not o.requires_grad
        ref = t.double().cpu() * c
        tol = (torch.finfo(t.dtype).eps / 2 * (1 + 2 ** -8) + 3 * U) * ref.abs() + TINY[t.dtype]
        assert ((o.double().cpu() - ref).abs() <= tol).all()
        if c == 1.0:
            assert torch.equal(o, t)


def tensors(sizes, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(*s, generator=g)).to(dt).to(DEV) for s in sizes]


SIZES = [[(1,)], [(3, 5)], [(7,), (8,), (9,), (0,), (1, 1)], [(8191,), (8192,), (8193,), (16385,)], [(12, 16, 2048), (12, 512, 16), (16, 512), (2048, 16)],
         [(k % 37 + 1, 3) for k in range(300)], [(2, 0)], [(1 << 20,), (5,), (333, 777)]]


@pytest.mark.parametrize("most", [1.0, 1e-3, 1e9, 0.0, math.inf])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("which", range(len(SIZES)))
def test_clip(which, dt, most):
    from smel.lora import clip_grads, clip_grads_, grad_norm
    ts = tensors(SIZES[which], DT[dt], which)
    before = [t.clone() for t in ts]
    out, norm = clip_grads(ts, most)
    check(ts, out, norm, most)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    assert torch.equal(grad_norm(ts), norm)
    assert torch.equal(clip_grads_(ts, most), norm)
    assert all(torch.equal(a, b) for a, b in zip(ts, out))
    check(before, *clip_grads(before, most / 8 if most < math.inf else most, math.inf), most / 8 if most < math.inf else most, math.inf)


def test_mixed_types_and_none():
    from smel.lora import clip_grads
    ts = [t for dt in DT.values() for t in tensors([(50, 33), (1,), (4096,)], dt, 3)]
    ts[1:1] = [None, None]
    check(ts, *clip_grads(ts, 2.0), 2.0)
    single, norm = clip_grads(ts[0], 2.0)
    assert isinstance(single, torch.Tensor)
    check(ts[:1], [single], norm, 2.0)
    assert clip_grads((t for t in ts), 2.0)[1] == clip_grads(ts, 2.0)[1]


def test_nothing():
    from smel.lora import clip_grads, clip_grads_, grad_norm
    assert clip_grads([], 1.0)[0] == [] and float(grad_norm([])) == 0 and float(clip_grads_([None], 1.0)) == 0
    z = torch.zeros(100, device=DEV)
    out, norm = clip_grads([z, z[:0]], 1.0)
    assert float(norm) == 0 and not out[0].any()
    assert float(grad_norm([z[:0]])) == 0


def test_large_and_small_values():
    """Squares beyond and below fp32's range: the norm is right as long as it is an fp32 number itself."""
    from smel.lora import clip_grads, grad_norm
    for v in (1e30, 3e-42, 1e-30, 2.0 ** 100):
        ts = [torch.full((1000,), v, device=DEV), torch.full((24,), -v, device=DEV)]
        assert abs(float(grad_norm(ts)) - 32 * float(ts[0][0])) <= max(1.01 * U * 32 * v, 2.0 ** -149)
        check(ts, *clip_grads(ts, 1.0), 1.0)
    big = torch.full((64,), 3e38, device=DEV)
    out, norm = clip_grads([big], 1.0)      # the norm is no fp32 number, the factor is
    assert math.isinf(float(norm)) and abs(float(out[0][0]) - 0.125) < 1e-6
    assert float(grad_norm([big], math.inf)) == float(big[0])


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_not_finite(kind):
    """NaN spoils the norm and every value, an infinity the norm: finite values go to 0, as the product says."""
    from smel.lora import clip_grads
    for at in (0, 77, 9000, 19999):
        a, b = tensors([(20000,), (50,)], torch.float32, 1)
        a[at] = float("nan")
        out, norm = clip_grads([b, a], 1.0, kind)
        assert math.isnan(float(norm)) and all(torch.isnan(o).all() for o in out)
        a[at] = -math.inf
        out, norm = clip_grads([b, a], 1.0, kind)
        assert math.isinf(float(norm)) and not out[0].any() and torch.isnan(out[1][at]) and torch.isnan(out[1]).sum() == 1
        a[(at + 5) % 20000] = float("nan")
        assert math.isnan(float(clip_grads([b, a], 1.0, kind)[1]))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_views(dt):
    """Odd offsets, transposed and permuted tensors (dense: taken as they lie), strided and expanded ones (through a copy)."""
    from smel.lora import clip_grads, clip_grads_
    base = tensors([(60, 301)], DT[dt], 5)[0]
    views = {"odd": lambda t: t.view(-1)[3:9004], "transposed": lambda t: t.t(), "permuted": lambda t: t[:, :300].reshape(60, 30, 10).permute(2, 0, 1),
             "slice": lambda t: t[:, 7:100], "rows": lambda t: t[::2], "steps": lambda t: t.view(-1)[::3], "negative": lambda t: t[5:6, 9:10]}
    for name, view in views.items():
        x = view(base.clone())
        out, norm = clip_grads([x, base], 3.0)
        check([x, base], out, norm, 3.0)
        own = base.clone()
        x, want = view(own), view(base.clone())
        rest = own.clone()
        assert torch.equal(clip_grads_([x, base.clone()], 3.0), norm)
        assert torch.equal(x, out[0]), name
        view(rest).zero_()
        if name not in ("transposed", "permuted"):      # nothing beside the view was written
            view(own).zero_()
            assert torch.equal(own, rest), name
    wide = base[:1].expand(5, 301)
    check([wide], *clip_grads([wide], 1.0), 1.0)


def test_in_place_is_seen_by_autograd():
    from smel.lora import clip_grads_
    p = torch.ones(10, device=DEV, requires_grad=True)
    x = p * 2
    y = x * x
    clip_grads_([x], 1.0)
    with pytest.raises(RuntimeError):      # x was saved before it was changed
        y.sum().backward()
    (p * 3).sum().backward()
    assert float(clip_grads_([p.grad], 0.5)) == pytest.approx(math.sqrt(90), rel=1e-6)
    assert torch.allclose(p.grad.norm(), torch.tensor(0.5, device=DEV))


def test_many_tensors_and_order():
    """More tensors than a launch takes; the same bits on every call, and as one launch's where the chunks are the same."""
    from smel.lora import clip_grads
    ts = tensors([(5000 + k,) for k in range(500)], torch.bfloat16, 2, 0.01)
    out, norm = clip_grads(ts, 1.0)
    check(ts, out, norm, 1.0)
    for _ in range(3):
        again, n2 = clip_grads(ts, 1.0)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, again))


def test_far_offsets():
    """A tensor past 2^31 values."""
    from smel.lora import clip_grads, clip_grads_
    n = (1 << 31) + 12345
    x = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    some = tensors([(9000,)], torch.bfloat16, 1)[0]
    x[:9000] = x[-9000:] = some
    out, norm = clip_grads([x], 1.0)
    ref = math.sqrt(2) * norm64([some])
    assert abs(float(norm) - ref) <= 1.01 * U * ref
    want, _ = clip_grads([some, some.clone()], 1.0)
    assert torch.equal(out[0][:9000], want[0]) and torch.equal(out[0][-9000:], want[0]) and not out[0][9000:9100].any()
    del out
    clip_grads_([x], 1.0)
    assert torch.equal(x[:9000], want[0]) and torch.equal(x[-9000:], want[0]) and not x[-9100:-9000].any()


def test_graph_and_streams():
    from smel.lora import clip_grads, clip_grads_
    ts = tensors([(300, 700), (17,), (9000,)], torch.float32, 4)
    src = [t.clone() for t in ts]
    ref, rn = clip_grads(ts, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grads(ts, 1.0)
        clip_grads_([t.clone() for t in ts], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph, inplace = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = clip_grads(ts, 1.0)
    with torch.cuda.graph(inplace):
        n2 = clip_grads_(ts, 1.0)
    for k in range(3):
        for t, s in zip(ts, src):
            t.copy_(s * (k + 1))
        for t in out:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want, wn = clip_grads([s * (k + 1) for s in src], 1.0)
        assert torch.equal(norm, wn) and all(torch.equal(a, b) for a, b in zip(out, want))
        inplace.replay()
        torch.cuda.synchronize()
        assert torch.equal(n2, wn) and all(torch.equal(a, b) for a, b in zip(ts, want))
    s2 = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s2):
            two, m2 = clip_grads(src[::-1], 0.5)
        one, m1 = clip_grads(src, 1.0)
        torch.cuda.synchronize()
        assert torch.equal(m1, rn) and all(torch.equal(a, b) for a, b in zip(one, ref))
        check(src[::-1], two, m2, 0.5)


def test_refusals():
    from smel._lib import SmelError
    from smel.lora import clip_grads, clip_grads_, grad_norm
    x = torch.ones(100, device=DEV)
    for bad in (lambda: clip_grads([x.double()], 1.0), lambda: clip_grads([x.long()], 1.0), lambda: clip_grads([x.cpu()], 1.0),
                lambda: clip_grads([x, x.cpu()], 1.0), lambda: clip_grads([x], -1.0), lambda: clip_grads([x], float("nan")),
                lambda: clip_grads([x], 1.0, 3.0), lambda: clip_grads([x], 1.0, eps=-1.0), lambda: grad_norm([x], 0.5),
                lambda: clip_grads_([x.to_sparse()], 1.0)):
        with pytest.raises(ValueError):
            bad()
    # the same memory twice: read it as often as you like, but write it once
    assert float(grad_norm([x, x, x[:0]])) == pytest.approx(math.sqrt(200))
    out, norm = clip_grads([x, x], 1.0)
    assert torch.equal(out[0], out[1])
    for bad in (lambda: clip_grads_([x, x], 1.0), lambda: clip_grads_([x[:60], x[59:]], 1.0), lambda: clip_grads_([x, x[10:20]], 1.0)):
        with pytest.raises(SmelError, match="overlap"):
            bad()
    with pytest.raises(ValueError, match="overlaps itself"):
        clip_grads_([x, torch.ones(1, 5, device=DEV).expand(7, 5)], 1.0)
    assert torch.equal(x, torch.ones(100, device=DEV))
    clip_grads_([x[:60], x[60:]], 1.0)


def test_parts_of_many_launches():
    """More parts than every block of the scaling adds up itself (8192): they go through a launch of their own."""
    from smel.lora import clip_grads, grad_norm
    g = torch.Generator(device=DEV).manual_seed(3)
    flat = 1e-3 * torch.randn(600, 140001, generator=g, device=DEV).bfloat16()
    ts = list(flat.unbind(0))
    n = float(torch.sqrt(flat.double().square().sum()))
    for kind, want in ((2.0, n), (math.inf, float(flat.abs().max()))):
        out, norm = clip_grads(ts, want / 4, kind)
        assert abs(float(norm) - want) <= 1.01 * U * want and torch.equal(norm, grad_norm(ts, kind))
        c = (want / 4) / (want + 1e-6)
        ref = flat.double() * c
        tol = (2.0 ** -8 * (1 + 2 ** -8) + 3 * U) * ref.abs() + TINY[torch.bfloat16]
        assert ((torch.stack(out).double() - ref).abs() <= tol).all()


def test_scalars_and_parameters():
    """0-dimensional tensors, parameters (the results carry no gradient), and gradients that are neighbours in one buffer."""
    from smel.lora import clip_grads, clip_grads_
    ts = [torch.tensor(3.0, device=DEV), torch.nn.Parameter(torch.full((4,), 2.0, device=DEV))]
    out, norm = clip_grads(ts, 1.0)
    check([t.detach() for t in ts], out, norm, 1.0)
    assert out[0].shape == () and not isinstance(out[1], torch.nn.Parameter)
    flat = torch.arange(1.0, 1001.0, device=DEV)
    want, n1 = clip_grads([flat], 5.0)
    assert torch.equal(clip_grads_(list(flat.split([1, 7, 500, 492])), 5.0), n1)
    assert torch.equal(flat, want[0])
