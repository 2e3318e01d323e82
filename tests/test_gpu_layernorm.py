"""Layer norm and the norm after a residual add (smel.norm over include/smel_norm.h) against the formula in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, s = eps(dtype) / 2 the half step of an output's type): a row's sums add at most
64 values one after the other on any path (32 in a thread, six levels of a wave, 16 waves and the tails), so mean and
variance are off by at most 64 u of the mean magnitude, xhat by 64 u (1 + M rstd) (1 + |xhat|) with M the row's largest |x|
(M rstd: what the subtraction of the mean cancels), and what is built from xhat by the same times the size of its terms. The
weights' gradients add up rows / 512 + 40 rows' terms on a path, each off by what xhat is. Every output is then rounded once
(s of its value); fp16 results also carry half of fp16's smallest step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
EPS = 1e-5
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(rows, n, dt, wdt, seed, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x = (r(rows, n) + offset * r(rows, 1)).to(dt)
    h = (r(rows, n) * 2).to(dt)
    w, b = (1 + 0.3 * r(n)).to(wdt), (0.2 * r(n)).to(wdt)
    return x, h, w, b, r(rows, n).to(dt), r(rows, n).to(dt)


def formula(x, w, b, dy, ds=None):
    """y, dx, dw, db in 64 bits and the bounds' parts; x: the rows that the norm reads."""
    x, dy = x.double(), dy.double()
    n = x.shape[1]
    w64 = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(n, dtype=torch.float64) if b is None else b.double()
    m = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + EPS)
    xhat = (x - m) * rstd
    g = dy * w64
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
    cancel = 64 * U * (1 + x.abs().amax(1, keepdim=True) * rstd)
    tol_x = cancel * (1 + xhat.abs())
    gm = g.abs().mean(1, keepdim=True)
    xm = 1 + xhat.abs().amax(1, keepdim=True)
    return {"y": (xhat * w64 + b64, tol_x * w64.abs() + 2 * U * b64.abs()),
            "dx": (dx, rstd * cancel * ((1 + xhat.abs()) * (gm * xm * 4) + 2 * g.abs()) + (2 * U * dx.abs())),
            "dw": ((dy * xhat).sum(0), (dy.abs() * (tol_x + (x.shape[0] / 512 + 40) * U * xhat.abs())).sum(0)),
            "db": (dy.sum(0), (x.shape[0] / 512 + 40) * U * dy.abs().sum(0))}


def close(got, want, what):
    ref, tol = want
    g = got.detach().cpu().double()
    assert g.shape == ref.shape, what
    bar = half(got.dtype) * (1 + 2 ** -8) * ref.abs() + TINY[got.dtype] + tol
    bad = ~((g - ref).abs() <= bar)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {((g - ref).abs() / bar).max()}"


def d(t, grad=True):
    return None if t is None else t.to(DEV).requires_grad_(grad)


SHAPES = [(1, 1), (5, 1), (3, 2), (2, 7), (1, 8), (9, 9), (300, 64), (67, 100), (2050, 128), (33, 511), (7, 513),
          (129, 1733), (23, 2048), (517, 2816), (1030, 2049), (5, 8191), (3, 8193), (2, 16384), (1, 16383)]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_layernorm(rows, n, dt, wide):
    from smel.norm import layernorm
    x, _, w, b, dy, _ = make(rows, n, DT[dt], torch.float32 if wide else DT[dt], rows * 31 + n)
    xg, wg, bg = d(x), d(w), d(b)
    y = layernorm(xg, wg, bg, EPS)
    gr = torch.autograd.grad(y, (xg, wg, bg), dy.to(DEV))
    want = formula(x, w, b, dy)
    for name, t in zip(("y", "dx", "dw", "db"), (y, *gr)):
        close(t, want[name], name)
    assert y.dtype == x.dtype and gr[1].dtype == w.dtype and gr[2].dtype == w.dtype
    with torch.no_grad():       # without gradients, and again: the same bits
        assert torch.equal(layernorm(xg, wg, bg, EPS), y)
    again = torch.autograd.grad(layernorm(xg, wg, bg, EPS), (xg, wg, bg), dy.to(DEV))
    assert all(torch.equal(a, c) for a, c in zip(gr, again))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 9), (67, 100), (300, 2048), (41, 2817), (3, 16384)])
def test_add_layernorm(rows, n, dt):
    from smel.norm import add_layernorm
    x, h, w, b, dy, ds = make(rows, n, DT[dt], DT[dt], rows + n)
    s64 = (h.float() + x.float()).to(x.dtype)       # one rounding of an exact or singly rounded fp32 sum
    xg, hg, wg, bg = d(x), d(h), d(w), d(b)
    s, y = add_layernorm(hg, xg, wg, bg, EPS)
    assert torch.equal(s.cpu(), s64)
    full = formula(s64, w, b, dy, ds)
    dh, dx, dw, db = torch.autograd.grad((s, y), (hg, xg, wg, bg), (ds.to(DEV), dy.to(DEV)), retain_graph=True)
    assert torch.equal(dh, dx)
    for name, t in zip(("y", "dx", "dw", "db"), (y, dx, dw, db)):
        close(t, full[name], name)
    dx, = torch.autograd.grad(y, xg, dy.to(DEV), retain_graph=True)          # the sum itself not used
    close(dx, formula(s64, w, b, dy)["dx"], "dx without ds")
    dx, dw = torch.autograd.grad(s, (xg, wg), ds.to(DEV), allow_unused=True)  # the norm not used
    assert torch.equal(dx.cpu(), ds) and dw is None


@pytest.mark.parametrize("have", ["none", "w", "b"])
def test_layernorm_without_weights(have):
    from smel.norm import layernorm
    x, _, w, b, dy, _ = make(70, 250, torch.bfloat16, torch.float32, 3)
    w, b = (w if have == "w" else None), (b if have == "b" else None)
    xg, wg, bg = d(x), d(w), d(b)
    y = layernorm(xg, wg, bg, EPS)
    leaves = [t for t in (xg, wg, bg) if t is not None]
    gr = torch.autograd.grad(y, leaves, dy.to(DEV))
    want = formula(x, w, b, dy)
    close(y, want["y"], "y")
    close(gr[0], want["dx"], "dx")
    if have != "none":
        close(gr[1], want["d" + have], "d" + have)


@pytest.mark.parametrize("frozen", ["x", "w", "b", "wb"])
def test_layernorm_gradients_asked_for(frozen):
    from smel.norm import layernorm
    x, _, w, b, dy, _ = make(45, 136, torch.float32, torch.float32, 5)
    ts = {"x": d(x, "x" not in frozen), "w": d(w, "w" not in frozen), "b": d(b, "b" not in frozen)}
    y = layernorm(ts["x"], ts["w"], ts["b"], EPS)
    y.backward(dy.to(DEV))
    want = formula(x, w, b, dy)
    for k, t in ts.items():
        if k in frozen:
            assert t.grad is None
        else:
            close(t.grad, want["dx" if k == "x" else "d" + k], k)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_layernorm_views(dt):
    """Column slices at an odd offset, rows far apart, transposed and expanded inputs, 3-D rows, a gradient that is a view."""
    from smel.norm import add_layernorm, layernorm
    g = torch.Generator().manual_seed(9)
    base = torch.randn(40, 301, generator=g).to(DT[dt])
    w, b = torch.randn(100, generator=g), torch.randn(100, generator=g)
    bd = base.to(DEV)
    views = {"slice": lambda t: t[:, 3:103], "rows": lambda t: t[::3, 101:201], "transposed": lambda t: t[:, :100].t()[:100, :40].t(),
             "3d": lambda t: t[:, 1:].view(40, 3, 100), "expanded": lambda t: t[:1, :100].expand(6, 100)}
    for name, view in views.items():
        x = view(base)
        xg = view(bd).detach().requires_grad_(True)
        dyb = torch.randn(*x.shape[:-1], 2 * x.shape[-1], generator=g).to(DT[dt])
        dy = dyb[..., ::2]
        y = layernorm(xg, w.to(DEV), b.to(DEV), EPS)
        dx, = torch.autograd.grad(y, xg, dyb.to(DEV)[..., ::2])
        want = formula(x.reshape(-1, 100), w, b, dy.reshape(-1, 100))
        close(y.reshape(-1, 100), want["y"], name)
        close(dx.reshape(-1, 100), want["dx"], name)
        s, y2 = add_layernorm(view(bd), view(bd), w.to(DEV), b.to(DEV), EPS)
        close(y2.reshape(-1, 100), formula((2 * x.float()).to(x.dtype).reshape(-1, 100), w, b, dy.reshape(-1, 100))["y"], name)


def test_layernorm_large_mean_and_constant_rows():
    """Rows far from zero keep their spread (the mean is taken out before squaring); a constant row gives b."""
    from smel.norm import layernorm
    g = torch.Generator().manual_seed(2)
    x = torch.randn(20, 700, generator=g) + 4096.0
    x[3] = 17.25
    w, b = torch.randn(700, generator=g), torch.randn(700, generator=g)
    dy = torch.randn(20, 700, generator=g)
    xg = d(x)
    y = layernorm(xg, w.to(DEV), b.to(DEV), EPS)
    dx, = torch.autograd.grad(y, xg, dy.to(DEV))
    want = formula(x, w, b, dy)
    close(y, want["y"], "y")
    close(dx, want["dx"], "dx")


def test_layernorm_special_values():
    """inf or NaN in a row spoils that row alone, of y and dx; the weights' gradients take it up."""
    from smel.norm import layernorm
    x, _, w, b, dy, _ = make(12, 300, torch.float32, torch.float32, 8)
    x[2, 5], x[7, 299] = float("nan"), float("inf")
    xg, wg = d(x), d(w)
    y = layernorm(xg, wg, b.to(DEV), EPS)
    dx, dw = torch.autograd.grad(y, (xg, wg), dy.to(DEV))
    spoilt = torch.zeros(12, dtype=torch.bool)
    spoilt[[2, 7]] = True
    assert torch.isnan(y.cpu()[spoilt]).all() and torch.isnan(dx.cpu()[spoilt]).all() and torch.isnan(dw.cpu()).all()
    want = formula(x[~spoilt], w, b, dy[~spoilt])
    close(y[~spoilt.to(DEV)], want["y"], "y")
    close(dx[~spoilt.to(DEV)], want["dx"], "dx")


def test_layernorm_empty():
    from smel.norm import add_layernorm, layernorm
    x = torch.empty(0, 40, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w, b = d(torch.ones(40)), d(torch.zeros(40))
    y = layernorm(x, w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not dw.any() and not db.any()
    s, y = add_layernorm(x, x.detach(), w, b, EPS)
    assert s.shape == y.shape == (0, 40)


def test_layernorm_against_differences():
    """dx, dw and db against the difference quotient of the kernel's own forward. Its distance from the gradient is the
    quotient's own error (measured in 64 bits on the formula) and the forward's rounding over the step: 2 tol / 2h."""
    from smel.norm import layernorm
    x, _, w, b, c, _ = make(6, 40, torch.float32, torch.float32, 12)
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g) for t in (x, w, b)]
    xg, wg, bg = d(x), d(w), d(b)
    gr = torch.autograd.grad(layernorm(xg, wg, bg, EPS), (xg, wg, bg), c.to(DEV))
    step = 2.0 ** -7
    for i in range(3):
        at = lambda k: [t + (k * step * dirs[i] if j == i else 0) for j, t in enumerate((x, w, b))]
        up, dn = at(1), at(-1)
        f = lambda a: (layernorm(*(t.to(DEV) for t in a), EPS).double().cpu() * c.double()).sum()
        f64 = lambda a: (formula(a[0], a[1], a[2], c)["y"][0] * c.double()).sum()
        quotient = (f(up) - f(dn)) / (2 * step)
        analytic = (gr[i].double().cpu() * dirs[i].double()).sum()
        w64 = formula(x, w, b, c)[("dx", "dw", "db")[i]][0]
        own_error = ((f64(up) - f64(dn)) / (2 * step) - (w64 * dirs[i].double()).sum()).abs()
        ref, tol = formula(up[0], up[1], up[2], c)["y"]
        rounding = ((tol + U * ref.abs()) * c.abs().double()).sum() / step
        assert (quotient - analytic).abs() <= own_error + rounding + 1e-4


def test_layernorm_graph_and_streams():
    """Forward and backward captured and replayed between eager work; calls on two streams at once."""
    from smel.norm import add_layernorm
    x, h, w, b, dy, ds = (t.to(DEV) for t in make(260, 1000, torch.bfloat16, torch.float32, 4))

    def step(x=x, h=h):
        ts = [t.detach().requires_grad_(True) for t in (x, h, w, b)]
        s, y = add_layernorm(ts[1], ts[0], ts[2], ts[3], EPS)
        return [s, y, *torch.autograd.grad((s, y), ts, (ds, dy))]

    ref = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.detach().fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, ref))
        assert all(torch.equal(a, c) for a, c in zip(step(), ref))
    other = step(x=h, h=(x * 2))
    torch.cuda.synchronize()
    s2 = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s2):
            two = step(x=h, h=(x * 2))
        one = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(one, ref))
        assert all(torch.equal(a, c) for a, c in zip(two, other))


def test_layernorm_refusals():
    from smel.norm import add_layernorm, layernorm
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (lambda: layernorm(x.double(), w, w, EPS), lambda: layernorm(x, w.bfloat16(), None, EPS),
                lambda: layernorm(x.bfloat16(), w.half(), None, EPS), lambda: layernorm(x, w[:4], None, EPS),
                lambda: layernorm(x, w.cpu(), None, EPS), lambda: layernorm(x, torch.ones(16, device=DEV)[::2], None, EPS),
                lambda: layernorm(x.bfloat16(), w, w.bfloat16(), EPS), lambda: layernorm(torch.zeros(2, 16385, device=DEV), None, None, EPS),
                lambda: layernorm(torch.zeros(2, 0, device=DEV), None, None, EPS), lambda: layernorm(x[0, 0], None, None, EPS),
                lambda: add_layernorm(x, x[:2], w, w, EPS), lambda: add_layernorm(x.bfloat16(), x, w, w, EPS)):
        with pytest.raises(ValueError):
            bad()
    xg = x.clone().requires_grad_(True)
    y = layernorm(xg, w, w, EPS)
    gx, = torch.autograd.grad(y, xg, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):      # once differentiable
        gx.sum().backward()


def test_layernorm_saved_tensors_moved():
    """Hooks that take saved tensors to the host and back (repacked) change nothing, strided rows included."""
    from smel.norm import add_layernorm, layernorm
    x, h, w, b, dy, ds = (t.to(DEV) for t in make(40, 120, torch.bfloat16, torch.float32, 3))
    for cut in (slice(None), slice(10, 110)):
        xs = x[:, cut].detach().requires_grad_(True)
        wg, bg = w[cut].clone().requires_grad_(True), b[cut].clone().requires_grad_(True)
        ref = torch.autograd.grad(layernorm(xs, wg, bg, EPS), (xs, wg, bg), dy[:, cut])
        with torch.autograd.graph.save_on_cpu():
            y = layernorm(xs, wg, bg, EPS)
        assert all(torch.equal(a, c) for a, c in zip(ref, torch.autograd.grad(y, (xs, wg, bg), dy[:, cut])))
    hg = h.detach().requires_grad_(True)
    ref, = torch.autograd.grad(add_layernorm(hg, x, w, b, EPS), hg, (ds, dy))
    with torch.autograd.graph.save_on_cpu():
        out = add_layernorm(hg, x, w, b, EPS)
    assert torch.equal(ref, torch.autograd.grad(out, hg, (ds, dy))[0])


def test_layernorm_backward_twice():
    from smel.norm import layernorm
    x, _, w, b, dy, _ = make(300, 96, torch.float16, torch.float16, 9)
    xg, wg, bg = d(x), d(w), d(b)
    y = layernorm(xg, wg, bg, EPS)
    one = torch.autograd.grad(y, (xg, wg, bg), dy.to(DEV), retain_graph=True)
    two = torch.autograd.grad(y, (xg, wg, bg), dy.to(DEV))
    assert all(torch.equal(a, c) for a, c in zip(one, two))


def test_layernorm_functional_transforms_refused():
    """torch.func's transforms have no rule for it and say so; ordinary calls go on after one."""
    from smel.norm import layernorm
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layernorm(t, w, None, EPS).sum())(x)
    assert layernorm(x.requires_grad_(True), w, None, EPS).requires_grad


def test_layernorm_far_offsets():
    """Rows whose offsets pass 2^31 elements: far apart in a view, and packed (two million rows): the same bits as alone."""
    from smel.norm import layernorm
    g = torch.Generator(device=DEV).manual_seed(1)
    w, b = torch.randn(96, generator=g, device=DEV), torch.randn(96, generator=g, device=DEV)
    far = torch.zeros(1100, 1 << 21, dtype=torch.bfloat16, device=DEV)[:, 5:101]
    near = torch.randn(1100, 96, generator=g, device=DEV).bfloat16()
    far.copy_(near)
    dy = torch.randn(1100, 96, generator=g, device=DEV).bfloat16()

    def grads(x, dy):
        ts = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layernorm(ts[0], ts[1], ts[2], EPS)
        return [y.detach(), *torch.autograd.grad(y, ts, dy)]
    assert all(torch.equal(p, q) for p, q in zip(grads(near, dy), grads(far, dy)))
    del far
    n, rows = 1024, (1 << 21) + 77
    x = torch.zeros(rows, n, dtype=torch.float16, device=DEV)
    some = torch.randn(100, n, generator=g, device=DEV).half()
    x[:100] = x[-100:] = some       # the same rows before and behind 2^31 elements, of one call
    xg = x.requires_grad_(True)
    y = layernorm(xg, None, None, EPS)
    dx, = torch.autograd.grad(y, xg, y.detach())
    assert torch.equal(y[:100], y[-100:]) and torch.equal(dx[:100], dx[-100:])
    assert not y[100:103].any() and not y[-101].any() and not dx[-101].any()
    close(y[-100:], formula(some.cpu(), None, None, torch.zeros_like(some).cpu())["y"], "y")


def test_layernorm_forward_mode_refused():
    """A tangent is not dropped: forward mode has no rule and says so, with and without gradients."""
    import torch.autograd.forward_ad as fw
    from smel.norm import add_layernorm, layernorm
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with fw.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for bad in (lambda d: layernorm(d(x), w, None, EPS), lambda d: layernorm(x, d(w), None, EPS),
                            lambda d: layernorm(x, w, d(w), EPS), lambda d: add_layernorm(d(x), x, w, w, EPS)):
                    with pytest.raises(NotImplementedError):
                        bad(lambda t: fw.make_dual(t, torch.ones_like(t)))
        plain = layernorm(x, w, None, EPS)      # without a tangent in the call
    assert torch.equal(plain, layernorm(x, w, None, EPS)) and not plain.requires_grad


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", [(7001, 1100), (14001, 520), (4700, 2056), (2500, 4104), (1100, 8200)])
def test_layernorm_backward_many_turns(rows, n, dt):
    """Rows enough that every block of the backward goes through its rows' buffers more than once, with a part of a turn at the
    end: blocks of 256, 512 and 1024 threads, several rows a block and one, four, two and one on their way."""
    from smel.norm import add_layernorm, layernorm
    x, h, w, b, dy, ds = make(rows, n, DT[dt], DT[dt], rows + n)
    xg, wg, bg = d(x), d(w), d(b)
    gr = torch.autograd.grad(layernorm(xg, wg, bg, EPS), (xg, wg, bg), dy.to(DEV))
    want = formula(x, w, b, dy)
    for name, t in zip(("dx", "dw", "db"), gr):
        close(t, want[name], name)
    if n > 2000:
        return
    s64 = (h.float() + x.float()).to(x.dtype)
    gr = torch.autograd.grad(add_layernorm(d(h), xg, wg, bg, EPS), (xg, wg, bg), (ds.to(DEV), dy.to(DEV)))
    want = formula(s64, w, b, dy, ds)
    for name, t in zip(("dx", "dw", "db"), gr):
        close(t, want[name], name)
