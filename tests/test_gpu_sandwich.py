"""The norms around a gated and scaled residual add (smel.norm.post_rmsnorm, sandwich_rmsnorm over include/smel_norm.h) against the
formula in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half = eps(dtype) / 2): a row's sums add at most 64 values one after the other on any path
(32 in a thread, six levels of a wave, 16 waves), so a sum of squares is off by 70 u and a reciprocal root by half of that and its own
roundings: 44 u. A sigmoid is off by 10 u. y and the backward are compared at the stream s that the kernel wrote (the next block
reads that one). The products behind a sum add its own terms' errors; weights' gradients add up rows / 512 + 40 rows' terms on a path.
Every output is then rounded once (half of its value; fp16 also half of its smallest step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
NAMES = ("h", "x", "w1", "w2", "gate", "scale")


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(rows, n, dt, wdt, seed, gate="none", scale="none", plus_one=False, pre=True, gate_dt=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    one = 0.0 if plus_one else 1.0
    t = {"h": (2 * r(rows, n)).to(dt), "x": (0.5 * r(rows, n) + 0.2 * r(rows, 1)).to(dt), "w1": (one + 0.3 * r(n)).to(wdt),
         "w2": (one + 0.3 * r(n)).to(wdt) if pre else None, "gate": None, "scale": None}
    if gate != "none":
        shape, gd = {"channel": ((n,), wdt), "token": ((rows, 1), gate_dt or dt), "full": ((rows, n), dt)}[gate]
        t["gate"] = r(*shape).to(gd)
    if scale == "tensor":
        t["scale"] = torch.full((1,), 0.7).to(dt)
    if scale == "wide":
        t["scale"] = torch.full((), -1.3)
    if scale == "number":
        t["scale"] = 0.6
    return t, r(rows, n).to(dt), r(rows, n).to(dt) if pre else None


def formula(t, s, ds, dy, act, plus_one):
    """Outputs and gradients in 64 bits with the bounds' parts; s: the stream as the kernel wrote it (None: not looked at)."""
    d = lambda v: v.double() if torch.is_tensor(v) else v  # noqa: E731
    h, x, one = d(t["h"]), d(t["x"]), 1.0 if plus_one else 0.0
    rows, n = x.shape
    w1 = d(t["w1"]) + one if t["w1"] is not None else torch.ones(n, dtype=torch.float64)
    w2 = d(t["w2"]) + one if t["w2"] is not None else torch.ones(n, dtype=torch.float64)
    z = t["gate"]
    g = torch.ones(1, 1, dtype=torch.float64) if z is None else torch.sigmoid(d(z)) if act else d(z)
    slope = g * (1 - g) if act else torch.ones_like(g)
    sc = 1.0 if t["scale"] is None else float(t["scale"])
    r1 = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * r1
    nn = xh * w1
    u = h + g * nn
    eu = 60 * U * (g * nn).abs() + 2 * U * (h.abs() + u.abs())
    out = {"s": (sc * u, abs(sc) * eu + U * (sc * u).abs())}
    q = r2 = sh = torch.zeros(1, 1, dtype=torch.float64)
    if s is not None:
        s = d(s)
        r2 = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
        sh = s * r2
        out["y"] = sh * w2, 50 * U * (sh * w2).abs()
    if ds is None and dy is None:
        return out
    zero = torch.zeros_like(x)
    dst, dyt = d(ds) if ds is not None else zero, d(dy) if dy is not None else zero
    q = dyt * w2
    e = dst + r2 * q
    m2, M2 = (q * sh).mean(1, keepdim=True), (q * sh).abs().mean(1, keepdim=True)
    dS = e - r2 * sh * m2
    tS = 2 * U * dst.abs() + r2 * U * (52 * q.abs() + 220 * sh.abs() * M2) + 2 * U * dS.abs()
    dh, th = sc * dS, abs(sc) * tS + 2 * U * (sc * dS).abs()
    out["h"] = dh, th
    dn = dh * g
    tn = g.abs() * th + 14 * U * dn.abs()
    v = g * nn
    BM = (v.abs() * (dst.abs() + r2 * q.abs())).mean(1, keepdim=True) + r2 * M2 * (v * sh).abs().mean(1, keepdim=True)
    m1 = (dn * w1 * xh).mean(1, keepdim=True)
    out["x"] = (r1 * (dn * w1 - xh * m1),
                r1 * (tn * w1.abs() + 50 * U * ((dn * w1).abs() + (xh * m1).abs()) + xh.abs() * abs(sc) * 420 * U * BM))
    path = (rows / 512 + 40) * U
    out["w1"] = (dn * xh).sum(0), (tn * xh.abs() + (50 * U + path) * (dn * xh).abs()).sum(0)
    out["w2"] = (dyt * sh).sum(0), ((50 * U + path) * (dyt * sh).abs()).sum(0)
    dg, tg = dh * nn * slope, (th * nn.abs() + 60 * U * (dh * nn).abs()) * slope.abs()
    if z is not None:
        if z.dim() == 1:
            out["gate"] = dg.sum(0), (tg + path * dg.abs()).sum(0)
        elif z.shape[1] == 1 and n != 1:
            BM1 = (nn.abs() * (dst.abs() + r2 * q.abs())).sum(1, keepdim=True) + r2 * M2 * (nn * sh).abs().sum(1, keepdim=True)
            out["gate"] = dg.sum(1, keepdim=True), slope.abs() * abs(sc) * 420 * U * BM1 + 20 * U * dg.sum(1, keepdim=True).abs()
        else:
            out["gate"] = dg, tg
    out["scale"] = (dS * u).sum(), (tS * u.abs() + eu * dS.abs() + 40 * U * (dS * u).abs()).sum()
    return out


def close(got, want, what):
    ref, tol = want
    g = got.detach().cpu().double()
    ref, tol = ref.reshape(g.shape), tol.reshape(g.shape)
    bar = half(got.dtype) * (1 + 2 ** -8) * ref.abs() + TINY[got.dtype] + tol
    if got.dtype is torch.float16:      # whose infinity stands for what is at least 65520, half a step above its largest value
        g, ref = g.clamp(-65520, 65520), ref.clamp(-65520, 65520)
    bad = ~((g - ref).abs() <= bar)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {((g - ref).abs() / bar).max()}"


def dev(t, grad=True, only=NAMES):
    return {k: v.to(DEV).requires_grad_(grad and k in only) if torch.is_tensor(v) else v for k, v in t.items()}


def call(t, pre, act, plus_one):
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    kw = dict(gate=t["gate"], gate_act="sigmoid" if act else None, scale=t["scale"])
    if pre:
        return sandwich_rmsnorm(t["h"], t["x"], t["w1"], t["w2"], EPS, plus_one, **kw)
    return (post_rmsnorm(t["h"], t["x"], t["w1"], EPS, plus_one, **kw),)


def leaves(t):
    return {k: v for k, v in t.items() if torch.is_tensor(v) and v.requires_grad}


def check(t, ds, dy, pre, act, plus_one, what=""):
    tg = dev(t)
    out = call(tg, pre, act, plus_one)
    gr = torch.autograd.grad(out, list(leaves(tg).values()), (ds.to(DEV), dy.to(DEV)) if pre else (ds.to(DEV),))
    s = out[0].detach().cpu()
    want = formula(t, s if pre else None, ds, dy, act, plus_one)
    close(out[0], want["s"], what + "s")
    if pre:
        close(out[1], want["y"], what + "y")
    for (k, v), gk in zip(leaves(tg).items(), gr):
        assert gk.shape == v.shape and gk.dtype == v.dtype
        close(gk, want[k], what + "d" + k)
    with torch.no_grad():       # without gradients: the same bits
        assert all(torch.equal(a, b) for a, b in zip(call(tg, pre, act, plus_one), out))
    again = torch.autograd.grad(call(tg, pre, act, plus_one), list(leaves(tg).values()), (ds.to(DEV), dy.to(DEV)) if pre else (ds.to(DEV),))
    assert all(torch.equal(a, b) for a, b in zip(gr, again))


SHAPES = [(1, 1), (5, 1), (3, 2), (2, 7), (1, 8), (9, 9), (300, 64), (67, 100), (2050, 128), (33, 511), (7, 513), (129, 1733), (23, 2048),
          (517, 2816), (1030, 2049), (5, 8191), (3, 8193), (2, 16384), (1, 16383)]
FORMS = [("none", False, "none"), ("channel", True, "tensor"), ("token", False, "wide"), ("full", True, "number"), ("channel", False, "none"),
         ("token", True, "none"), ("full", False, "tensor")]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_sandwich(rows, n, dt, wide):
    k = SHAPES.index((rows, n)) + 2 * wide + list(DT).index(dt)
    for i in (k, k + 3):
        gate, act, scale = FORMS[i % 7]
        pre, plus_one = i % 3 != 1, i % 2 == 1
        t, ds, dy = make(rows, n, DT[dt], torch.float32 if wide else DT[dt], rows * 31 + n, gate, scale, plus_one, pre)
        check(t, ds, dy, pre, act, plus_one, f"{gate} {act} {scale} {pre}: ")


@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("scale", ["none", "number", "tensor", "wide"])
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_every_form(gate, act, scale, pre):
    for dt, n in (("bf16", 200), ("fp32", 2500)):
        for gate_dt in (None, torch.float32) if gate == "token" else (None,):
            t, ds, dy = make(45, n, DT[dt], DT[dt], 8, gate, scale, False, pre, gate_dt)
            check(t, ds, dy, pre, act, False)


@pytest.mark.parametrize("only", [("h",), ("x",), ("w1",), ("w2",), ("gate",), ("scale",), ("h", "x"), ("w1", "gate"), ("x", "scale")])
@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_gradients_asked_for(only, gate):
    for pre in (True, False):
        if not pre and only == ("w2",):
            continue
        t, ds, dy = make(37, 264, torch.bfloat16, torch.float32, 11, gate, "tensor", False, pre)
        tg = dev(t, True, only)
        out = call(tg, pre, True, False)
        torch.autograd.backward(out, (ds.to(DEV), dy.to(DEV)) if pre else (ds.to(DEV),))
        want = formula(t, out[0].detach().cpu() if pre else None, ds, dy, True, False)
        for k, v in tg.items():
            if torch.is_tensor(v):
                if k in only:
                    close(v.grad, want[k], k)
                else:
                    assert v.grad is None


def test_one_output_used():
    """The stream alone, or the normed rows alone, carry a gradient."""
    for scale in ("none", "tensor"):
        t, ds, dy = make(60, 300, torch.bfloat16, torch.bfloat16, 4, "full", scale)
        tg = dev(t)
        s, y = call(tg, True, False, False)
        ks = list(leaves(tg))
        s64 = s.detach().cpu()
        gr = torch.autograd.grad(y, [tg[k] for k in ks], dy.to(DEV), retain_graph=True)
        want = formula(t, s64, None, dy, False, False)
        for k, g in zip(ks, gr):
            close(g, want[k], k)
        ks.remove("w2")
        gr = torch.autograd.grad(s, [tg[k] for k in ks], ds.to(DEV), retain_graph=True)
        want = formula(t, None, ds, None, False, False)
        for k, g in zip(ks, gr):
            close(g, want[k], k)
        dw2, = torch.autograd.grad(s, tg["w2"], ds.to(DEV), allow_unused=True)
        assert dw2 is None or not dw2.any()


def test_without_weights():
    for w1, w2 in ((None, "w2"), ("w1", None), (None, None)):
        for plus_one in (False, True):
            t, ds, dy = make(30, 130, torch.float32, torch.float32, 4, "none", "none", plus_one)
            t["w1"], t["w2"] = t["w1"] if w1 else None, t["w2"] if w2 else None
            ref = dict(t)
            if plus_one:       # no weight is 1 either way
                ref = {**t, "w1": t["w1"] if w1 else torch.zeros(130), "w2": t["w2"] if w2 else torch.zeros(130)}
            tg = dev(t)
            out = call(tg, True, False, plus_one)
            ls = leaves(tg)
            gr = torch.autograd.grad(out, list(ls.values()), (ds.to(DEV), dy.to(DEV)))
            want = formula(ref, out[0].detach().cpu(), ds, dy, False, plus_one)
            close(out[0], want["s"], "s")
            close(out[1], want["y"], "y")
            for k, g in zip(ls, gr):
                close(g, want[k], k)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_views(dt):
    """Column slices at odd offsets, rows far apart, transposed and expanded inputs, 3-D rows, strided gradients and gates."""
    g = torch.Generator().manual_seed(9)
    a, b = torch.randn(40, 301, generator=g).to(DT[dt]), torch.randn(40, 301, generator=g).to(DT[dt])
    views = {"slice": lambda t: t[:, 3:103], "rows": lambda t: t[::3, 101:201], "transposed": lambda t: t[:, :100].t()[:100, :40].t(),
             "3d": lambda t: t[:, 1:].view(40, 3, 100), "expanded": lambda t: t[:1, :100].expand(6, 100), "1d": lambda t: t[2, 5:105]}
    for name, view in views.items():
        h, x = view(a), view(b)
        for gate in ("channel", "token", "full"):
            shape = {"channel": (100,), "token": (*x.shape[:-1], 1), "full": tuple(x.shape)}[gate]
            wide = torch.randn(*shape[:-1], 2 * shape[-1], generator=g).to(DT[dt])
            dsw, dyw = (torch.randn(*x.shape[:-1], 200, generator=g).to(DT[dt]) for _ in range(2))
            w1, w2 = (1 + torch.randn(100, generator=g) / 3).to(DT[dt]), (1 + torch.randn(100, generator=g) / 3).to(DT[dt])
            tg = {"h": view(a.to(DEV)).detach(), "x": view(b.to(DEV)).detach(), "w1": w1.to(DEV), "w2": w2.to(DEV),
                  "gate": wide.to(DEV)[..., ::2].detach(), "scale": torch.full((1,), 0.5, device=DEV)}
            ls = {k: v.requires_grad_(True) for k, v in tg.items()}
            out = call(tg, True, True, False)
            gr = torch.autograd.grad(out, list(ls.values()), (dsw.to(DEV)[..., ::2], dyw.to(DEV)[..., 1::2]))
            flat = lambda v: v.reshape(-1, v.shape[-1])  # noqa: E731
            zg = wide[..., ::2]
            t = {"h": flat(h), "x": flat(x), "w1": w1, "w2": w2, "gate": zg if zg.dim() == 1 and zg.shape[0] == 100 else flat(zg),
                 "scale": torch.full((1,), 0.5)}
            want = formula(t, flat(out[0].detach().cpu()), flat(dsw[..., ::2]), flat(dyw[..., 1::2]), True, False)
            close(out[0], want["s"], name)
            close(out[1], want["y"], name)
            for k, gk in zip(ls, gr):
                assert gk.shape == ls[k].shape
                close(gk, want[k], f"{name} {gate} d{k}")


def test_special_values():
    """inf or NaN in a row spoils that row alone; rows of zeros give finite results; a scale of 0 gives zero rows and its gradient."""
    t, ds, dy = make(12, 300, torch.float32, torch.float32, 8, "full")
    clean = {k: v.clone() if torch.is_tensor(v) else v for k, v in t.items()}
    t["x"][2, 5], t["h"][7, 299], t["gate"][9, 0] = float("nan"), float("inf"), float("nan")
    tg, cg = dev(t), dev(clean)
    out, ref = call(tg, True, False, False), call(cg, True, False, False)
    gr = torch.autograd.grad(out, (tg["h"], tg["x"], tg["gate"], tg["w1"]), (ds.to(DEV), dy.to(DEV)))
    gc = torch.autograd.grad(ref, (cg["h"], cg["x"], cg["gate"], cg["w1"]), (ds.to(DEV), dy.to(DEV)))
    fine = torch.ones(12, dtype=torch.bool, device=DEV)
    fine[[2, 7, 9]] = False
    for a, b in zip((*out, *gr[:3]), (*ref, *gc[:3])):
        assert torch.equal(a[fine], b[fine])
    assert torch.isnan(out[1][~fine]).any(1).all() and torch.isnan(gr[3]).all()
    for dt in DT.values():
        t, ds, dy = make(6, 70, dt, dt, 8, "token", "tensor")
        t["x"].zero_()
        t["h"][3:].zero_()
        check(t, ds, dy, True, False, False)
        t["scale"] = torch.zeros(1, dtype=dt)
        tg = dev(t)
        s, y = call(tg, True, False, False)
        dsc, dh = torch.autograd.grad(s, (tg["scale"], tg["h"]), ds.to(DEV))
        assert not s.any() and not y.any() and not dh.any()
        close(dsc, formula(t, None, ds, None, False, False)["scale"], "dscale at 0")


def test_empty():
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    h = torch.empty(0, 40, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w, gate, sc = (torch.ones(40, device=DEV, requires_grad=True), torch.ones(40, device=DEV, requires_grad=True),
                   torch.ones((), device=DEV, requires_grad=True))
    s, y = sandwich_rmsnorm(h, h.detach(), w, w.detach(), EPS, gate=gate, scale=sc)
    dh, dw, dg, dsc = torch.autograd.grad((s, y), (h, w, gate, sc), (torch.empty_like(s), torch.empty_like(y)))
    assert s.shape == y.shape == dh.shape == (0, 40) and not dw.any() and not dg.any() and not dsc.any()
    assert post_rmsnorm(h.view(0, 40), h.detach(), None, EPS).shape == (0, 40)
    s, y = sandwich_rmsnorm(h, h, w, None, EPS, gate=torch.empty(0, 1, device=DEV))
    assert s.shape == (0, 40)


@pytest.mark.parametrize("gate,act", [("channel", True), ("token", True), ("full", False)])
def test_against_differences(gate, act):
    """Every gradient against the difference quotient of the kernel's own forward. Its distance from the gradient is the quotient's own
    error (measured in 64 bits on the formula) and the forward's rounding over the step. fp32 rows, whose s is rounded by 2^-24: the
    normed rows see that rounding, too."""
    t, cs, cy = make(6, 40, torch.float32, torch.float32, 12, gate, "tensor")
    g = torch.Generator().manual_seed(1)
    tg = dev(t)
    ls = leaves(tg)
    out = call(tg, True, act, False)
    gr = dict(zip(ls, torch.autograd.grad(out, list(ls.values()), (cs.to(DEV), cy.to(DEV)))))
    step = 2.0 ** -7

    def f64(v):
        a = formula(v, None, None, None, act, False)["s"][0]
        b = formula(v, a, None, None, act, False)["y"][0]
        return (a * cs.double()).sum() + (b * cy.double()).sum()

    def rounding(v):
        w = formula(v, None, None, None, act, False)["s"]
        y, ty = formula(v, w[0], None, None, act, False)["y"]
        r2w = (y / w[0]).abs()
        es = w[1] + U * w[0].abs()
        return (es * cs.abs()).sum() + ((ty + U * y.abs() + r2w * (es + w[0].abs() * (es / w[0].abs()).amax(1, keepdim=True))) * cy.abs()).sum()
    for k in ls:
        v = torch.randn(t[k].shape, generator=g)
        up, dn = {**t, k: t[k] + step * v}, {**t, k: t[k] - step * v}

        def f(at):
            a, b = call(dev(at, False), True, act, False)
            return (a.double().cpu() * cs.double()).sum() + (b.double().cpu() * cy.double()).sum()
        quotient = (f(up) - f(dn)) / (2 * step)
        got = (gr[k].double().cpu() * v.double()).sum()
        s64 = formula(t, None, None, None, act, False)["s"][0]
        ref = (formula(t, s64, cs, cy, act, False)[k][0].reshape(v.shape) * v.double()).sum()
        own = ((f64(up) - f64(dn)) / (2 * step) - ref).abs()
        assert (quotient - got).abs() <= own + (rounding(up) + rounding(dn)) / (2 * step) + 1e-4, k


def test_graph_and_streams():
    t, ds, dy = make(260, 1000, torch.bfloat16, torch.bfloat16, 4, "channel", "tensor")
    ds, dy = ds.to(DEV), dy.to(DEV)
    base = dev(t, False)

    def run(**kw):
        ls = {k: v.detach().requires_grad_(True) for k, v in {**base, **kw}.items()}
        out = call(ls, True, True, False)
        return [*out, *torch.autograd.grad(out, list(ls.values()), (ds, dy))]
    ref = [v.clone() for v in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        for v in out:
            v.detach().fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, ref))
        assert all(torch.equal(a, c) for a, c in zip(run(), ref))
    other = run(h=base["x"], x=base["h"])
    torch.cuda.synchronize()
    s2 = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s2):
            two = run(h=base["x"], x=base["h"])
        one = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(one, ref)) and all(torch.equal(a, c) for a, c in zip(two, other))


def test_refusals():
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    x, w = torch.zeros(4, 8, device=DEV), torch.ones(8, device=DEV)
    b = x.bfloat16()
    for bad in (lambda: post_rmsnorm(x.double(), x.double(), w, EPS), lambda: post_rmsnorm(x, x[:2], w, EPS), lambda: post_rmsnorm(x, b, w, EPS),
                lambda: post_rmsnorm(x, x, w[:4], EPS), lambda: post_rmsnorm(x, x, w.cpu(), EPS), lambda: post_rmsnorm(x.cpu(), x, w, EPS),
                lambda: post_rmsnorm(x, x.cpu(), w, EPS), lambda: post_rmsnorm(x, x, w.bfloat16(), EPS), lambda: post_rmsnorm(b, b, w.half(), EPS),
                lambda: post_rmsnorm(x, x, torch.ones(16, device=DEV)[::2], EPS), lambda: sandwich_rmsnorm(b, b, w, w.bfloat16(), EPS),
                lambda: post_rmsnorm(x, x, w, EPS, gate=torch.ones(4, device=DEV)), lambda: post_rmsnorm(x, x, w, EPS, gate=torch.ones(2, 1, device=DEV)),
                lambda: post_rmsnorm(b, b, w, EPS, gate=x), lambda: post_rmsnorm(x, x, w, EPS, gate=w.cpu()),
                lambda: post_rmsnorm(b, b, w, EPS, gate=w.bfloat16()), lambda: post_rmsnorm(b, b, None, EPS, gate=w.half()),
                lambda: post_rmsnorm(b, b, None, EPS, gate=torch.ones(4, 1, device=DEV).half()), lambda: post_rmsnorm(x, x, w, EPS, gate_act="tanh"),
                lambda: post_rmsnorm(x, x, w, EPS, scale=w), lambda: post_rmsnorm(x, x, w, EPS, scale=torch.ones(1)),
                lambda: post_rmsnorm(b, b, w, EPS, scale=torch.ones(1, device=DEV).half()), lambda: post_rmsnorm(x[0, 0], x[0, 0], None, EPS),
                lambda: post_rmsnorm(torch.zeros(2, 16385, device=DEV), torch.zeros(2, 16385, device=DEV), None, EPS),
                lambda: post_rmsnorm(torch.zeros(2, 0, device=DEV), torch.zeros(2, 0, device=DEV), None, EPS)):
        with pytest.raises(ValueError):
            bad()
    xg = x.clone().requires_grad_(True)
    y = post_rmsnorm(xg, xg, w, EPS)
    gx, = torch.autograd.grad(y, xg, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):      # once differentiable
        gx.sum().backward()


def test_saved_tensors_moved_and_twice():
    for cut in (slice(None), slice(10, 110)):
        t, ds, dy = make(40, 120, torch.bfloat16, torch.float32, 3, "token", "tensor")
        tg = {k: v.to(DEV) for k, v in t.items()}
        tg = {k: (v[..., cut] if v.shape[-1] == 120 else v).detach() for k, v in tg.items()}
        ls = {k: v.requires_grad_(True) for k, v in tg.items()}
        go = (ds.to(DEV)[:, cut], dy.to(DEV)[:, cut])
        out = call(tg, True, True, True)
        ref = torch.autograd.grad(out, list(ls.values()), go, retain_graph=True)
        two = torch.autograd.grad(out, list(ls.values()), go)
        with torch.autograd.graph.save_on_cpu():
            out = call(tg, True, True, True)
        moved = torch.autograd.grad(out, list(ls.values()), go)
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(ref, two, moved))


def test_transforms_and_forward_mode_refused():
    import torch.autograd.forward_ad as fw
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: post_rmsnorm(t, x, w, EPS).sum())(x)
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for bad in (lambda: post_rmsnorm(d(x), x, w, EPS), lambda: post_rmsnorm(x, d(x), w, EPS), lambda: post_rmsnorm(x, x, d(w), EPS),
                            lambda: sandwich_rmsnorm(x, x, w, d(w), EPS), lambda: post_rmsnorm(x, x, w, EPS, gate=d(w)),
                            lambda: post_rmsnorm(x, x, w, EPS, scale=d(w[:1]))):
                    with pytest.raises(NotImplementedError):
                        bad()
        plain = post_rmsnorm(x, x, w, EPS)
    assert torch.equal(plain, post_rmsnorm(x, x, w, EPS)) and not plain.requires_grad


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n", [(7001, 1100), (14001, 520), (40001, 60), (4700, 2056), (2500, 4104), (1100, 8200)])
def test_many_turns(rows, n, dt):
    """Rows enough that every block of the backward goes through its rows' buffers more than once, with a part of a turn at the end."""
    gate, scale = {1100: ("channel", "tensor"), 520: ("full", "none"), 60: ("channel", "wide"), 2056: ("token", "number"),
                   4104: ("channel", "none"), 8200: ("full", "tensor")}[n]
    t, ds, dy = make(rows, n, DT[dt], DT[dt], rows + n, gate, scale)
    check(t, ds, dy, True, True, False)


def test_far_offsets():
    """Rows whose offsets pass 2^31 elements: far apart in a view, and packed: the same bits as alone."""
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(96, generator=g, device=DEV)
    near, hn, ds, dy, gate = (torch.randn(1100, 96, generator=g, device=DEV).bfloat16() for _ in range(5))

    def grads(h, x, gate, ds, dy, w=w):
        ls = [v.detach().requires_grad_(True) for v in (h, x, gate)] + ([w.detach().requires_grad_(True)] if w is not None else [])
        from smel.norm import sandwich_rmsnorm
        out = sandwich_rmsnorm(ls[0], ls[1], ls[3] if w is not None else None, w, EPS, gate=ls[2], scale=0.5)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, ls, (ds, dy))]
    ref = grads(hn, near, gate, ds, dy)
    far = torch.zeros(1100, 1 << 21, dtype=torch.bfloat16, device=DEV)
    far[:, 5:101], far[:, 300:396] = near, hn
    assert all(torch.equal(a, b) for a, b in zip(ref, grads(far[:, 300:396], far[:, 5:101], gate, ds, dy)))
    del far
    n, rows = 1024, (1 << 21) + 77
    some = [torch.randn(100, n, generator=g, device=DEV).half() for _ in range(5)]

    def big(v):
        b = torch.zeros(rows, n, dtype=torch.float16, device=DEV)
        b[:100] = b[-100:] = v
        return b
    alone = grads(*some, w=None)
    got = grads(*(big(v) for v in some), w=None)
    for a, b in zip(got, alone):
        assert torch.equal(a[:100], b) and torch.equal(a[-100:], b) and not a[100:103].any() and not a[-101].any()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_one_tensor_in_several_places(dt):
    """The stream, the block's output and the gate may be one tensor: its gradient is the sum of theirs (each rounded once, and the
    sums rounded: three half steps of the parts)."""
    t, ds, dy = make(33, 260, DT[dt], DT[dt], 21)
    x = t["x"]
    apart = dev({**t, "h": x.clone(), "x": x.clone(), "gate": x.clone()})
    out = call(apart, True, True, False)
    parts = torch.autograd.grad(out, [apart[k] for k in ("h", "x", "gate")], (ds.to(DEV), dy.to(DEV)))
    xg = x.to(DEV).requires_grad_(True)
    one = {**dev(t), "h": xg, "x": xg, "gate": xg}
    same = call(one, True, True, False)
    assert all(torch.equal(a, b) for a, b in zip(out, same))
    dx, = torch.autograd.grad(same, xg, (ds.to(DEV), dy.to(DEV)))
    size = sum(p.double().abs() for p in parts)
    assert ((dx.double() - sum(p.double() for p in parts)).abs() <= 3 * half(x.dtype) * size).all()


def test_one_column():
    """Rows of one column: a gate of [rows, 1] is one per element of the rows' dtype, one per token in fp32."""
    for dt in DT.values():
        for gate_dt in (dt, torch.float32):
            t, ds, dy = make(50, 1, dt, dt, 3, "token", "tensor", gate_dt=gate_dt)
            check(t, ds, dy, True, True, False)


def test_four_dimensions():
    from smel.norm import sandwich_rmsnorm
    g = torch.Generator().manual_seed(5)
    h, x = (torch.randn(2, 3, 4, 72, generator=g).bfloat16().to(DEV) for _ in range(2))
    gate = torch.randn(2, 3, 4, 1, generator=g).bfloat16().to(DEV)
    s, y = sandwich_rmsnorm(h, x, None, None, EPS, gate=gate)
    s2, y2 = sandwich_rmsnorm(h.view(24, 72), x.view(24, 72), None, None, EPS, gate=gate.view(24, 1))
    assert s.shape == y.shape == h.shape and torch.equal(s.view(24, 72), s2) and torch.equal(y.view(24, 72), y2)
