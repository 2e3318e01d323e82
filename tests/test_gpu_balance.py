"""The router's balance loss (smel.loss.balance_loss over include/smel_loss.h) against its definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24): logits of magnitude under 32 give z - max exact to 32 u, an exponential and
its share of a row's sum to 64 u of its value (exp 3 u, the row's sum 16 u, two products); P adds positive terms, at most
tokens / 1024 + 300 one after the other on a path, so loss is off by at most (64 + that + 8) u of its value. A gradient p (v -
p.v) is off by 128 u of p (|v_e| + sum p |v|) (v centred) and rounded once to its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def make(T, E, K, dt, seed):
    g = torch.Generator().manual_seed(seed)
    z = (1.5 * torch.randn(T, E, generator=g) + torch.randn(E, generator=g)).to(DT[dt])
    topi = z.float().topk(K, dim=1).indices if T else torch.zeros(0, K, dtype=torch.int64)
    return z, topi


def definition(z, topi, mask=None, offsets=None, coef=1.0, go=1.0):
    """loss, counts [S, E], dlogits and dlogits' error scale, one sequence after the other in 64 bits."""
    T, E = z.shape
    K = topi.shape[1]
    off = [0, T] if offsets is None else [min(max(int(o), 0), T) for o in offsets]
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask
    S = len(off) - 1
    loss, live = 0.0, 0
    counts = torch.zeros(S, E, dtype=torch.int64)
    dz, err = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    for s in range(S):
        rows = [t for t in range(off[s], off[s + 1]) if keep[t]]
        if not rows:
            continue
        live += 1
        ids = topi[rows].reshape(-1)
        ids = ids[(ids >= 0) & (ids < E)]
        counts[s] = torch.bincount(ids, minlength=E)
        p = torch.softmax(z[rows].double(), 1)
        f = counts[s].double() * E / (K * len(rows))
        loss = loss + coef * (f * p.mean(0)).sum()
        v = coef * go * (f - f.mean()) / len(rows)
        dz[rows] = p * (v - (p * v).sum(1, keepdim=True))
        err[rows] = 128 * U * p * (v.abs() + (p * v.abs()).sum(1, keepdim=True))
    live = max(live, 1)
    return torch.as_tensor(loss, dtype=torch.float64) / live, counts, dz / live, err / live


def check(z, topi, mask=None, offsets=None, coef=1.0, go=1.0, offs_dtype=torch.int64, view=None):
    from smel.loss import balance_loss
    dev = lambda t: None if t is None else t.to(DEV)
    zg = (z.to(DEV) if view is None else view(z)).detach().requires_grad_(True)
    off = None if offsets is None else torch.tensor(offsets, dtype=offs_dtype, device=DEV)
    loss, counts = balance_loss(zg, dev(topi), mask=dev(mask), offsets=off, coef=coef)
    dz, = torch.autograd.grad(loss, zg, torch.tensor(go, device=DEV))
    wl, wc, wz, err = definition(z, topi, mask, offsets, coef, go)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int64 and not counts.requires_grad
    assert torch.equal(counts.cpu(), wc if offsets is not None else wc[0])
    assert abs(loss.item() - wl.item()) <= (372 + z.shape[0] / 1024) * U * abs(wl.item())
    assert dz.dtype == z.dtype and dz.shape == z.shape
    bar = torch.finfo(z.dtype).eps / 2 * 1.01 * wz.abs() + TINY[z.dtype] + err
    diff = (dz.cpu().double() - wz).abs()
    assert (diff <= bar).all(), f"{int((diff > bar).sum())} of {diff.numel()}, worst {(diff / bar.clamp_min(1e-300)).max()}"
    with torch.no_grad():
        l2, c2 = balance_loss(zg, dev(topi), mask=dev(mask), offsets=off, coef=coef)
    assert torch.equal(l2, loss) and torch.equal(c2, counts)
    return loss, counts, dz


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 8, 2), (2, 2, 1), (17, 8, 8), (23, 128, 8), (64, 64, 4), (65, 65, 3),
                                   (129, 100, 1), (300, 257, 16), (517, 256, 8), (700, 512, 10), (4099, 129, 8)])
def test_balance(T, E, K, dt):
    z, topi = make(T, E, K, dt, T + E)
    check(z, topi, coef=0.5, go=64.0)


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("offs", [torch.int32, torch.int64])
def test_balance_sequences_and_mask(ids, offs):
    """Empty sequences at the start, inside and at the end, sequences of one token, ones that end inside a chunk, a tail
    behind the last, a head before the first; masked tokens hold NaN."""
    T, E, K = 500, 96, 4
    z, topi = make(T, E, K, "fp32", 5)
    g = torch.Generator().manual_seed(3)
    mask = torch.rand(T, generator=g) > 0.3
    mask[100:130] = False
    zn = z.clone()
    zn[~mask] = float("nan")
    for offsets in ([0, 0, 1, 2, 2, 2, 40, 100, 130, 131, 480, 480], [7, 90, 450], [0, 500], list(range(0, 501)), [3, 3], [0, 700]):
        check(z, topi.to(ids), None, offsets, 0.3, 2.0, offs)
        check(zn, topi.to(ids), mask, offsets, 0.3, 2.0, offs)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T,E,K,offsets", [(2048, 3, 1, None), (2049, 64, 6, None), (8231, 509, 3, None), (8231, 481, 2, [0, 8000, 8000, 8229]),
                                           (16384, 512, 2, [9, 14000, 16384]), (4500, 130, 2, [5, 1300, 1333, 4499]),
                                           (6000, 31, 2, list(range(0, 6001, 60)))])
def test_balance_long(T, E, K, offsets, dt):
    """On both sides of the sizes at which blocks, chunks and the number of blocks that add a sequence's slots change; ids out of
    range count nowhere."""
    z, topi = make(T, E, K, dt, T)
    topi[::7, 0] = -1
    topi[3::11, K - 1] = E
    mask = torch.rand(T, generator=torch.Generator().manual_seed(E)) > 0.2
    check(z, topi.int(), mask, offsets, 1.0, 3.0)


def test_balance_nothing_counts():
    """No token, no counted token, only empty sequences: loss 0, counts 0, gradient 0."""
    z, topi = make(40, 16, 2, "bf16", 1)
    for mask, offsets in ((torch.zeros(40, dtype=torch.bool), None), (None, [0, 0, 0]), (None, [40, 40])):
        loss, counts, dz = check(torch.full_like(z, float("nan")) if mask is not None else z, topi, mask, offsets)
        assert loss.item() == 0 and not counts.any() and not dz.any()
    z0, t0 = make(0, 16, 2, "bf16", 1)
    loss, counts, dz = check(z0, t0)
    assert loss.item() == 0 and not counts.any() and dz.shape == (0, 16)


def test_balance_even_router_and_same_picks():
    """Every expert picked alike: the loss is coef whatever the logits, the gradient exactly zero. Ids twice in a row count
    twice; ids outside [0, E) nowhere."""
    E, T = 8, 64
    z = torch.randn(T, E, generator=torch.Generator().manual_seed(0))
    even = (torch.arange(T * 2).reshape(T, 2)) % E
    loss, counts, dz = check(z, even, coef=0.25)
    assert not dz.any() and (counts == 16).all()
    assert abs(loss.item() - 0.25) <= 400 * U * 0.25
    odd = torch.tensor([[1, 1], [7, -1], [8, 3], [-(1 << 40), 1 << 40]]).repeat(16, 1)
    _, counts, _ = check(z, odd)
    assert counts.tolist() == [0, 32, 0, 16, 0, 0, 0, 16]


def test_balance_special_logits():
    """Experts at -inf get no share and no gradient; large logits do not overflow; a NaN row spoils the loss and its own
    gradient, no other row's."""
    z, topi = make(50, 32, 4, "fp32", 2)
    z[:, 3] = float("-inf")
    z[4, 5:] = float("-inf")
    topi = z.topk(4, dim=1).indices
    check(z, topi)
    from smel.loss import balance_loss
    big = (z * 1e30).to(DEV).requires_grad_(True)
    loss, _ = balance_loss(big, topi.to(DEV))
    dz, = torch.autograd.grad(loss, big)
    assert torch.isfinite(loss) and torch.isfinite(dz).all()
    z[9, 0] = float("nan")
    zg = z.to(DEV).requires_grad_(True)
    loss, _ = balance_loss(zg, topi.to(DEV))
    dz, = torch.autograd.grad(loss, zg)
    assert torch.isnan(loss) and torch.isnan(dz[9]).any() and torch.isfinite(torch.cat((dz[:9], dz[10:]))).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_balance_views(dt):
    z, topi = make(77, 60, 3, dt, 4)
    wide = torch.zeros(77, 97, dtype=z.dtype, device=DEV)

    def cut(z):
        wide[:, 5:65] = z.to(DEV)
        return wide[:, 5:65]
    check(z, topi, view=cut)
    check(z, topi, view=lambda z: z.t().contiguous().to(DEV).t())
    from smel.loss import balance_loss
    ids = torch.zeros(77, 6, dtype=torch.int64, device=DEV)
    ids[:, ::2] = topi.to(DEV)
    mask = torch.zeros(77, 2, dtype=torch.bool, device=DEV)
    mask[::2, 0] = True
    a = balance_loss(z.to(DEV), ids[:, ::2], mask=mask[:, 0])
    b = balance_loss(z.to(DEV), topi.to(DEV), mask=mask[:, 0].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_balance_against_differences():
    """The gradient against the difference quotient of the kernel's own loss; its distance is the quotient's own error
    (measured in 64 bits) and the loss's rounding over the step."""
    from smel.loss import balance_loss
    z, topi = make(12, 20, 3, "fp32", 6)
    zg = z.to(DEV).requires_grad_(True)
    loss, _ = balance_loss(zg, topi.to(DEV))
    dz, = torch.autograd.grad(loss, zg)
    move = torch.randn(z.shape, generator=torch.Generator().manual_seed(2))
    h = 2.0 ** -5
    f = lambda a: balance_loss(a.to(DEV), topi.to(DEV))[0].double().cpu()
    f64 = lambda a: definition(a, topi)[0]
    up, dn = z + h * move, z - h * move
    quotient = (f(up) - f(dn)) / (2 * h)
    own = ((f64(up) - f64(dn)) / (2 * h) - (definition(z, topi)[2] * move.double()).sum()).abs()
    assert (quotient - (dz.double().cpu() * move.double()).sum()).abs() <= own + 373 * U * f64(up).abs() / h + 1e-6


def test_balance_graph_and_streams():
    from smel.loss import balance_loss
    z, topi = make(900, 256, 8, "bf16", 7)
    z2, topi2 = make(900, 256, 8, "bf16", 8)
    off = torch.tensor([0, 100, 640, 880], device=DEV)
    go = torch.tensor(3.0, device=DEV)
    a, b = (z.to(DEV), topi.to(DEV)), (z2.to(DEV), topi2.to(DEV))

    def step(z, topi):
        zg = z.detach().requires_grad_(True)
        loss, counts = balance_loss(zg, topi, offsets=off)
        return [loss, counts, torch.autograd.grad(loss, zg, go)[0]]

    ref, ref2 = [t.clone() for t in step(*a)], [t.clone() for t in step(*b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*a)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, ref))
        assert all(torch.equal(x, y) for x, y in zip(step(*b), ref2))
    for _ in range(3):
        with torch.cuda.stream(side):
            two = step(*b)
        one = step(*a)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(one, ref)) and all(torch.equal(x, y) for x, y in zip(two, ref2))


@pytest.mark.parametrize("dt,H", [("bf16", 128), ("fp32", 128), ("bf16", 96)])
def test_route_logits_and_their_gradient(dt, H):
    """route(with_logits): the same routing as without; logits of the rounding of x W^T; dx joins both gradients. Logits and
    products of H terms carry H u + one rounding in 16 bits, a gradient row E u and three roundings (dlogits of either part,
    their sum), dx one more: all against sums of magnitudes."""
    from smel.loss import balance_loss
    from smel.moe import route
    T, E, K = 70, 16, 2
    g = torch.Generator().manual_seed(11)
    x = torch.randn(T, H, generator=g).to(DT[dt])
    gw = (torch.randn(E, H, generator=g) * 0.1).to(DT[dt])
    plain = route(x.to(DEV), gw.to(DEV), K)
    xg = x.to(DEV).requires_grad_(True)
    probs, topv, topi, lg = route(xg, gw.to(DEV), K, with_logits=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, (probs, topv, topi)))
    assert lg.shape == (T, E) and lg.dtype == x.dtype and lg.requires_grad
    half = torch.finfo(x.dtype).eps / 2
    mag = x.double().abs() @ gw.double().abs().t()
    want = x.double() @ gw.double().t()
    assert ((lg.detach().cpu().double() - want).abs() <= half * 1.01 * want.abs() + H * U * mag).all()
    loss, counts = balance_loss(lg, topi, coef=0.1)
    assert counts.sum().item() == T * K
    dl, = torch.autograd.grad(loss, lg, retain_graph=True)
    cot = torch.randn(T, K, generator=g).to(DT[dt])
    only_v, = torch.autograd.grad(topv, xg, cot.to(DEV), retain_graph=True)
    only_l, = torch.autograd.grad(loss, xg, retain_graph=True)
    both, = torch.autograd.grad((topv, loss), xg, (cot.to(DEV), torch.ones((), device=DEV)))
    dl = dl.cpu().double()
    wl = dl @ gw.double()
    magl = dl.abs() @ gw.double().abs()
    assert ((only_l.cpu().double() - wl).abs() <= (half * 1.01) * wl.abs() + (3 * half + E * U) * magl).all()
    pv = plain[0].cpu().double()
    sel = topi.cpu()
    # topv = p_k / sum of the picked p: its own gradient through the softmax
    pk = pv.gather(1, sel)
    s = pk.sum(1, keepdim=True)
    dpk = (cot.double() - (cot.double() * pk).sum(1, keepdim=True) / s) / s
    dp = torch.zeros_like(pv).scatter(1, sel, dpk)
    dv = pv * (dp - (dp * pv).sum(1, keepdim=True))
    wb = (dv + dl) @ gw.double()
    magb = (dv.abs() + dl.abs() + pv * ((dp * pv).abs().sum(1, keepdim=True) + dp.abs())) @ gw.double().abs()
    assert ((both.cpu().double() - wb).abs() <= (half * 1.01) * wb.abs() + (4 * half + (E + 64) * U) * magb).all()
    assert torch.isfinite(only_v).all()


def test_balance_refusals():
    from smel.loss import balance_loss
    z, t = torch.zeros(6, 8, device=DEV), torch.zeros(6, 2, dtype=torch.int64, device=DEV)
    m, o = torch.ones(6, dtype=torch.bool, device=DEV), torch.tensor([0, 6], device=DEV)
    for bad in (lambda: balance_loss(z.double(), t), lambda: balance_loss(z[0], t), lambda: balance_loss(z, t[:5]),
                lambda: balance_loss(z, t.float()), lambda: balance_loss(z, t.cpu()), lambda: balance_loss(z, t, mask=m[:5]),
                lambda: balance_loss(z, t, mask=m.long()), lambda: balance_loss(z, t, offsets=o[:1]),
                lambda: balance_loss(z, t, offsets=o.float()), lambda: balance_loss(z, t, offsets=o.cpu())):
        with pytest.raises(ValueError):
            bad()
    from smel._lib import SmelError
    with pytest.raises(SmelError, match="experts"):
        balance_loss(torch.zeros(2, 600, device=DEV), t[:2])
    with pytest.raises(SmelError, match="K="):
        balance_loss(z, t[:, :0])
    zg = z.clone().requires_grad_(True)
    loss, _ = balance_loss(zg, t)
    zg.data.add_(0)
    with torch.no_grad():
        zg.add_(1)
    with pytest.raises(RuntimeError):      # changed in place before the backward
        loss.backward()


def test_balance_saved_tensors_moved():
    """Hooks that take saved tensors to the host and back (repacked) change nothing, strided rows included; twice is the same."""
    from smel.loss import balance_loss
    z, topi = make(200, 48, 4, "bf16", 3)
    wide = torch.zeros(200, 70, dtype=z.dtype, device=DEV)
    wide[:, 11:59] = z.to(DEV)
    off = torch.tensor([0, 30, 200], device=DEV)
    for t in (z.to(DEV), wide[:, 11:59]):
        zg = t.detach().requires_grad_(True)
        loss, _ = balance_loss(zg, topi.to(DEV), offsets=off)
        ref, = torch.autograd.grad(loss, zg, retain_graph=True)
        assert torch.equal(ref, torch.autograd.grad(loss, zg)[0])
        with torch.autograd.graph.save_on_cpu():
            loss, _ = balance_loss(zg, topi.to(DEV), offsets=off)
        assert torch.equal(ref, torch.autograd.grad(loss, zg)[0])


@pytest.mark.parametrize("dt,H", [("bf16", 128), ("fp32", 128), ("bf16", 96)])
def test_route_gemma4_logits_and_their_gradient(dt, H):
    """The same routing as without; the logits' gradient alone and with topv's is the sum of the two alone, to the roundings of
    dlogits' sum and of dx (the norm's backward mixes a row)."""
    from smel.loss import balance_loss
    from smel.moe import route_gemma4
    T, E, K = 70, 16, 2
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g)
    W = {"router.scale": (1 + 0.1 * r(H)).to(DEV, DT[dt]), "router.proj.weight": r(E, H).to(DEV, DT[dt]),
         "router.per_expert_scale": (1 + 0.1 * r(E)).to(DEV, DT[dt])}
    h = (2 * r(T, H)).to(DEV, DT[dt])
    plain = route_gemma4(h, W, K, 1e-6)
    hg = h.detach().requires_grad_(True)
    probs, topv, topi, lg = route_gemma4(hg, W, K, 1e-6, with_logits=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, (probs, topv, topi)))
    half = torch.finfo(lg.dtype).eps / 2
    soft = torch.softmax(lg.detach().double(), 1)
    # probs are the softmax of the logits (of the unrounded ones where the bf16 rows run on the fp32 kernels)
    assert ((probs.double() - soft).abs() <= soft * (64 * U + 4 * half * lg.detach().double().abs().amax(1, keepdim=True))).all()
    loss, _ = balance_loss(lg, topi)
    cot = r(T, K).to(DEV) * 1e-3
    only_l, = torch.autograd.grad(loss, hg, retain_graph=True)
    only_v, = torch.autograd.grad(topv, hg, cot, retain_graph=True)
    both, = torch.autograd.grad((topv, loss), hg, (cot, torch.ones((), device=DEV)))
    a, p, q = both.double(), only_l.double(), only_v.double()
    scale = p.abs() + q.abs()
    assert p.abs().max() > 0 and ((a - p - q).abs() <= 16 * half * (scale + scale.amax(1, keepdim=True))).all()


def test_balance_far_offsets():
    """Rows whose offsets pass 2^31 elements: the same bits as packed ones."""
    from smel.loss import balance_loss
    z, topi = make(1100, 40, 4, "bf16", 9)
    far = torch.zeros(1100, 1 << 21, dtype=torch.bfloat16, device=DEV)[:, 3:43]
    far.copy_(z.to(DEV))
    out = []
    for t in (z.to(DEV), far):
        zg = t.detach().requires_grad_(True)
        loss, counts = balance_loss(zg, topi.to(DEV))
        out.append((loss.detach(), counts, torch.autograd.grad(loss, zg)[0]))
    assert all(torch.equal(p, q) for p, q in zip(*out))


def test_balance_forward_mode_refused():
    """A tangent is not dropped: forward mode has no rule and says so, with and without gradients."""
    import torch.autograd.forward_ad as fw
    from smel.loss import balance_loss
    z, topi = make(20, 8, 2, "fp32", 3)
    z, topi = z.to(DEV), topi.to(DEV)
    with fw.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                balance_loss(fw.make_dual(z, torch.ones_like(z)), topi)
        loss, counts = balance_loss(z, topi)
    again, counts2 = balance_loss(z, topi)
    assert torch.equal(loss, again) and torch.equal(counts, counts2) and not loss.requires_grad


@pytest.mark.parametrize("run", [5, 1 << 20])
def test_balance_run_of_empty_sequences(run):
    """Offsets that repeat, inside a chunk, at the start and at the end before a padded tail (a buffer of fixed length filled up with
    its last value): nothing that a block walks through one by one. A walk takes a trip to memory for each."""
    from smel.loss import balance_loss
    T, E, K = 300, 16, 2
    z, topi = make(T, E, K, "fp32", 5)
    cuts = [0] * run + [40, 41, 41, 60] + [60] * run + [61, 130, 130, 130, 250] + [250] * run
    used = [s for s in range(len(cuts) - 1) if cuts[s] < cuts[s + 1]]
    wl, wc, wz, err = definition(z, topi, None, [0, 40, 41, 60, 61, 130, 250], 1.0, 1.0)
    zg, off, ids = z.to(DEV).requires_grad_(True), torch.tensor(cuts, device=DEV), topi.to(DEV)
    ms = []
    for _ in range(2):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        loss, counts = balance_loss(zg, ids, offsets=off)
        e1.record()
        torch.cuda.synchronize()
        ms.append(e0.elapsed_time(e1))
    dz, = torch.autograd.grad(loss, zg)
    assert abs(loss.item() - wl.item()) <= 372 * U * wl.item()
    assert torch.equal(counts[used].cpu(), wc) and counts.sum().item() == 250 * K
    assert ((dz.cpu().double() - wz).abs() <= U * wz.abs() + err).all()
    assert min(ms) < 100, ms      # 227 with a walk of 2^20 trips to memory, 10 without


@pytest.mark.parametrize("T,S", [(131072, 4096), (65536, 0)])
def test_balance_keeps_what_the_backward_reads(T, S):
    """Between forward and backward: 16 bytes a token, the weights of each sequence's experts, under 1 MB of the workspace, and the
    results; not the slots of the sums (16 MB in the first case)."""
    from smel.loss import balance_loss
    E, K = 256, 2
    z = torch.randn(T, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16().requires_grad_(True)
    topi = z.detach().float().topk(K, dim=1).indices
    off = torch.arange(0, T + 1, T // S, device=DEV) if S else None
    warm = balance_loss(z, topi, offsets=off)
    ref, = torch.autograd.grad(warm[0], z)
    del warm
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss, counts = balance_loss(z, topi, offsets=off)
    kept = torch.cuda.memory_allocated() - before
    results = 8 * max(S, 1) * E + 4
    assert kept <= 16 * T + 4 * (max(S, 1) * E + 1) + results + (1 << 20) + 4096, kept
    # what the workspace's memory holds by then does not matter
    torch.empty(64 << 20, dtype=torch.uint8, device=DEV).fill_(255)
    assert torch.equal(torch.autograd.grad(loss, z)[0], ref)
