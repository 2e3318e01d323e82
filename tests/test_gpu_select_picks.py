"""Which experts smel.moe.select_experts picks, and their weights, exactly: the ids have to be those of a stable sort of the scores that
the same call returns (their sum with the bias in fp32, groups by the fp32 sum of their best two), so nothing hangs on how a score is
rounded. Ties, rows of NaN and infinities and switched-off rows lie between ordinary ones, in the same wave where a wave takes four
tokens (4096 tokens and more), over lists of 1 to 16 experts a lane."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [  # T, E, K, groups, kept
    (37, 64, 6, 1, 1), (4100, 64, 6, 1, 1), (4101, 64, 8, 8, 3), (4103, 128, 8, 1, 1), (4099, 100, 9, 4, 2), (4097, 112, 16, 16, 3),
    (61, 128, 8, 4, 2), (63, 256, 8, 8, 4), (4097, 256, 8, 8, 4), (4098, 256, 16, 1, 1), (45, 495, 7, 33, 9), (43, 512, 16, 1, 1),
    (4096, 512, 10, 16, 4), (41, 511, 16, 7, 3), (39, 510, 12, 17, 5), (4100, 5, 5, 1, 1)]


def inputs(kind, T, E, seed):
    g = torch.Generator().manual_seed(seed)
    z = 1.5 * torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)
    clean = z.clone()
    special = torch.zeros(T, dtype=torch.bool)
    if kind == "ties":
        z = torch.randint(-2, 2, (T, E), generator=g).float()
        clean = z.clone()
    if kind == "special":
        special[1::3] = True
        for i, t in enumerate(range(1, T, 3)):
            k = i % 9
            if k == 0:
                z[t] = math.nan
            elif k == 1:
                z[t, torch.randperm(E, generator=g)[:max(1, E // 3)]] = math.nan
            elif k == 2:
                z[t] = -math.inf
            elif k == 3:
                z[t, torch.randperm(E, generator=g)[:E - 2]] = -math.inf
            elif k == 4:
                z[t, torch.randperm(E, generator=g)[:2]] = math.inf
            elif k == 5:
                z[t] = torch.finfo(torch.float32).min
            elif k == 6:
                z[t] = -120.0 + torch.rand(E, generator=g) * 60      # sigmoids from nothing to 1e-26
            elif k == 7:
                z[t] = 16 + torch.rand(E, generator=g) * 4           # sigmoids of few different values
            else:
                z[t, torch.randperm(E, generator=g)[:E // 2]] = torch.finfo(torch.float32).max
    return z, clean, special, 0.1 * torch.randn(E, generator=g), torch.randn(T, 16, generator=g)


def order(c):
    """c as numbers that sort as the picks do: NaN as -infinity, both infinities as numbers."""
    c = torch.where(c.isnan(), -math.inf, c).double()
    return c.clamp(-1e300, 1e300)


def picks(s, bias, K, groups, kept):
    c = s if bias is None else s + bias      # fp32
    T, E = c.shape
    v = order(c)
    if kept < groups:
        cg = torch.where(c.isnan(), -math.inf, c).view(T, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
        best = order(cg[:, :, 0] + cg[:, :, 1] if cg.shape[2] > 1 else cg[:, :, 0])
        keep = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, best.sort(dim=1, descending=True, stable=True).indices[:, :kept], True)
        v = torch.where(keep[:, :, None], v.view(T, groups, -1), -1.5e300).view(T, E)
    return v.sort(dim=1, descending=True, stable=True).indices[:, :K]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kind", ["random", "ties", "special"])
@pytest.mark.parametrize("T,E,K,groups,kept", SHAPES)
def test_picks_and_weights(T, E, K, groups, kept, kind, score):
    from smel.moe import select_experts
    z, clean, special, bias, d = inputs(kind, T, E, T + E)
    for b in (None, bias):
        kw = dict(score=score, bias=None if b is None else b.to(DEV), groups=groups, top_groups=kept, renorm=False, with_scores=True)

        def run(z):
            zg = z.to(DEV).requires_grad_(True)
            topv, topi, s = select_experts(zg, K, **kw)
            return topv.detach().cpu(), topi.cpu(), s.cpu(), torch.autograd.grad(topv, zg, d[:, :K].to(DEV))[0].cpu()
        topv, topi, s, dz = run(z)
        assert torch.equal(topi, picks(s, b, K, groups, kept))
        # the weights are the scores that were compared, bit for bit
        torch.testing.assert_close(topv, s.gather(1, topi), rtol=0, atol=0, equal_nan=True)
        if kind == "special":
            fine = ~special
            assert all(torch.equal(p[fine], q[fine]) for p, q in zip((topv, topi, s, dz), run(clean)))
            off = torch.isneginf(z).all(1)
            assert not topv[off].any() and not s[off].any() and not dz[off].any()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_weights_are_the_scores(dt):
    """Logits of 16 bits; scaled weights, and renormalised ones in their order."""
    from smel.moe import select_experts
    z = inputs("random", 300, 256, 1)[0].to({"bf16": torch.bfloat16, "fp16": torch.float16}[dt])
    for score in ("sigmoid", "softmax"):
        topv, topi, s = select_experts(z.to(DEV), 8, score, renorm=False, scale=4.0, with_scores=True)
        assert torch.equal(topv, 4 * s.gather(1, topi)) and (topv[:, 1:] <= topv[:, :-1]).all()
        topv = select_experts(z.to(DEV), 8, score)[0]
        assert (topv[:, 1:] <= topv[:, :-1]).all()


def test_not_a_number_stays():
    """A NaN logit's sigmoid is NaN (and counts as -infinity), a softmax row with one, or with an infinity, is NaN throughout; all else
    is a number. Infinite and far logits have the scores 0 and 1."""
    from smel.moe import select_experts
    for T in (40, 4101):
        z, _, _, _, _ = inputs("special", T, 64, 9)
        topv, topi, s = (t.cpu() for t in select_experts(z.to(DEV), 4, renorm=False, with_scores=True))
        assert torch.equal(s.isnan(), z.isnan()) and (s[z < -104] == 0).all() and (s[z > 17] == 1).all() and (s[z == 0] == 0.5).all()
        some = (~z.isnan()).sum(1) >= 4
        assert not topv[some].isnan().any() and topv[z.isnan().all(1)].isnan().all()
        s = select_experts(z.to(DEV), 4, "softmax", with_scores=True)[2].cpu()
        assert torch.equal(s.isnan(), (z.isnan() | (z == math.inf)).any(1, keepdim=True).expand(T, 64))
