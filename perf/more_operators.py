"""More operators of the training step around the MoE layer, as measurable cases: the choice of experts from sigmoid or softmax
scores with groups and a bias, the norms on both sides of a residual add with its gate and scale, and the clipping of all
gradients by their global norm.

  select  ``smel.moe.select_experts``: weights and ids of the picks and (train) the gradient of the router's logits
  norm    ``smel.norm.post_rmsnorm`` / ``sandwich_rmsnorm``: the residual stream, the normed rows and (train) every gradient
  clip    ``smel.lora.clip_grads``: the global norm and every gradient scaled by it

Sizes are those of the two model shapes this package runs (hidden 2048 with 256 experts of 512, hidden 2816 with 128 experts of
704, top-8, LoRA rank 16 on twelve experts a layer), its tests' token counts, and odd ones around them.
"""
import math
import os
import random
import sys

import torch

_PKG = os.path.join(os.getcwd(), "smel-ft_amd")   # the package of the tree this runs in
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_TINY = 1e-20      # beside the sum of the picked scores
_CLIP_EPS = 1e-6   # beside the norm

_MAX_LOGITS = 32768 * 256
_MAX_ROWS = 32749 * 2048
_MAX_GRADS = 1 << 28


def _select(T, E, K, dtype, train, score="sigmoid", bias=True, groups=1, kept=1, renorm=True, off=0):
    return {"op": "select", "T": T, "E": E, "K": K, "dtype": dtype, "train": train, "score": score, "bias": bias,
            "groups": groups, "kept": kept, "renorm": renorm, "off": off}


def _norm(rows, cols, dtype, train, pre=True, gate="none", act=False, scale="none", trained=False, wide=False, plus_one=False):
    return {"op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "pre": pre, "gate": gate, "act": act,
            "scale": scale, "trained": trained, "wide": wide, "plus_one": plus_one}


def _clip_lora(layers, k, H, I, Is, r, dtype, most=1.0):
    return {"op": "clip", "layers": layers, "k": k, "H": H, "I": I, "Is": Is, "r": r, "dtype": dtype, "max": most}


def _clip_any(tensors, elems, dtype, most=1.0, sizes=0):
    return {"op": "clip", "layers": 0, "tensors": tensors, "elems": elems, "dtype": dtype, "max": most, "sizes": sizes}


def listed():
    return [
        # one token of a decoding step: eight groups of experts, four of them kept
        {"name": "select_eval_1", **_select(1, 256, 8, "bf16", False, groups=8, kept=4)},
        # a training step on one short sequence: softmax scores, no groups
        {"name": "select_train_517", **_select(517, 128, 8, "bf16", True, "softmax", False)},
        # a packed row, logits kept in 32 bits
        {"name": "select_train_4092", **_select(4092, 256, 8, "f32", True, groups=8, kept=4)},
        # a large batch, some experts switched off by their logits
        {"name": "select_train_32768", **_select(32768, 256, 8, "bf16", True, groups=8, kept=4, off=6)},
        # one token of a decoding step
        {"name": "norm_eval_1x2816", **_norm(1, 2816, "bf16", False, scale="frozen")},
        # a short sequence: a gate per channel, trained with both norms' weights, kept in 32 bits
        {"name": "norm_train_517x2048", **_norm(517, 2048, "f16", True, gate="channel", trained=True, wide=True)},
        # the block's end over a full packed row: frozen weights and layer scale
        {"name": "norm_train_4096x2816", **_norm(4096, 2816, "bf16", True, scale="frozen")},
        # odd sizes in 32 bits, a gate per token, no norm behind
        {"name": "post_train_1021x1733", **_norm(1021, 1733, "f32", True, pre=False, gate="token", act=True, scale="trained", trained=True)},
        # a large batch with a sigmoid gate from a projection
        {"name": "norm_train_32749x2048", **_norm(32749, 2048, "bf16", True, gate="full", act=True, plus_one=True)},
        # a layer's LoRA gradients: twelve selected experts and the shared one, rank 16
        {"name": "clip_layer_r16", **_clip_lora(1, 12, 2048, 512, 512, 16, "f32")},
        # five layers' of the other shape
        {"name": "clip_5_layers_r16", **_clip_lora(5, 12, 2816, 704, 2112, 16, "f32")},
        # the gradients of full matrices, of any size
        {"name": "clip_matrices", **_clip_any(21, (1 << 28) - 12345, "bf16", sizes=3)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["select", "norm", "clip", "select", "norm", "norm", "clip_lora"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.75
    if kind == "select":
        G = rng.choice([1, 1, 1, 2, 4, 8, 8, rng.randint(2, 12)])
        gs = rng.choice([8, 16, 32, 64, rng.randint(2, 64)]) if G > 1 else rng.choice([64, 128, 256, 512, rng.randint(2, 511)])
        gs = min(gs, 512 // G)
        E = G * gs
        kept = rng.randint(1, G)
        K = rng.randint(1, min(16, kept * gs, max(1, E // 2)))
        score = rng.choice(["sigmoid", "sigmoid", "softmax"])
        return _select(_log(rng, 1, min(131072, _MAX_LOGITS // E)), E, K, dtype, train, score, score == "sigmoid" or rng.random() < 0.3,
                       G, kept, rng.random() < 0.8, rng.choice([0, 0, 1]) if E >= 2 * K + 2 else 0)
    if kind == "norm":
        cols = rng.choice([64, 128, 512, 2048, 2816, 4096, 16384, _log(rng, 8, 16384), _log(rng, 8, 16384)])
        most = _MAX_ROWS // cols // (2 if dtype == "f32" else 1)
        gate = rng.choice(["none", "none", "channel", "token", "full"])
        return _norm(_log(rng, 1, min(131072, most)), cols, dtype, train, rng.random() < 0.75, gate, gate != "none" and rng.random() < 0.5,
                     rng.choice(["none", "frozen", "trained"]), rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.4)
    most = rng.choice([1.0, 1.0, 0.01, 1e9])
    if kind == "clip":
        return _clip_any(rng.randint(1, 48), _log(rng, 64, _MAX_GRADS // (2 if dtype == "f32" else 1)), dtype, most, rng.randrange(1 << 20))
    H, I = rng.choice([(2048, 512), (2816, 704)])
    return _clip_lora(rng.randint(1, 5), rng.randint(1, 16), H, I, rng.choice([512, 2112]), rng.choice([4, 6, 8, 16, 32]), dtype, most)


# ------------------------------------------------------------------------------------------------ inputs


def _seed(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)


def _apart(z, bias, case):
    """Rows whose picks do not hang on a rounding: in 64 bits, each of the first K + 1 choices is the next one's equal or well
    above it, and so are the last group kept and the first one dropped."""
    d = z.double()
    s = torch.sigmoid(d) if case["score"] == "sigmoid" else torch.softmax(d, dim=1)
    c = s if bias is None else s + bias.double()
    G, K, T = case["groups"], case["K"], z.shape[0]
    far = lambda hi, lo: (hi == lo) | (hi - lo > 4e-6 * (1e-3 + hi.abs()))  # noqa: E731
    ok = torch.ones(T, dtype=torch.bool, device=DEV)
    if case["kept"] < G:
        cg = c.view(T, G, -1)
        best = cg.topk(min(2, cg.shape[2]), dim=2).values.sum(dim=2)
        top = best.sort(dim=1, descending=True, stable=True)
        ok &= far(top.values[:, case["kept"] - 1], top.values[:, case["kept"]])
        keep = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, top.indices[:, :case["kept"]], True)
        c = torch.where(keep[:, :, None], cg, -torch.inf).view(T, -1)
    top = c.topk(min(K + 1, c.shape[1]), dim=1).values
    return ok & far(top[:, :-1], top[:, 1:]).all(dim=1)


def _prepare_select(case, g, dt):
    T, E = case["T"], case["E"]
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    bias = 0.05 * rand(E) if case["bias"] else None
    load = 0.5 * rand(E)       # some experts are more popular than others
    off = torch.randperm(E, generator=g, device=DEV)[:case["off"]]

    def fresh(n):
        z = (1.5 * rand(n, E) + load).to(dt)
        z[:, off] = -torch.inf
        return z
    z = fresh(T)
    for _ in range(30):
        bad = (~_apart(z, bias, case)).nonzero().flatten()
        if not bad.numel():
            break
        z[bad] = fresh(bad.numel())
    else:
        z[bad] = z[_apart(z, bias, case).nonzero()[0]]
    return {"case": case, "bias": bias, "logits": z.requires_grad_(case["train"]), "go": 1e-2 * rand(T, case["K"])}


def _prepare_norm(case, g, dt):
    R, n, t = case["rows"], case["cols"], case["train"]
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    loud = 1 + 8 * (torch.rand(n, generator=g, device=DEV) > 0.99)     # channels of large values, as residual streams have
    wdt = torch.float32 if case["wide"] else dt
    tw = t and case["trained"]
    one = 0.0 if case["plus_one"] else 1.0
    st["h"] = (2 * rand(R, n) * loud).to(dt).requires_grad_(t)
    st["x"] = (0.3 * rand(R, n) * loud).to(dt).requires_grad_(t)
    st["w1"] = (one + 0.2 * rand(n)).to(wdt).requires_grad_(tw)
    st["w2"] = (one + 0.2 * rand(n)).to(wdt).requires_grad_(tw) if case["pre"] else None
    st["gate"] = None
    if case["gate"] == "channel":
        st["gate"] = (0.5 + 0.3 * rand(n)).to(wdt).requires_grad_(tw)
    if case["gate"] == "token":
        st["gate"] = rand(R, 1).to(dt).requires_grad_(t)
    if case["gate"] == "full":
        st["gate"] = rand(R, n).to(dt).requires_grad_(t)
    st["scale"] = None if case["scale"] == "none" else torch.full((1,), 0.8, device=DEV).to(dt)
    if case["scale"] == "trained":
        st["scale"].requires_grad_(t)
    st["ds"] = (1e-2 * rand(R, n)).to(dt) if t else None
    st["dy"] = (1e-2 * rand(R, n)).to(dt) if t and case["pre"] else None
    return st


def _grad_shapes(case):
    """Of each layer A_gate, B_gate, A_up, B_up, A_down, B_down of the k experts and of the shared one; or matrices' sizes, odd ones
    and few large ones among them, that make up ``elems`` elements."""
    if case["layers"]:
        k, r, H = case["k"], case["r"], case["H"]
        one = lambda lead, i: [(*lead, r, H), (*lead, i, r), (*lead, r, H), (*lead, i, r), (*lead, r, i), (*lead, H, r)]  # noqa: E731
        return (one((k,), case["I"]) + one((), case["Is"])) * case["layers"]
    rng = random.Random(case["sizes"])
    share = [math.exp(rng.uniform(0, 6)) for _ in range(case["tensors"])]
    return [(max(1, int(case["elems"] * s / sum(share))),) for s in share]


def prepare(case, seed):
    g, dt = _seed(seed), _DT[case["dtype"]]
    if case["op"] == "select":
        return _prepare_select(case, g, dt)
    if case["op"] == "norm":
        return _prepare_norm(case, g, dt)
    shapes = _grad_shapes(case)
    size = 3.0 / math.sqrt(sum(math.prod(s) for s in shapes))        # a global norm of about 3
    return {"case": case, "grads": [(size * torch.randn(*s, generator=g, device=DEV)).to(dt) for s in shapes]}


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if case["op"] == "select":
        return _run_select(state, case)
    if case["op"] == "norm":
        return _run_norm(state, case)
    if own:
        from smel.lora import clip_grads
        out, norm = clip_grads(state["grads"], case["max"])
        return [norm, *out]
    return _plain_clip(state["grads"], case["max"])


def _run_select(st, case):
    z = st["logits"]
    if own:
        from smel.moe import select_experts
        topv, topi = select_experts(z, case["K"], score=case["score"], bias=st["bias"], groups=case["groups"],
                                    top_groups=case["kept"], renorm=case["renorm"], scale=2.5)
        return [topv, topi, torch.autograd.grad(topv, z, st["go"])[0]] if case["train"] else [topv, topi]
    with torch.no_grad():
        return _plain_select(st, case)


def _plain_select(st, case):
    z, K, G = st["logits"].float(), case["K"], case["groups"]
    T = z.shape[0]
    if case["score"] == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
    else:
        s = torch.exp(z - z.amax(dim=1, keepdim=True))
        s = s / s.sum(dim=1, keepdim=True)
    c = s if st["bias"] is None else s + st["bias"]
    if case["kept"] < G:
        cg = c.view(T, G, -1)
        best = cg.topk(min(2, cg.shape[2]), dim=2).values.sum(dim=2)
        first = best.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, first, True)
        c = torch.where(keep[:, :, None], cg, -torch.inf).view(T, -1)
    topi = c.sort(dim=1, descending=True, stable=True).indices[:, :K]
    sk = s.gather(1, topi)
    total = sk.sum(dim=1, keepdim=True) + _TINY if case["renorm"] else 1.0
    topv = 2.5 * sk / total
    if not case["train"]:
        return [topv, topi]
    d = 2.5 * st["go"]
    if case["renorm"]:
        d = (d - (d * sk).sum(dim=1, keepdim=True) / total) / total
    if case["score"] == "sigmoid":
        dz = torch.zeros_like(s).scatter_(1, topi, d * sk * (1 - sk))
    else:
        dz = s * (torch.zeros_like(s).scatter_(1, topi, d) - (d * sk).sum(dim=1, keepdim=True))
    return [topv, topi, dz.to(st["logits"].dtype)]


def _run_norm(st, case):
    if own:
        from smel.norm import post_rmsnorm, sandwich_rmsnorm
        act = "sigmoid" if case["act"] else None
        if case["pre"]:
            out = sandwich_rmsnorm(st["h"], st["x"], st["w1"], st["w2"], _EPS, case["plus_one"], gate=st["gate"], gate_act=act, scale=st["scale"])
        else:
            out = (post_rmsnorm(st["h"], st["x"], st["w1"], _EPS, case["plus_one"], gate=st["gate"], gate_act=act, scale=st["scale"]),)
        if not case["train"]:
            return list(out)
        return [*out, *torch.autograd.grad(out, _leaves(st), (st["ds"], st["dy"]) if case["pre"] else (st["ds"],))]
    with torch.no_grad():
        return _plain_norm(st, case)


def _leaves(st):
    return [t for t in (st["h"], st["x"], st["w1"], st["w2"], st["gate"], st["scale"]) if t is not None and t.requires_grad]


def _plain_norm(st, case):
    one = 1.0 if case["plus_one"] else 0.0
    h, x, dt = st["h"].float(), st["x"].float(), st["x"].dtype
    w1 = st["w1"].float() + one
    r1 = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    xhat = x * r1
    n = xhat * w1
    gate = None if st["gate"] is None else st["gate"].float()
    if case["act"]:
        gate = 1 / (1 + torch.exp(-gate))
    u = h + (n if gate is None else gate * n)
    scale = None if st["scale"] is None else st["scale"].float()
    s = (u if scale is None else u * scale).to(dt)
    out = [s]
    if case["pre"]:
        v, w2 = s.float(), st["w2"].float() + one
        r2 = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS)
        shat = v * r2
        out.append((shat * w2).to(dt))
    if not case["train"]:
        return out
    d, dw2 = st["ds"].float(), None
    if case["pre"]:
        dy = st["dy"].float()
        q = dy * w2
        d = d + r2 * (q - shat * (q * shat).mean(dim=1, keepdim=True))
        dw2 = (dy * shat).sum(dim=0)
    dscale = None if scale is None else (d * u).sum().reshape(1)
    if scale is not None:
        d = d * scale
    out.append(d.to(dt))
    dn = d if gate is None else d * gate
    q = dn * w1
    out.append((r1 * (q - xhat * (q * xhat).mean(dim=1, keepdim=True))).to(dt))
    if st["w1"].requires_grad:
        out.append((dn * xhat).sum(dim=0).to(st["w1"].dtype))
    if dw2 is not None and st["w2"].requires_grad:
        out.append(dw2.to(st["w2"].dtype))
    if gate is not None and st["gate"].requires_grad:
        dg = d * n
        if case["act"]:
            dg = dg * (gate * (1 - gate))
        dg = dg.sum(dim=0) if case["gate"] == "channel" else dg.sum(dim=1, keepdim=True) if case["gate"] == "token" else dg
        out.append(dg.to(st["gate"].dtype))
    if scale is not None and st["scale"].requires_grad:
        out.append(dscale.to(dt))
    return out


def _plain_clip(grads, most):
    norm = torch.sqrt(torch.stack([(t.float() ** 2).sum() for t in grads]).sum())
    c = (most / (norm + _CLIP_EPS)).clamp(max=1.0)
    return [norm, *((t.float() * c).to(t.dtype) for t in grads)]


# ------------------------------------------------------------------------------------------------ work, definition


def work(case):
    es = _BYTES[case["dtype"]]
    if case["op"] == "select":
        T, E, K = case["T"], case["E"], case["K"]
        return {"bytes": T * E * es * (2 if case["train"] else 1) + T * K * (16 if case["train"] else 12),
                "flops": T * E * (12 if case["train"] else 8)}
    if case["op"] == "norm":
        N = case["rows"] * case["cols"]
        extra = 1 if case["gate"] == "full" else 0
        tensors = 3 + case["pre"] + extra
        if case["train"]:      # the stream's gradient is its own input's where neither a norm nor a scale follows
            tensors += 2 + case["pre"] + extra + (1 if case["pre"] or case["scale"] != "none" else 0)
        return {"bytes": tensors * N * es, "flops": N * (40 if case["train"] else 12)}
    N = sum(math.prod(s) for s in _grad_shapes(case))
    return {"bytes": 2 * N * es, "flops": 3 * N}


def exact(case, seed):
    st = prepare(case, seed)
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    if case["op"] == "select":
        z = d(st["logits"]).requires_grad_(True)
        s = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, dim=1)
        c = s.detach().clone() if st["bias"] is None else s.detach() + d(st["bias"])
        G, T, E = case["groups"], *z.shape
        if G > 1:
            size = E // G
            rank = torch.stack([c[:, i * size:(i + 1) * size].sort(dim=1).values[:, -2:].sum(dim=1) for i in range(G)], dim=1)
            order = torch.argsort(-rank, dim=1, stable=True)
            dropped = torch.zeros_like(rank).scatter_(1, order[:, case["kept"]:], 1.0).bool()
            c[dropped.repeat_interleave(size, dim=1)] = -torch.inf
        ids = torch.argsort(-c, dim=1, stable=True)[:, :case["K"]]
        v = torch.take_along_dim(s, ids, dim=1)
        if case["renorm"]:
            v = v / (v.sum(dim=1, keepdim=True) + _TINY)
        v = 2.5 * v
        out = [v.detach(), None]
        if case["train"]:
            out.append(torch.autograd.grad(v, z, d(st["go"]))[0])
        return out
    if case["op"] == "norm":
        rows = {k: d(st[k]) for k in ("h", "x", "w1", "w2", "gate", "scale")}
        leaves = [k for k in rows if rows[k] is not None and st[k].requires_grad]
        for k in leaves:
            rows[k].requires_grad_(True)
        rms = lambda t, w: t / torch.sqrt(t.square().mean(dim=1, keepdim=True) + _EPS) * ((1 + w) if case["plus_one"] else w)  # noqa: E731
        y = rms(rows["x"], rows["w1"])
        if rows["gate"] is not None:
            y = y * (torch.sigmoid(rows["gate"]) if case["act"] else rows["gate"])
        s = rows["h"] + y
        if rows["scale"] is not None:
            s = s * rows["scale"]
        stored = s.detach().to(st["x"].dtype).double().requires_grad_(True)      # the stream's own rounding
        out = [stored.detach()]
        ds = d(st["ds"])
        late = []
        if case["pre"]:
            y = rms(stored, rows["w2"])
            out.append(y.detach())
            if case["train"]:
                late = torch.autograd.grad(y, [stored] + [rows["w2"]] * ("w2" in leaves), d(st["dy"]))
                ds = ds + late[0]
        if case["train"]:
            early = [k for k in leaves if k != "w2"]
            got = dict(zip(early, torch.autograd.grad(s, [rows[k] for k in early], ds)))
            if "w2" in leaves:
                got["w2"] = late[1]
            out += [got[k] for k in leaves]
        return out
    total = math.sqrt(sum(float(d(t).square().sum()) for t in st["grads"]))
    c = min(1.0, case["max"] / (total + _CLIP_EPS))
    return [torch.tensor(total, dtype=torch.float64, device=DEV), *(d(t) * c for t in st["grads"])]
