"""Operators of the training step around the MoE layer, as measurable cases: the router's balance loss with its counts and
gradient, layer norm with the gradients of its weights, and the orthogonalisation of the LoRA factors' updates.

  balance  ``smel.loss.balance_loss``: loss, tokens per expert and (train) the gradient of the router's logits
  ln       ``smel.norm.layernorm`` / ``add_layernorm``: rows, residual sum and (train) dx, dw, db
  ortho    ``smel.lora.orthogonalize``: one update, or the list of a layer's

Sizes are those of the two model shapes this package runs (hidden 2048 with 256 experts of 512, hidden 2816 with 128
experts of 704, top-8), its tests' token counts, and odd ones around them.
"""
import math
import os
import sys

import torch

_PKG = os.path.join(os.getcwd(), "smel-ft_amd")   # the package of the tree this runs in
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-5
_COEFFS = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_NORM_EPS = 1e-7
_COEF = 0.01

_MAX_ELEMS = 32749 * 2048        # of layer norm's rows
_MAX_PROBS = 32768 * 256         # of the router's logits
_MAX_UPDATE = 36 * 128 * 2816    # of the updates, and 128 times as many products


def _balance(T, E, K, dtype, train, seqs=0, masked=0.0):
    return {"op": "balance", "T": T, "E": E, "K": K, "dtype": dtype, "train": train, "seqs": seqs, "masked": masked}


def _ln(rows, cols, dtype, train, add=False, wide=False, bias=True):
    return {"op": "ln", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "add": add, "wide": wide, "bias": bias}


def _ortho(batch, m, n, dtype):
    return {"op": "ortho", "batch": batch, "m": m, "n": n, "dtype": dtype}


def listed():
    return [
        # the load of a short prompt's experts: forward only, latency counts
        {"name": "balance_eval_23", **_balance(23, 128, 8, "f32", False)},
        # a training step on one short sequence
        {"name": "balance_train_517", **_balance(517, 256, 8, "bf16", True)},
        # a packed row of several sequences with a padded tail and masked tokens: the loss of each sequence
        {"name": "balance_train_packed_4092", **_balance(4092, 256, 8, "bf16", True, seqs=9, masked=0.1)},
        # a large batch, logits in 32 bits
        {"name": "balance_train_32768", **_balance(32768, 256, 8, "f32", True)},
        # a few tokens at inference
        {"name": "ln_eval_23x2048", **_ln(23, 2048, "bf16", False)},
        # a short sequence, weights kept in 32 bits
        {"name": "ln_train_517x2816", **_ln(517, 2816, "f16", True, wide=True)},
        # the residual add and the norm after it, forward and backward, over a full packed row
        {"name": "add_ln_train_4092x2048", **_ln(4092, 2048, "bf16", True, add=True)},
        # odd sizes in 32 bits, rows that start at no 16-byte boundary
        {"name": "ln_train_1021x1733", **_ln(1021, 1733, "f32", True, bias=False)},
        # a large batch
        {"name": "ln_train_32749x2048", **_ln(32749, 2048, "bf16", True)},
        # one factor's update
        {"name": "ortho_16x2048", **_ortho(1, 16, 2048, "f32")},
        # every update of a layer's LoRA: twelve selected experts and the shared one, rank 16
        {"name": "ortho_layer_r16", "op": "ortho_layer", "k": 12, "H": 2048, "I": 512, "Is": 512, "r": 16, "dtype": "f32"},
        # factors of a high rank on three projections of twelve experts
        {"name": "ortho_36x128x2816", **_ortho(36, 128, 2816, "bf16")},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["balance", "ln", "ortho", "ortho", "ln", "balance", "ortho_layer"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.75
    if kind == "balance":
        E = rng.choice([8, 64, 128, 256, 512, rng.randint(2, 511)])
        T = _log(rng, 1, min(131072, _MAX_PROBS // E))
        seqs = 0 if rng.random() < 0.5 else _log(rng, 1, min(T, 4096))
        return _balance(T, E, rng.randint(1, max(1, min(E // 2, 16))), dtype, train, seqs, rng.choice([0.0, 0.0, 0.1, 0.9]))
    if kind == "ln":
        cols = rng.choice([64, 128, 512, 2048, 2816, 4096, 16384, _log(rng, 8, 16384), _log(rng, 8, 16384)])
        most = _MAX_ELEMS // cols // (2 if dtype == "f32" else 1)
        return _ln(_log(rng, 1, min(131072, most)), cols, dtype, train, rng.random() < 0.4, rng.random() < 0.3,
                   rng.random() < 0.8)
    if kind == "ortho":
        r = rng.choice([4, 8, 16, 32, 64, 128, _log(rng, 1, 128)])
        n = _log(rng, r, 16384)
        batch = _log(rng, 1, max(1, min(256, _MAX_UPDATE // (r * n * (2 if dtype == "f32" else 1)))))
        m, n = (r, n) if rng.random() < 0.5 else (n, r)
        return _ortho(batch, m, n, dtype)
    H, I = rng.choice([(2048, 512), (2816, 704)])
    r = rng.choice([4, 6, 8, 16, 32])
    return {"op": "ortho_layer", "k": rng.randint(1, 16), "H": H, "I": I, "Is": rng.choice([512, 2112]), "r": r,
            "dtype": dtype}


# ------------------------------------------------------------------------------------------------ inputs


def _seed(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _update(g, shape, dtype):
    """An update as training gives it: singular values spread over three decades (a few directions carry a factor's
    gradient), at the size of a gradient."""
    *lead, m, n = shape
    r = min(m, n)
    scale = torch.pow(10.0, -3.0 * torch.arange(r, device=DEV) / max(1, r - 1))
    left = torch.randn(*lead, r, r, generator=g, device=DEV) * scale
    x = left @ torch.randn(*lead, r, max(m, n), generator=g, device=DEV) * 1e-3
    return (x if m <= n else x.transpose(-1, -2)).to(dtype).contiguous()


def prepare(case, seed):
    g = _seed(seed)
    dt = _DT[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["op"] == "balance":
        T, E, K = case["T"], case["E"], case["K"]
        z = (1.5 * rand(T, E) + rand(E)).to(dt)
        st["topi"] = z.float().topk(K, dim=1).indices
        st["mask"] = st["offsets"] = None
        if case["masked"]:
            st["mask"] = torch.rand(T, generator=g, device=DEV) >= case["masked"]
            z[~st["mask"]] = float("nan")     # what a padded row holds is nobody's business
        if case["seqs"]:
            used = max(1, T - T // 50)        # a padded tail behind the last sequence
            cuts = torch.randint(0, used + 1, (case["seqs"] - 1,), generator=g, device=DEV).sort().values
            ends = torch.tensor([used], device=DEV)
            st["offsets"] = torch.cat((ends * 0, cuts, ends))
        st["logits"] = z.requires_grad_(case["train"])
        st["go"] = rand(()).abs() + 0.5
        return st
    if case["op"] == "ln":
        R, n = case["rows"], case["cols"]
        wdt = torch.float32 if case["wide"] else dt
        loud = 1 + 8 * (torch.rand(n, generator=g, device=DEV) > 0.99)     # channels of large values, as residual streams have
        row = lambda: ((rand(R, n) + 0.3 * rand(R, 1)) * loud).to(dt)  # noqa: E731
        t = case["train"]
        st["x"] = row().requires_grad_(t)
        st["h"] = row().requires_grad_(t) if case["add"] else None
        st["w"] = (1 + 0.2 * rand(n)).to(wdt).requires_grad_(t)
        st["b"] = (0.1 * rand(n)).to(wdt).requires_grad_(t) if case["bias"] else None
        st["dy"] = (1e-2 * rand(R, n)).to(dt) if t else None
        st["ds"] = (1e-2 * rand(R, n)).to(dt) if t and case["add"] else None
        return st
    if case["op"] == "ortho":
        st["g"] = [_update(g, (case["batch"], case["m"], case["n"]), dt)]
        return st
    st["g"] = [_update(g, s, dt) for s in _layer_shapes(case)]
    return st


def _layer_shapes(case):
    """A_gate, B_gate, A_up, B_up, A_down, B_down of the k experts and of the shared one."""
    k, r, H = case["k"], case["r"], case["H"]
    one = lambda lead, i: [(*lead, r, H), (*lead, i, r), (*lead, r, H), (*lead, i, r), (*lead, r, i), (*lead, H, r)]  # noqa: E731
    return one((k,), case["I"]) + one((), case["Is"])


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if case["op"] == "balance":
        return _run_balance(state, case)
    if case["op"] == "ln":
        return _run_ln(state, case)
    if own:
        from smel.lora import orthogonalize
        return orthogonalize(state["g"])
    return _plain_ortho(state["g"])


def _run_balance(st, case):
    if own:
        from smel.loss import balance_loss
        loss, counts = balance_loss(st["logits"], st["topi"], mask=st["mask"], offsets=st["offsets"], coef=_COEF)
        if not case["train"]:
            return [loss, counts]
        return [loss, counts, torch.autograd.grad(loss, st["logits"], st["go"])[0]]
    with torch.no_grad():
        return _plain_balance(st, case)


def _plain_balance(st, case):
    z, topi = st["logits"], st["topi"]
    T, E = z.shape
    K = topi.shape[1]
    if st["mask"] is None and st["offsets"] is None:      # one group of all tokens
        p = torch.softmax(z.float(), dim=1)
        counts = torch.zeros(E, dtype=torch.int64, device=DEV)
        counts.scatter_add_(0, topi.reshape(-1), torch.ones(T * K, dtype=torch.int64, device=DEV))
        v = counts.float() * (_COEF * E / (K * T * T))
        loss = (p.sum(dim=0) * v).sum()
        if not case["train"]:
            return [loss, counts]
        v = v * st["go"]
        return [loss, counts, (p * (v - (p * v).sum(dim=1, keepdim=True))).to(z.dtype)]
    valid = torch.ones(T, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]
    S = 1
    seq = torch.zeros(T, dtype=torch.int64, device=DEV)
    if st["offsets"] is not None:
        S = st["offsets"].numel() - 1
        seq = torch.searchsorted(st["offsets"], torch.arange(T, device=DEV), right=True) - 1
        valid = valid & (seq < S)
        seq = seq.clamp(max=S - 1)
    p = torch.softmax(torch.where(valid[:, None], z.float(), 0.0), dim=1) * valid[:, None]
    n = torch.zeros(S, dtype=torch.int64, device=DEV).scatter_add_(0, seq, valid.long())
    counts = torch.zeros(S * E, dtype=torch.int64, device=DEV)
    counts.scatter_add_(0, (seq[:, None] * E + topi).reshape(-1), valid[:, None].expand(T, K).reshape(-1).long())
    counts = counts.view(S, E)
    live = (n > 0).sum().clamp(min=1)
    size = n.clamp(min=1).float()[:, None]
    v = counts.float() * (_COEF * E / K) / (size * size * live)
    P = torch.zeros(S, E, device=DEV).index_add_(0, seq, p)
    loss = (P * v).sum()
    if st["offsets"] is None:
        counts = counts[0]
    if not case["train"]:
        return [loss, counts]
    vt = (v * st["go"])[seq]
    return [loss, counts, (p * (vt - (p * vt).sum(dim=1, keepdim=True))).to(z.dtype)]


def _run_ln(st, case):
    x, h, w, b = st["x"], st["h"], st["w"], st["b"]
    if own:
        from smel.norm import add_layernorm, layernorm
        params = [t for t in (h, x, w, b) if t is not None]
        if case["add"]:
            s, y = add_layernorm(h, x, w, b, _EPS)
            if not case["train"]:
                return [s, y]
            return [s, y, *torch.autograd.grad((s, y), params, (st["ds"], st["dy"]))]
        y = layernorm(x, w, b, _EPS)
        return [y] if not case["train"] else [y, *torch.autograd.grad(y, params, st["dy"])]
    with torch.no_grad():
        return _plain_ln(st, case)


def _plain_ln(st, case):
    x, h, w, b = st["x"], st["h"], st["w"].float(), st["b"]
    out = []
    if case["add"]:
        x = (h.float() + x.float()).to(x.dtype)
        out.append(x)
    v = x.float()
    v = v - v.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS)
    xhat = v * rstd
    y = xhat * w
    out.append((y if b is None else y + b.float()).to(x.dtype))
    if not case["train"]:
        return out
    dy = st["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True))
    if case["add"]:
        dx = dx + st["ds"].float()
    dx = dx.to(x.dtype)
    out += [dx, dx] if case["add"] else [dx]
    out.append((dy * xhat).sum(dim=0).to(st["w"].dtype))
    if b is not None:
        out.append(dy.sum(dim=0).to(b.dtype))
    return out


def _iterate(x):
    """The Newton-Schulz products on [B, r, n] matrices, r <= n."""
    a, b, c = _COEFFS
    x = x / (torch.sqrt((x * x).sum(dim=(1, 2), keepdim=True)) + _NORM_EPS)
    for _ in range(_STEPS):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x


def _plain_ortho(gs):
    """Updates of one shape (after the longer side is laid along the columns) go through the products as one batch."""
    flat = [t.reshape(-1, *t.shape[-2:]).float() for t in gs]
    flat = [t if t.shape[1] <= t.shape[2] else t.transpose(1, 2) for t in flat]
    groups = {}
    for i, t in enumerate(flat):
        groups.setdefault(t.shape[1:], []).append(i)
    out = [None] * len(gs)
    for ids in groups.values():
        x = torch.cat([flat[i] for i in ids]) if len(ids) > 1 else flat[ids[0]]
        parts = _iterate(x).split([flat[i].shape[0] for i in ids])
        for i, y in zip(ids, parts):
            m, n = gs[i].shape[-2:]
            out[i] = (y if m <= n else y.transpose(1, 2)).to(gs[i].dtype).reshape(gs[i].shape)
    return out


# ------------------------------------------------------------------------------------------------ work, definition


def work(case):
    es = _BYTES[case["dtype"]]
    if case["op"] == "balance":
        T, E, K, S = case["T"], case["E"], case["K"], max(1, case["seqs"])
        probs = T * E * es
        return {"bytes": probs * (2 if case["train"] else 1) + T * K * 8 + (T if case["masked"] else 0) + S * E * 8,
                "flops": T * E * (10 if case["train"] else 4)}
    if case["op"] == "ln":
        N = case["rows"] * case["cols"]
        tensors = (4 if case["add"] else 2) + ((3 if case["add"] else 2) if case["train"] else 0)
        return {"bytes": tensors * N * es, "flops": N * (20 if case["train"] else 8)}
    shapes = [(case["batch"], case["m"], case["n"])] if case["op"] == "ortho" else _layer_shapes(case)
    sides = [(math.prod(s[:-2]), min(s[-2:]), max(s[-2:])) for s in shapes]
    # the Gram matrix's half, the square of the short side in every step, and the last product
    return {"bytes": sum(2 * b * r * n * es for b, r, n in sides),
            "flops": sum(b * (r * r * n * 3 + (4 * _STEPS - 3) * r ** 3) for b, r, n in sides)}


def exact(case, seed):
    st = prepare(case, seed)
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    if case["op"] == "balance":
        z, topi = d(st["logits"]), st["topi"]
        T, E = z.shape
        K = topi.shape[1]
        keep = torch.ones(T, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"].clone()
        seq = torch.zeros(T, dtype=torch.int64, device=DEV)
        S = 1
        if st["offsets"] is not None:
            off = st["offsets"]
            S = off.numel() - 1
            lens = off[1:] - off[:-1]
            seq = torch.full((T,), S, dtype=torch.int64, device=DEV)
            seq[:int(off[-1])] = torch.repeat_interleave(torch.arange(S, device=DEV), lens)
            keep &= seq < S
        rows = keep.nonzero().flatten()
        zz = z[rows].requires_grad_(True)
        sq = seq[rows]
        p = torch.exp(zz - torch.logsumexp(zz, dim=1, keepdim=True))
        n = torch.bincount(sq, minlength=S)
        counts = torch.bincount((sq[:, None] * E + topi[rows]).flatten(), minlength=S * E).view(S, E)
        full = n > 0
        P = torch.zeros(S, E, dtype=torch.float64, device=DEV).index_add(0, sq, p)
        share = counts.double() / (K * n.clamp(min=1)[:, None])
        mean = P / n.clamp(min=1)[:, None]
        loss = _COEF * E * (share * mean).sum() / max(1, int(full.sum()))
        out = [loss.detach(), None]
        if case["train"]:
            gz = torch.zeros_like(z)
            if rows.numel():
                gz[rows] = torch.autograd.grad(loss, zz)[0] * st["go"].double()
            out.append(gz)
        return out
    if case["op"] == "ln":
        x, w, b, h = d(st["x"]), d(st["w"]), d(st["b"]), d(st["h"])
        out = []
        if case["add"]:
            x = (st["h"].detach().double() + x).to(st["x"].dtype)     # the stream's own rounding
            out.append(x.double())
            x = x.double()
        leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = w * (x - mean) / torch.sqrt(var + _EPS)
        y = y if b is None else y + b
        out.append(y.detach())
        if case["train"]:
            gr = list(torch.autograd.grad(y, leaves, d(st["dy"])))
            if case["add"]:
                gr[0] = gr[0] + d(st["ds"])
                gr.insert(0, gr[0])
            out += gr
        return out
    a, b, c = _COEFFS
    out = []
    for t in st["g"]:
        x = d(t)
        wide = x.shape[-2] <= x.shape[-1]
        x = x / (torch.linalg.matrix_norm(x)[..., None, None] + _NORM_EPS)
        for _ in range(_STEPS):
            s = torch.matmul(x, x.mT.contiguous()) if wide else torch.matmul(x.mT.contiguous(), x)
            q = a * torch.eye(s.shape[-1], dtype=s.dtype, device=DEV) + b * s + c * torch.matmul(s, s)
            x = torch.matmul(q, x) if wide else torch.matmul(x, q)
        out.append(x)
    return out
