"""LoRA parameter sets of the selected routed experts and of the shared / dense MLP: the adapter format of the
reference's smel/lora.py (classes ExpertsLoRA, MLPLoRA, LayerLoRA, BlockLoRA; parameters A_gate, B_gate, A_up,
B_up, A_down, B_down in that order, fp32, A [.., r, in] uniform in +-1/sqrt(in) (kaiming_uniform with a = sqrt(5)),
B [.., out, r] zero), so adapters written by either load into the other.

The MoE layer never multiplies these factors in Python: smel.moe lays them out as a 32-wide K-extension of the
grouped-GEMM kernels. ``lora_linear`` / ``lora_gate_up`` are the dense helpers of the API (torch ops);
``orthogonalize`` makes the factors' updates orthogonal on the GPU (include/smel_ortho.h), ``clip_grads`` scales the gradients
down to a global norm (include/smel_clip.h).
"""
from __future__ import annotations

import json
import math
import os
from array import array

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib

_PROJ = ("gate", "up", "down")


def _uniform_fan_in(a: torch.Tensor) -> torch.Tensor:
    """Every [r, in] matrix of ``a`` uniform in +-1/sqrt(in): kaiming_uniform_ with a = sqrt(5) gives
    gain sqrt(2 / (1 + 5)) and bound gain * sqrt(3 / in), which is that."""
    bound = 1.0 / math.sqrt(a.shape[-1])
    with torch.no_grad():
        for m in a.view(-1, *a.shape[-2:]):
            m.uniform_(-bound, bound)
    return a


class _LoRASet(nn.Module):
    """The six factors of a gated MLP's LoRA, with ``lead`` leading dims (() for one MLP, (k,) for k experts):
    A_p [*lead, r, in_p], B_p [*lead, out_p, r] for p = gate, up (in = hidden, out = inter) and down (in = inter,
    out = hidden); scale = alpha / r."""

    def __init__(self, lead: tuple, hidden: int, inter: int, r: int, alpha: float):
        super().__init__()
        self.r, self.alpha, self.scale = r, alpha, alpha / r
        io = {"gate": (hidden, inter), "up": (hidden, inter), "down": (inter, hidden)}
        for p in _PROJ:
            fan_in, fan_out = io[p]
            setattr(self, f"A_{p}", nn.Parameter(_uniform_fan_in(torch.empty(*lead, r, fan_in))))
            setattr(self, f"B_{p}", nn.Parameter(torch.zeros(*lead, fan_out, r)))

    def _deltas(self, idx):
        """(scale B_p) A_p for the three projections at index ``idx`` of the leading dims (fp32; B is scaled before
        the product, the order of smel/lora.py:31-36, so merged weights round as the reference's)."""
        def one(p):
            return torch.matmul(getattr(self, f"B_{p}")[idx].float() * self.scale, getattr(self, f"A_{p}")[idx].float())
        return tuple(one(p) for p in _PROJ)


class ExpertsLoRA(_LoRASet):
    """LoRA of k selected experts of one layer (smel/lora.py:14-36): slot j belongs to expert ``expert_ids[j]``."""

    def __init__(self, expert_ids, hidden: int, inter: int, r: int = 16, alpha: float = 32.0):
        ids = [int(e) for e in expert_ids]
        super().__init__((len(ids),), hidden, inter, r, alpha)
        self.register_buffer("expert_ids", torch.tensor(ids, dtype=torch.long), persistent=True)

    def delta(self, j: int):
        """Dense weight deltas of slot j: (d_gate [I, H], d_up [I, H], d_down [H, I]), fp32."""
        return self._deltas(j)


class MLPLoRA(_LoRASet):
    """LoRA of one gated MLP: the shared expert, or Gemma 4's dense MLP (smel/lora.py:39-58)."""

    def __init__(self, hidden: int, inter: int, r: int = 16, alpha: float = 32.0):
        super().__init__((), hidden, inter, r, alpha)

    def delta(self):
        return self._deltas(())


def _add_low_rank(y, xa, B, scale):
    """y + scale (xa B^T), B cast to the rows' dtype. For rows given as a matrix, one addmm: the low-rank product's
    sum, its scaling and the add round once (the reference's epilogue form); other shapes scale and add the rounded
    product, as the reference does for them."""
    bt = B.to(xa.dtype).t()
    if xa.dim() == 2:
        return torch.addmm(y, xa, bt, alpha=scale)
    return y + scale * (xa @ bt)


def lora_linear(x, w, A, B, scale):
    """x w^T + scale (x A^T) B^T with the LoRA factors in x's dtype (smel/lora.py:61-69)."""
    y = x @ w.t()
    if A is None:
        return y
    return _add_low_rank(y, x @ A.to(x.dtype).t(), B, scale)


def lora_gate_up(x, w_gate_up, A_gate, B_gate, A_up, B_up, scale):
    """(gate, up) of a gated MLP from its stacked [2I, H] weight (smel/lora.py:72-83): one base GEMM over the stacked
    weight and one rank-2r projection x [A_gate; A_up]^T, whose two halves go through B_gate and B_up into the gate
    and up halves. Rows of any leading shape (flattened to a matrix for the products)."""
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    I = w_gate_up.shape[0] // 2
    base = x2 @ w_gate_up.t()
    g, u = base[:, :I], base[:, I:]
    if A_gate is not None:
        r = A_gate.shape[0]
        xa = x2 @ torch.cat((A_gate, A_up)).to(x.dtype).t()
        g, u = _add_low_rank(g, xa[:, :r], B_gate, scale), _add_low_rank(u, xa[:, r:], B_up, scale)
    return g.reshape(*lead, I), u.reshape(*lead, I)


# ------------------------------------------------------------------------------------------------ updates

_ORTHO_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
ORTHO_MAX_RANK = 128   # of the shorter side
# a smel_ortho_job (include/smel_ortho.h) as orthogonalize packs it: 8 bytes each
_ORTHO_JOB = ("x", "y", "batch", "rows", "cols", "x_batch", "x_row", "x_col", "dtype")


def _ortho_operand(t: torch.Tensor):
    """t [..., m, n] as [batch, m, n] with unit stride along one side: a view where there is one, else a copy."""
    if t.dim() > 3:
        try:
            t = t.view(-1, *t.shape[-2:])
        except RuntimeError:
            t = t.reshape(-1, *t.shape[-2:]).contiguous()
    elif t.dim() == 2:
        t = t.unsqueeze(0)
    _, m, n = t.shape
    if not (n == 1 or t.stride(2) == 1 or m == 1 or t.stride(1) == 1):
        t = t.contiguous()
    return t


def orthogonalize(update, steps: int = 5, coeffs=(3.4445, -4.7750, 2.0315), eps: float = 1e-7):
    """Orthogonalised updates by Newton-Schulz products, as the Muon optimiser makes them of its momentum: for every matrix
    G of the last two dimensions, X = G / (|G|_F + eps), then ``steps`` times

        X <- a X + b (X X^T) X + c (X X^T)^2 X

    which moves every singular value towards 1 and keeps the singular vectors. ``update``: a tensor [..., m, n] (bf16,
    fp16, fp32; a factor's gradient or momentum) or a sequence of them, e.g. every factor's of a block, which go through
    few launches together; the shorter side (a LoRA's rank) is at most 128. Returns the same shapes and dtypes,
    contiguous, without gradients. The products run in 64 bits, up to 6 steps of these coefficients on the rank's r x r matrices
    alone, so small singular values keep their directions; 7 to 12 steps take two such passes, more a pass over the update for
    each (include/smel_ortho.h)."""
    single = isinstance(update, torch.Tensor)
    ts = (update,) if single else tuple(update)
    a, b, c = (float(v) for v in coeffs)
    if not 0 <= int(steps) <= 64:
        raise ValueError(f"orthogonalize takes 0 to 64 steps, got {steps}")
    if not eps >= 0:
        raise ValueError(f"orthogonalize: eps must not be negative, got {eps}")
    if not ts:
        return []
    if not ts[0].is_cuda:
        _lib.one_device(ts[0])
    jobs, outs, keep = array("q"), [], []
    add, dev = jobs.extend, ts[0].device
    with torch.no_grad(), _lib.on_device_of(ts[0]):
        for t in ts:     # a layer has a dozen: what each costs here is the call's time
            shape = t.shape
            code = _ORTHO_DTYPES.get(t.dtype)
            if code is None or len(shape) < 2:
                raise ValueError(f"orthogonalize takes bf16, fp16 or fp32 matrices, got {tuple(shape)} {t.dtype}")
            rows, cols = shape[-2], shape[-1]
            if rows > ORTHO_MAX_RANK and cols > ORTHO_MAX_RANK:
                raise ValueError(f"orthogonalize takes matrices whose shorter side is at most {ORTHO_MAX_RANK}, got "
                                 f"{tuple(shape)}")
            if t.device != dev:
                _lib.one_device(ts[0], t)
            values, size = t.numel(), rows * cols
            if t.is_contiguous():
                y = torch.empty_like(t)
                if values:
                    add((t.data_ptr(), y.data_ptr(), values // size, rows, cols, size, cols, 1, code))
            else:
                y = t.new_empty(shape)
                if values:
                    x = _ortho_operand(t)
                    keep.append(x)
                    add((x.data_ptr(), y.data_ptr(), *x.shape, *x.stride(), code))
            outs.append(y)
        n = len(jobs) // len(_ORTHO_JOB)
        addr = jobs.buffer_info()[0]
        need = _lib.load().smel_orthogonalize_ws(addr, n, int(steps), a)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        _lib.call("smel_orthogonalize", addr, n, int(steps), a, b, c, float(eps), ws.data_ptr(), need, _lib.stream())
    return outs[0] if single else outs


# ------------------------------------------------------------------------------------------------ the gradients' norm

_CLIP_JOB = ("in", "out", "n", "dtype")      # a smel_clip_job (include/smel_clip.h): 8 bytes each
_NORM_TYPES = {2.0: 0, math.inf: 1}


def _flat(t: torch.Tensor) -> bool:
    """Whether t's values fill t.numel() elements of memory from its first on, in whatever order of dimensions."""
    at = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _clip_call(grads, max_norm, norm_type, eps, inplace):
    """(the scaled tensors, the norm) of grads; max_norm None: the norm alone."""
    what = "grad_norm" if max_norm is None else "clip_grads"
    ts = (grads,) if isinstance(grads, torch.Tensor) else tuple(grads)
    kind = _NORM_TYPES.get(float(norm_type))
    if kind is None:
        raise ValueError(f"{what} takes norm_type 2 or inf, got {norm_type}")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"{what}: max_norm must not be negative, got {max_norm}")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    first = next((t for t in ts if t is not None), None)
    if first is None:
        return list(ts), torch.zeros((), dtype=torch.float32)
    if not first.is_cuda:
        _lib.one_device(first)
    _lib.refuse_tangents(what, ts)
    jobs, outs, keep, back = array("q"), [], [], []
    add, put, codes, index, like = jobs.extend, outs.append, _ORTHO_DTYPES, first.get_device(), torch.empty_like
    copies = max_norm is not None and not inplace
    with torch.no_grad(), _lib.on_device_of(first):
        for t in ts:     # a block has hundreds: what each costs here is the call's time
            if t is None:
                put(None)
                continue
            code = codes.get(t.dtype)
            if code is None or t.layout is not torch.strided:
                raise ValueError(f"{what} takes bf16, fp16 or fp32 tensors, got {t.dtype} {t.layout}")
            if t.get_device() != index:
                _lib.one_device(first, t)
            x = t
            if not t.is_contiguous() and not _flat(t):
                if inplace and 0 in t.stride() and any(st == 0 and size > 1 for st, size in zip(t.stride(), t.shape)):
                    raise ValueError(f"{what} in place: a tensor of shape {tuple(t.shape)} and strides {t.stride()} overlaps itself")
                x = t.contiguous()
                keep.append(x)
                if inplace:
                    back.append((t, x))
            at = x.data_ptr()
            if copies:
                x = like(x)
                add((at, x.data_ptr(), x.numel(), code))
                put(x)
            else:
                add((at, at, x.numel(), code))
                put(t)
        n = len(jobs) // len(_CLIP_JOB)
        addr = jobs.buffer_info()[0]
        need = _lib.load().smel_clip_ws(addr, n)
        ws, norm = first.new_empty(need, dtype=torch.uint8), first.new_empty((), dtype=torch.float32)
        if max_norm is not None:
            _lib.call("smel_clip_grads", addr, n, kind, max_norm, float(eps), norm.data_ptr(), ws.data_ptr(), need,
                      _lib.stream())
        else:
            _lib.call("smel_grad_norm", addr, n, kind, norm.data_ptr(), ws.data_ptr(), need, _lib.stream())
        for t, x in back:
            t.copy_(x)
        if inplace:     # what autograd kept of them is out of date
            torch.autograd.graph.increment_version([t for t in ts if t is not None])
    return outs, norm


def grad_norm(grads, norm_type: float = 2.0):
    """The norm of all values of all tensors together (an fp32 scalar on their GPU, on the host where there is no tensor; a constant to
    autograd; no host synchronisation): norm_type 2 (sums in 64 bits) or inf (the largest magnitude). ``grads``: a tensor or a sequence
    (bf16, fp16, fp32; None entries are passed over). A NaN anywhere gives NaN."""
    return _clip_call(grads, None, norm_type, 0.0, False)[1]


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, eps: float = 1e-6):
    """(clipped, norm): every tensor times min(1, max_norm / (norm + eps)) with ``norm`` the norm of all of them together, as
    ``grad_norm`` gives it; new tensors of the same shapes and dtypes, without gradients (None stays None), one tensor for one tensor.
    A norm that is infinite or NaN gives what the product with that factor gives."""
    outs, norm = _clip_call(grads, float(max_norm), norm_type, eps, False)
    return (outs[0] if isinstance(grads, torch.Tensor) else outs), norm


def clip_grads_(grads, max_norm: float, norm_type: float = 2.0, eps: float = 1e-6):
    """``clip_grads`` in place; returns the norm before. Dense tensors that are within the norm already are not written. The tensors must
    not overlap (dense ones that do, one given twice among them, are refused before anything is written; strided ones go through
    copies, and get their own values back where the factor is 1).
    Autograd sees the change, as of any in-place operation."""
    return _clip_call(grads, float(max_norm), norm_type, eps, True)[1]


class LayerLoRA(nn.Module):
    """The LoRA of one layer: ``experts`` (ExpertsLoRA or None) and ``shared`` (MLPLoRA or None)."""

    def __init__(self, experts: ExpertsLoRA | None, shared: MLPLoRA | None):
        super().__init__()
        self.experts = experts
        self.shared = shared


class BlockLoRA(nn.Module):
    """The LoRA of a block of layers, keyed by absolute layer index (smel/lora.py:93-125)."""

    def __init__(self, layers: dict):
        super().__init__()
        self.layers = nn.ModuleDict({str(k): v for k, v in layers.items()})

    def get(self, l: int):
        key = str(l)
        return self.layers[key] if key in self.layers else None

    @classmethod
    def build(cls, selection: dict, hidden: int, inter: int, shared_inter: int, r: int, alpha: float,
              shared: bool = True):
        """selection {layer: [expert ids]} -> one LayerLoRA per layer (no ExpertsLoRA for an empty selection)."""
        def layer(ids):
            ex = ExpertsLoRA(ids, hidden, inter, r, alpha) if len(ids) else None
            return LayerLoRA(ex, MLPLoRA(hidden, shared_inter, r, alpha) if shared else None)
        return cls({int(l): layer(ids) for l, ids in selection.items()})

    @classmethod
    def load(cls, path, dims, device="cuda"):
        """An adapter folder (adapter_config.json + adapter.safetensors, the reference trainer's output format) ->
        (BlockLoRA on ``device``, the config dict). ``dims`` supplies hidden, moe_inter and shared_inter."""
        from safetensors.torch import load_file
        with open(os.path.join(path, "adapter_config.json")) as f:
            meta = json.load(f)
        sel = {int(l): ids for l, ids in meta["experts"].items()}
        block = cls.build(sel, dims.hidden, dims.moe_inter, dims.shared_inter, meta["r"], meta["alpha"],
                          shared=meta["shared_lora"])
        block.load_state_dict(load_file(os.path.join(path, "adapter.safetensors")))
        return block.to(device), meta
