"""RMSNorm family of the frozen layers around the MoE block, and layer norm with trained weights, on the HIP kernels of
libsmel_moe.so (include/smel_norm.h): one launch forward, one backward (with trained weights: two, the second adds up the
weights' gradients).

  rmsnorm(x, w, eps, plus_one)          y = x * rstd * (1 + w) (Qwen3.5/3.6), x * rstd * w (Gemma 4), x * rstd (w None)
  add_rmsnorm(h, x, w, eps, plus_one)   s = h + x (the residual add), y = rmsnorm(s)
  gated_rmsnorm(x, z, w, eps)           y = w * norm(x) * silu(z)  (output norm of Gated DeltaNet)
  layernorm(x, w, b, eps)               y = (x - mean) * rstd * w + b
  add_layernorm(h, x, w, b, eps)        s = h + x, y = layernorm(s)
  post_rmsnorm(h, x, w, eps, plus_one, gate, gate_act, scale)             s = scale (h + gate rmsnorm(x)): behind a block
  sandwich_rmsnorm(h, x, w_post, w_pre, eps, plus_one, gate, gate_act, scale)    the same s, and y = rmsnorm(s) before the next

Of the RMSNorm functions the API is the reference's smel/norm.py:252-275 (``supported``, ``ENABLED``, ``MAX_COLS`` and the three functions,
same arguments and return values). Their weights are frozen, so backward gives dx (and dz) only, as there.
fp32 math with the reference's rounding points (the residual sum rounded to the stream's dtype, the gated norm's
``n`` and ``w n`` rounded); saved for backward: the rows the norm read and one fp32 rstd per row:

    xhat = x * rstd,  g = dy * w',  dx = rstd * (g - xhat * mean(g * xhat))     (w' = 1 + w, w or 1)

Structure: one autograd node (``_NormFn``) serves the three kinds; a kind is a forward launch and a backward launch
over [rows, n] operands. There is no fallback: without the library every call raises. ``supported`` answers the same
question as the reference's (16-bit rows on the GPU, frozen contiguous weights of the rows' dtype, at most MAX_COLS
columns), so a caller that routes other cases to its own torch code keeps doing so.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

MAX_COLS = 16384
ENABLED = True   # callers switch the kernels off to compare with their torch code

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_RMS, _ADD, _GATED = "rms", "add", "gated"


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype not in _DTYPES:
        raise ValueError(f"smel norms take bf16 or fp16 rows, got {t.dtype}")
    return _DTYPES[t.dtype]


def _check_weight(w, x):
    if w is not None and (w.dtype != x.dtype or w.numel() != x.shape[-1] or not w.is_contiguous()):
        raise ValueError(f"norm weight must be a contiguous [{x.shape[-1]}] tensor of {x.dtype}")


def _row_layout(x: torch.Tensor):
    """(rows [R, n] with unit column stride, row pitch in elements) of the plain norm's input: a view of x when its
    rows are evenly spaced without overlap (a column slice of a wider projection is read in place; smel/norm.py
    reads such views the same way, :148-154), else a packed copy."""
    n = x.shape[-1]
    try:
        rows = x.view(-1, n)
    except RuntimeError:          # leading dims not flattenable into one stride
        rows = None
    if rows is None or rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < n):
        rows = x.reshape(-1, n).contiguous()
    return rows, (rows.stride(0) if rows.shape[0] > 1 else n)


def _packed(t: torch.Tensor) -> torch.Tensor:
    """t as a packed [R, n] tensor (a view when t already is one)."""
    return t.reshape(-1, t.shape[-1]).contiguous()


class _NormFn(torch.autograd.Function):
    """forward(kind, eps, w_mode, w, a, b): kind "rms" (a = x), "add" (a = h, b = x; returns s and y) or "gated"
    (a = x, b = z). w_mode: 0 no weight, 1 w, 2 (1 + w)."""

    @staticmethod
    def forward(ctx, kind, eps, w_mode, w, a, b):
        _lib.require_device(a, b, w)
        _check_weight(w, a)
        dt, stream, p = _dtype_code(a), _lib.stream(), _lib.ptr
        ctx.kind, ctx.w_mode = kind, w_mode
        ctx.set_materialize_grads(False)
        if kind == _RMS:
            x2, pitch = _row_layout(a)
            R, n = x2.shape
            y = torch.empty(a.shape, device=a.device, dtype=a.dtype)
            rstd = torch.empty(R, device=a.device, dtype=torch.float32)
            _lib.call("smel_rmsnorm_fwd", p(x2), R, n, pitch, p(w), w_mode, float(eps), dt, p(y), p(rstd), stream)
            ctx.save_for_backward(x2, w, rstd)
            ctx.pitch, ctx.shapes = pitch, (a.shape,)
            return y
        a2, b2 = _packed(a), _packed(b)
        R, n = a2.shape
        rstd = torch.empty(R, device=a.device, dtype=torch.float32)
        y = torch.empty(a.shape, device=a.device, dtype=a.dtype)
        if kind == _ADD:
            s = torch.empty(a.shape, device=a.device, dtype=a.dtype)
            _lib.call("smel_add_rmsnorm_fwd", p(a2), p(b2), R, n, p(w), w_mode, float(eps), dt, p(s), p(y), p(rstd),
                      stream)
            ctx.save_for_backward(s, w, rstd)       # the norm's input is the rounded sum
            return s, y
        _lib.call("smel_gated_rmsnorm_fwd", p(a2), p(b2), R, n, p(w), float(eps), dt, p(y), p(rstd), stream)
        ctx.save_for_backward(a2, b2, w, rstd)
        ctx.shapes = (a.shape, b.shape)
        return y

    @staticmethod
    @_lib.once
    def backward(ctx, *grads):
        p, stream = _lib.ptr, _lib.stream()
        if ctx.kind == _RMS:
            x2, w, rstd = ctx.saved_tensors
            dy = grads[0]
            if dy is None:
                return None, None, None, None, None, None
            R, n = x2.shape
            dx = torch.empty(ctx.shapes[0], device=x2.device, dtype=x2.dtype)
            _lib.call("smel_rmsnorm_bwd", p(_packed(dy)), p(x2), R, n, ctx.pitch, p(w), ctx.w_mode, p(rstd), None,
                      _dtype_code(x2), p(dx), stream)
            return None, None, None, None, dx, None
        if ctx.kind == _ADD:
            # s feeds the norm and the residual stream: both inputs of the add get ds + the norm's dx (summed in
            # fp32 before one rounding); without a gradient through y it is ds alone
            s, w, rstd = ctx.saved_tensors
            ds, dy = grads
            if dy is None:
                return None, None, None, None, ds, ds
            s2 = s.reshape(-1, s.shape[-1])
            R, n = s2.shape
            d = torch.empty(s.shape, device=s.device, dtype=s.dtype)
            _lib.call("smel_rmsnorm_bwd", p(_packed(dy)), p(s2), R, n, n, p(w), ctx.w_mode, p(rstd),
                      p(_packed(ds)) if ds is not None else None, _dtype_code(s), p(d), stream)
            return None, None, None, None, d, d
        x2, z2, w, rstd = ctx.saved_tensors
        dout = grads[0]
        if dout is None:
            return None, None, None, None, None, None
        R, n = x2.shape
        dx = torch.empty(ctx.shapes[0], device=x2.device, dtype=x2.dtype)
        dz = torch.empty(ctx.shapes[1], device=z2.device, dtype=z2.dtype)
        _lib.call("smel_gated_rmsnorm_bwd", p(_packed(dout)), p(x2), p(z2), R, n, p(w), p(rstd), _dtype_code(x2),
                  p(dx), p(dz), stream)
        return None, None, None, None, dx, dz


def _w_mode(w, plus_one: bool) -> int:
    return 0 if w is None else (2 if plus_one else 1)


def supported(x, *weights):
    """Whether the kernels take this call: a GPU bf16/fp16 input of at most MAX_COLS columns whose norm weights are
    frozen, contiguous, of the input's dtype and shape [n_cols] (smel/norm.py:252-259)."""
    if not ENABLED or not x.is_cuda or x.dtype not in _DTYPES or x.shape[-1] > MAX_COLS:
        return False
    n = x.shape[-1]

    def fits(w):
        return w is None or (w.dtype == x.dtype and tuple(w.shape) == (n,) and w.is_contiguous()
                             and not w.requires_grad)
    return all(fits(w) for w in weights)


def rmsnorm(x, w, eps, plus_one):
    return _NormFn.apply(_RMS, eps, _w_mode(w, plus_one), w, x, None)


def add_rmsnorm(h, x, w, eps, plus_one):
    """(h + x, rmsnorm(h + x)): the residual add and the norm after it."""
    return _NormFn.apply(_ADD, eps, 2 if plus_one else 1, w, h, x)


def gated_rmsnorm(x, z, w, eps):
    return _NormFn.apply(_GATED, eps, 1, w, x, z)


# ------------------------------------------------------------------------------------------------ layer norm

_LN_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _ln_refuse(x, h, w, b):
    """Raises what is wrong with the call."""
    _lib.one_device(x, h, w, b)
    if x.dtype not in _LN_DTYPES:
        raise ValueError(f"layer norm takes bf16, fp16 or fp32 rows, got {x.dtype}")
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"layer norm takes rows of 1 to {MAX_COLS} columns, got shape {tuple(x.shape)}")
    if h is not None and (h.shape != x.shape or h.dtype != x.dtype):
        raise ValueError(f"the two addends differ: {tuple(h.shape)} {h.dtype} and {tuple(x.shape)} {x.dtype}")
    for t in (w, b):
        if t is not None and (t.dtype not in (x.dtype, torch.float32) or tuple(t.shape) != (x.shape[-1],)
                              or not t.is_contiguous()):
            raise ValueError(f"layer norm weights must be contiguous [{x.shape[-1]}] tensors of {x.dtype} or float32")
    raise ValueError(f"layer norm's weight is {w.dtype} and its bias {b.dtype}")


def _ln_check(x, h, w, b) -> tuple:
    """(columns, the rows' type code, the weights' type code) of a call that the kernels take; a small norm is the host's
    time, so each tensor is looked at once."""
    dt = _LN_DTYPES.get(x.dtype)
    if dt is None or x.dim() == 0 or not x.is_cuda:
        _ln_refuse(x, h, w, b)
    n, dev = x.shape[-1], x.device
    ok = 1 <= n <= MAX_COLS
    if h is not None:
        ok = ok and h.shape == x.shape and h.dtype is x.dtype and h.device == dev
    wd = None
    for t in (w, b):
        if t is not None:
            ok = ok and (wd is None or t.dtype is wd) and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() \
                and t.device == dev
            wd = t.dtype
    wt = dt if wd is None or wd is x.dtype else 2
    if not ok or (wt == 2 and wd is not None and wd is not torch.float32):
        _ln_refuse(x, h, w, b)
    return n, dt, wt


def _rows_of(x, n: int):
    """(rows with unit column stride, their count, their pitch): x itself where it is packed."""
    if x.is_contiguous():
        return x, x.numel() // n, n
    rows, pitch = _row_layout(x)
    return rows, rows.shape[0], pitch


def _ln_forward(x, h, w, b, eps, n, dt, wt):
    """(rows the norm read, their count, s or None, y, stats)."""
    if h is None:
        x2, R, pitch = _rows_of(x, n)
        h2 = s = sp = None
    else:
        x2, h2 = x.contiguous(), h.contiguous()
        R, pitch = x2.numel() // n, n
        s = torch.empty_like(x2)
        sp = s.data_ptr()
    y = torch.empty_like(x2) if x2.is_contiguous() and x2.shape == x.shape else x.new_empty(x.shape)
    stats = x.new_empty(2 * R, dtype=torch.float32)     # a row's mean and rstd
    p = _lib.ptr
    _lib.call("smel_layernorm_fwd", x2.data_ptr(), p(h2), R, n, pitch, p(w), p(b), eps, dt, wt, sp, y.data_ptr(),
              stats.data_ptr(), _lib.stream())
    return (x2 if h is None else s), R, s, y, stats


def _ln_backward(ctx, *grads):
    """dx (the same for both addends), dw and db, each only where it is asked for."""
    rows, w, stats = ctx.saved_tensors
    add, n, R, dt, wt, shape, wdt = ctx.call
    pitch = n if rows.is_contiguous() else rows.stride(0)     # of what comes back: hooks on saved tensors may repack it
    ds, dy = grads if add else (None, grads[0])
    if dy is None:      # the sum alone was used (or nothing)
        return ds, ds if add else None, None, None, None, None
    nx, nh, nw, nb = ctx.needs_input_grad[:4]
    want_x = nx or nh
    p = _lib.ptr
    dy2 = dy.contiguous()
    ds2 = ds.contiguous() if ds is not None and want_x else None
    dx = rows.new_empty(shape) if want_x else None
    dw = rows.new_empty(n, dtype=wdt) if nw else None
    db = rows.new_empty(n, dtype=wdt) if nb else None
    ws, ws_n = None, 0
    if nw or nb:
        ws_n = _lib.load().smel_layernorm_bwd_ws_floats(R, n)
        ws = rows.new_empty(ws_n, dtype=torch.float32)
    _lib.call("smel_layernorm_bwd", dy2.data_ptr(), rows.data_ptr(), R, n, pitch, p(w), stats.data_ptr(), p(ds2), dt, wt,
              p(dx), p(dw), p(db), p(ws), ws_n, _lib.stream())
    return dx, dx if add else None, dw, db, None, None


class _LayerNormFn(torch.autograd.Function):
    """forward(x, h, w, b, eps, the call's (columns, types)): y, or (s, y) with the residual addend h. Saved: the rows that
    the norm read and two fp32 numbers a row."""

    @staticmethod
    def forward(ctx, x, h, w, b, eps, call):
        n, dt, wt = call
        rows, R, s, y, stats = _ln_forward(x, h, w, b, eps, n, dt, wt)
        ctx.save_for_backward(rows, w, stats)
        ctx.call = (h is not None, n, R, dt, wt, x.shape, torch.float32 if wt == 2 else x.dtype)
        ctx.set_materialize_grads(False)
        return y if h is None else (s, y)

    backward = staticmethod(_lib.once(_ln_backward))     # on the forward's device: autograd's thread has set it


def _ln(x, h, w, b, eps):
    call = _ln_check(x, h, w, b)
    with _lib.on_device_of(x):
        if torch.is_grad_enabled() and (x.requires_grad or h is not None and h.requires_grad or w is not None and w.requires_grad
                                        or b is not None and b.requires_grad) or _lib.forward_mode():
            return _lib.apply(_LayerNormFn, x, h, w, b, float(eps), call)
        _, _, s, y, _ = _ln_forward(x, h, w, b, float(eps), *call)
    return y if h is None else (s, y)


def layernorm(x, w, b, eps):
    """(x - mean) rstd w + b over the last dimension: bf16, fp16 or fp32 rows of any stride; w and b (either may be None: 1
    and 0) of the rows' dtype or fp32, trained: backward gives dx, dw and db. fp32 math, one rounding."""
    return _ln(x, None, w, b, eps)


def add_layernorm(h, x, w, b, eps):
    """(h + x, layernorm(h + x)): the residual add, rounded to the stream's dtype, and the norm after it."""
    return _ln(x, h, w, b, eps)


# ------------------------------------------------------------------------------------------------ around the residual add

_GATE_NONE, _GATE_CHANNEL, _GATE_TOKEN, _GATE_FULL = 0, 1, 2, 3
_GATE_ACTS = {None: 0, "sigmoid": 1}


def _sw_refuse(h, x, w1, w2, gate, scale):
    """Raises what is wrong with the call."""
    _lib.one_device(x, h, w1, w2, gate, scale)
    if x.dtype not in _LN_DTYPES:
        raise ValueError(f"the norms around a residual add take bf16, fp16 or fp32 rows, got {x.dtype}")
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"the norms around a residual add take rows of 1 to {MAX_COLS} columns, got shape {tuple(x.shape)}")
    if h.shape != x.shape or h.dtype != x.dtype:
        raise ValueError(f"the stream and the block's output differ: {tuple(h.shape)} {h.dtype} and {tuple(x.shape)} {x.dtype}")
    n = x.shape[-1]
    for t in (w1, w2):
        if t is not None and (t.dtype not in (x.dtype, torch.float32) or tuple(t.shape) != (n,) or not t.is_contiguous()):
            raise ValueError(f"norm weights must be contiguous [{n}] tensors of {x.dtype} or float32")
    if gate is not None:
        token, full = (*x.shape[:-1], 1), tuple(x.shape)
        if tuple(gate.shape) not in ((n,), token, full):
            raise ValueError(f"a gate has shape [{n}], {list(token)} or {list(full)}, got {tuple(gate.shape)}")
        if gate.dtype not in (x.dtype, torch.float32) or gate.dtype != x.dtype and tuple(gate.shape) == full and full not in ((n,), token):
            raise ValueError(f"a gate of {gate.dtype} with rows of {x.dtype}")
    if scale is not None and (scale.numel() != 1 or scale.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"the scale is a number or one element of {x.dtype} or float32, got {tuple(scale.shape)} {scale.dtype}")
    raise ValueError("norm weights and a gate per channel must have one dtype")


def _sw_check(h, x, w1, w2, gate, scale) -> tuple:
    """(columns, the rows' type code, the weights' type code, the gate's kind) of a call that the kernels take."""
    dt = _LN_DTYPES.get(x.dtype)
    if dt is None or x.dim() == 0 or not x.is_cuda:
        _sw_refuse(h, x, w1, w2, gate, scale)
    n, dev, shape = x.shape[-1], x.device, x.shape
    ok = 1 <= n <= MAX_COLS and h.shape == shape and h.dtype is x.dtype and h.device == dev
    kind, wd = _GATE_NONE, None
    weights = (w1, w2)
    if gate is not None:
        ok = ok and gate.device == dev and (gate.dtype is x.dtype or gate.dtype is torch.float32)
        # of one row without leading dimensions: per channel where its dtype is the weights', whose gate that has to be
        if gate.dim() == 1 and gate.shape[0] == n and (x.dim() > 1 or all(w is None or w.dtype is gate.dtype for w in weights)):
            kind, weights = _GATE_CHANNEL, (w1, w2, gate.contiguous() if ok else None)
        elif gate.shape == shape and (n != 1 or gate.dtype is x.dtype):
            kind = _GATE_FULL
            ok = ok and gate.dtype is x.dtype
        else:
            kind = _GATE_TOKEN
            ok = ok and gate.dim() == x.dim() and gate.shape[-1] == 1 and gate.shape[:-1] == shape[:-1]
    for t in weights:
        if t is not None:
            ok = ok and (wd is None or t.dtype is wd) and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() \
                and t.device == dev
            wd = t.dtype
    wt = dt if wd is None or wd is x.dtype else 2
    if scale is not None:
        ok = ok and scale.device == dev and scale.numel() == 1 and (scale.dtype is x.dtype or scale.dtype is torch.float32)
    if not ok or (wt == 2 and wd is not None and wd is not torch.float32):
        _sw_refuse(h, x, w1, w2, gate, scale)
    return n, dt, wt, kind


def _sw_call(n, dt, wt, kind, act, plus_one, eps, w1, w2, gate, scale, scale_value):
    """The call's part that forward and backward share."""
    c, p = _lib.Sandwich(), _lib.ptr
    c.w1, c.w2, c.gate, c.scale = p(w1), p(w2), p(gate), p(scale)
    c.cols, c.eps, c.scale_value = n, eps, scale_value
    c.dtype, c.wtype, c.gate_kind, c.gate_act, c.plus_one = dt, wt, kind, act, plus_one
    c.gate_type = 2 if gate is not None and gate.dtype is torch.float32 else dt
    c.scale_type = 2 if scale is not None and scale.dtype is torch.float32 else dt
    return c


def _sw_forward(h, x, w1, w2, gate, scale, pre, rest, train):
    """(the rows of x, s, y or None, stats or None, the contiguous gate)."""
    n, dt, wt, kind, act, plus_one, eps, scale_value = rest
    if gate is not None:
        gate = gate.contiguous()
    c = _sw_call(n, dt, wt, kind, act, plus_one, eps, w1, w2, gate, scale, scale_value)
    x2, R, c.x_stride = _rows_of(x, n)
    h2, _, c.h_stride = _rows_of(h, n)
    if x2 is x:
        s, y = torch.empty_like(x), torch.empty_like(x) if pre else None
    else:
        s, y = x.new_empty(x.shape), x.new_empty(x.shape) if pre else None
    stats = x.new_empty(2 * R, dtype=torch.float32) if train else None     # a row's two reciprocal root mean squares
    c.x, c.h, c.s, c.y, c.stats = x2.data_ptr(), h2.data_ptr(), s.data_ptr(), _lib.ptr(y), _lib.ptr(stats)
    c.rows, c.pre = R, pre
    _lib.call("smel_sandwich_fwd", ctypes.byref(c), _lib.stream())
    return x2, s, y, stats, gate


def _sw_backward(ctx, ds, dy=None):
    """Gradients of h, x, w1, w2, gate and scale, each only where it is asked for."""
    x2, s, h, w1, w2, gate, scale, stats = ctx.saved_tensors
    pre, R, shape, rest = ctx.call
    n, dt, wt, kind, act, plus_one, eps, scale_value = rest
    nh, nx, nw1, nw2, ng, nsc = ctx.needs_input_grad[:6]
    none = (None, None, None)
    if ds is None and dy is None:
        return (None,) * 6 + none
    c = _sw_call(n, dt, wt, kind, act, plus_one, eps, w1, w2, gate, scale, scale_value)
    c.rows, c.x_stride = R, n if x2.is_contiguous() else x2.stride(0)     # of what comes back: hooks on saved tensors may repack it
    ds2 = ds.contiguous() if ds is not None else None
    dy2 = dy.contiguous() if dy is not None else None
    p = _lib.ptr
    new = (lambda: torch.empty_like(x2)) if x2.shape == shape and x2.is_contiguous() else (lambda: x2.new_empty(shape))
    passed = dy is None and scale is None and scale_value == 1.0     # the stream's gradient goes through as it is
    dh = ds if passed else new() if nh else None
    dx = new() if nx else None
    dw1 = torch.empty_like(w1) if nw1 else None
    dw2 = torch.empty_like(w2) if nw2 else None
    dg = torch.empty_like(gate) if ng else None
    dsc = torch.empty_like(scale) if nsc else None
    c.x, c.s, c.ds, c.dy, c.stats = x2.data_ptr(), p(s), p(ds2), p(dy2), stats.data_ptr()
    c.dh, c.dx, c.dw1, c.dw2, c.dgate, c.dscale = None if passed else p(dh), p(dx), p(dw1), p(dw2), p(dg), p(dsc)
    if nsc:
        h2, _, c.h_stride = _rows_of(h, n)
        c.h = h2.data_ptr()
    ws, ws_n = None, _lib.load().smel_sandwich_bwd_ws_floats(ctypes.byref(c))
    if ws_n:
        ws = x2.new_empty(ws_n, dtype=torch.float32)
    if nx or nw1 or nw2 or ng or nsc or not passed and nh:
        _lib.call("smel_sandwich_bwd", ctypes.byref(c), p(ws), ws_n, _lib.stream())
    return (dh if nh else None, dx, dw1, dw2, dg, dsc) + none


class _SandwichFn(torch.autograd.Function):
    """forward(h, x, w1, w2, gate, scale, pre, keep h, the call's numbers): s, or (s, y) with ``pre``. Saved: x's rows, s (pre), the
    gate, two fp32 numbers a row, and h for a trained scale."""

    @staticmethod
    def forward(ctx, h, x, w1, w2, gate, scale, pre, rest, _):
        x2, s, y, stats, gate = _sw_forward(h, x, w1, w2, gate, scale, pre, rest, True)
        ctx.save_for_backward(x2, s if pre else None, h if ctx.needs_input_grad[5] else None, w1, w2, gate, scale, stats)
        ctx.call = (pre, stats.shape[0] // 2, x.shape, rest)
        ctx.set_materialize_grads(False)
        return (s, y) if pre else s

    backward = staticmethod(_lib.once(_sw_backward))     # on the forward's device: autograd's thread has set it


def _sandwich(h, x, w1, w2, eps, plus_one, gate, gate_act, scale, pre):
    act = _GATE_ACTS.get(gate_act)
    if act is None:
        raise ValueError(f"gate_act is None or 'sigmoid', got {gate_act!r}")
    value = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        scale, value = None, float(scale)
    rest = (*_sw_check(h, x, w1, w2, gate, scale), act, bool(plus_one), float(eps), value)
    with _lib.on_device_of(x):
        if torch.is_grad_enabled() and (h.requires_grad or x.requires_grad or w1 is not None and w1.requires_grad
                                        or w2 is not None and w2.requires_grad or gate is not None and gate.requires_grad
                                        or scale is not None and scale.requires_grad) or _lib.forward_mode():
            return _lib.apply(_SandwichFn, h, x, w1, w2, gate, scale, pre, rest, None)
        _, s, y, _, _ = _sw_forward(h, x, w1, w2, gate, scale, pre, rest, False)
    return (s, y) if pre else s


def post_rmsnorm(h, x, w, eps, plus_one=False, gate=None, gate_act=None, scale=None):
    """scale (h + gate rmsnorm(x)): the norm behind a block, its gate, the residual add and the residual scale, rounded once.

    h, x [..., n]: the residual stream and the block's output, bf16, fp16 or fp32 rows of any stride. w [n] (None: 1; 1 + w with
    ``plus_one``), of the rows' dtype or fp32. gate: a value per channel [n] (the weights' dtype), per token [..., 1] (the rows' dtype
    or fp32) or per element [..., n] (the rows' dtype); of a lone row [n], a gate [n] is the one whose dtype it has. ``gate_act``
    "sigmoid": the gate's sigmoid. scale: a number or one element on
    the GPU. Backward gives every gradient that is asked for: of h, x, w, the gate and the scale."""
    return _sandwich(h, x, w, None, eps, plus_one, gate, gate_act, scale, False)


def sandwich_rmsnorm(h, x, w_post, w_pre, eps, plus_one=False, gate=None, gate_act=None, scale=None):
    """(s, y): s = ``post_rmsnorm(h, x, w_post, ...)`` and y = rmsnorm(s) with w_pre, the norm before the next block (of the rounded
    s, as the next block would read it). w_pre None: weight 1."""
    return _sandwich(h, x, w_post, w_pre, eps, plus_one, gate, gate_act, scale, True)
