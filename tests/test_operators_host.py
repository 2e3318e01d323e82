"""What the layer norm, balance loss and orthogonalisation entry points refuse, on the host before any launch (no GPU)."""
import ctypes

import pytest
import torch


def _L():
    from smel import _lib
    return _lib.load()


def test_layernorm_refusals():
    L = _L()
    f = lambda x=16, h=None, rows=4, cols=64, stride=64, dt=0, wt=0, s=None, y=16, st=16: L.smel_layernorm_fwd(
        x, h, rows, cols, stride, None, None, 1e-5, dt, wt, s, y, st, None)
    assert f(cols=0) == -1 and f(rows=-1) == -1 and f(cols=16385) == -2 and f(stride=63) == -1
    assert f(dt=3) == -1 and f(dt=-1) == -1 and f(dt=2, wt=0) == -1 and f(dt=0, wt=1) == -1
    assert f(x=None) == -1 and f(y=None) == -1 and f(st=None) == -1 and f(h=16) == -1      # h without s
    assert f(rows=0, x=None, y=None, st=None) == 0
    b = lambda dy=16, x=16, rows=4, cols=64, stride=64, dt=0, wt=0, dx=16, dw=None, ws=None, n=0: L.smel_layernorm_bwd(
        dy, x, rows, cols, stride, None, 16, None, dt, wt, dx, dw, None, ws, n, None)
    assert b(dy=None) == -1 and b(x=None) == -1 and b(cols=20000) == -2 and b(stride=1) == -1 and b(wt=1) == -1
    need = L.smel_layernorm_bwd_ws_floats(4, 64)
    assert need > 0 and b(dw=16) == -1 and b(dw=16, ws=16, n=need - 1) == -1 and b"workspace" in L.smel_last_error()
    assert L.smel_layernorm_bwd_ws_floats(0, 64) == 0 and b(rows=0, dx=None) == 0


def test_balance_refusals():
    L = _L()
    need = L.smel_balance_ws_bytes(100, 16, 3)
    assert need > 0 and L.smel_balance_ws_bytes(100, 600, 1) == 0

    def f(z=16, ldl=16, dt=0, topi=16, T=100, E=16, K=2, off=16, S=3, loss=16, counts=16, stats=16, w=16, ws=16, n=need):
        return L.smel_balance_fwd(z, ldl, dt, topi, 1, T, E, K, None, off, 1, S, 1.0, loss, counts, stats, w, ws, n, None)
    g = lambda z=16, st=16, w=16, go=16, dz=16, E=16: L.smel_balance_bwd(z, 16, 0, 100, E, 3, st, w, go, dz, None)
    assert f(E=513, ldl=513) == -2 and f(E=0) == -2 and f(T=-1) == -2 and f(T=(1 << 24) + 1) == -2 and f(S=0) == -2 and f(S=(1 << 22) + 1) == -2
    assert f(off=None) == -1 and f(dt=3) == -1 and f(ldl=15) == -1 and f(z=None) == -1 and f(topi=None) == -1
    assert f(K=0) == -2 and f(K=65) == -2 and f(loss=None) == -1 and f(counts=None) == -1 and f(w=None) == -1
    assert f(stats=8) == -1 and g(st=8) == -1
    assert f(ws=None) == -1 and f(ws=8) == -1 and f(n=need - 1) == -1 and b"workspace" in L.smel_last_error()
    assert g(z=None) == -1 and g(st=None) == -1 and g(w=None) == -1 and g(go=None) == -1 and g(dz=None) == -1 and g(E=600) == -2
    assert L.smel_balance_bwd(None, 16, 0, 0, 16, 1, None, None, None, None, None) == 0


def test_orthogonalize_refusals():
    from array import array
    L = _L()

    def f(x=16, y=16, batch=2, rows=16, cols=64, xb=1024, xr=64, xc=1, dt=1, steps=5, eps=1e-7, ws=16, n=1 << 40):
        job = array("q", (x, y, batch, rows, cols, xb, xr, xc, dt))
        return L.smel_orthogonalize(job.buffer_info()[0], 1, steps, 3.0, -4.0, 2.0, eps, ws, n, None)
    assert f(rows=129, cols=200) == -2 and b"short side" in L.smel_last_error()
    assert f(batch=-1) == -1 and f(rows=-1) == -1 and f(dt=3) == -1 and f(x=0) == -1 and f(y=0) == -1
    assert f(x=18) == -1 and f(y=17, dt=0) == -1 and f(xr=-64) == -1 and f(xr=2, xc=64 * 3) == -1
    assert f(steps=-1) == -1 and f(steps=65) == -1 and f(eps=-1.0) == -1 and f(eps=float("nan")) == -1
    assert f(ws=None) == -1 and f(ws=24) == -1 and f(n=100) == -1 and b"workspace" in L.smel_last_error()
    assert f(cols=1 << 31) == -2 and f(batch=1 << 31) == -2
    assert f(batch=0, ws=None, n=0) == 0 and f(rows=0, ws=None, n=0) == 0
    assert L.smel_orthogonalize(None, 0, 5, 1.0, 1.0, 1.0, 0.0, None, 0, None) == 0
    assert L.smel_orthogonalize(None, 1, 5, 1.0, 1.0, 1.0, 0.0, None, 0, None) == -1


def test_job_layout_matches_header():
    # nine 8-byte fields, as the binding packs them
    assert ctypes.sizeof(ctypes.c_int64) * 9 == 72


def test_python_refusals():
    """CPU tensors, wrong types and shapes raise ValueError before anything runs."""
    from smel.lora import orthogonalize
    from smel.loss import balance_loss
    from smel.norm import add_layernorm, layernorm
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        layernorm(x, w, w, 1e-5)
    with pytest.raises(ValueError, match="GPU"):
        add_layernorm(x, x, w, w, 1e-5)
    with pytest.raises(ValueError, match="GPU"):
        balance_loss(x, torch.zeros(4, 2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        orthogonalize(x)
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(x, steps=65)
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(x, eps=-1.0)
    assert orthogonalize([]) == []


def test_orthogonalize_workspace_of_steps():
    """Steps beyond a pass keep the matrices in the workspace: its size says so, and a call with less is refused."""
    from array import array
    L = _L()
    for rows, cols in ((16, 2048), (24, 70), (2048, 60), (100, 129)):
        job = array("q", (16, 16, 3, rows, cols, rows * cols, cols, 1, 1))
        at = job.buffer_info()[0]
        ws = lambda steps, a=3.4445: L.smel_orthogonalize_ws(at, 1, steps, a)
        call = lambda steps, n: L.smel_orthogonalize(at, 1, steps, 3.4445, -4.0, 2.0, 1e-7, 16, n, None)
        assert ws(0) == ws(6) and ws(6) + 3 * rows * cols * 8 <= ws(7) == ws(12) == ws(64)
        assert ws(13, 1.875) == ws(6) and ws(14, 1.875) == ws(7) and ws(64, 1.0) == ws(6)
        assert call(7, ws(7) - 1) == -1 and b"workspace" in L.smel_last_error()
        assert call(6, ws(6) - 1) == -1


def test_job_fields_match_header():
    """The fields of smel_ortho_job, by name and order, are those that the binding packs, each of 8 bytes."""
    import os
    import re
    from smel import lora
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "smel_ortho.h")).read(), flags=re.S)
    body = re.search(r"typedef struct smel_ortho_job \{(.*?)\} smel_ortho_job;", src, re.S).group(1)
    fields = []
    for line in body.split(";"):
        if line.strip():
            m = re.fullmatch(r"\s*(?:const\s+)?(void\s*\*|int64_t)\s*(.+?)\s*", line, re.S)
            assert m, line      # pointers and int64_t alone: 8 bytes, without gaps
            fields += [f.strip() for f in m.group(2).split(",")]
    assert tuple(fields) == lora._ORTHO_JOB


def test_orthogonalize_takes_many_columns():
    """Columns beyond what a launch's grid takes are split over launches, not refused; a side of 2^30 is the limit."""
    from array import array
    L = _L()

    def ws(batch, rows, cols, dt=0):
        job = array("q", (16, 16, batch, rows, cols, rows * cols, cols, 1, dt))
        return L.smel_orthogonalize_ws(job.buffer_info()[0], 1, 5, 3.4445)
    assert 0 < ws(65536, 1, 65536) and 0 < ws(1 << 20, 1 << 14, 3) and 0 < ws(256, 128, 1 << 21) and 0 < ws(3, 64, (1 << 29) + 1, 1)
    assert 0 < ws(1, 16, (1 << 30) - 1) and ws(1, 16, 1 << 30) == -1
