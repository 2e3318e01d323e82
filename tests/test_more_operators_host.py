"""What the expert selection, the norms around a residual add and the clipping refuse, on the host before any launch (no GPU)."""
import ctypes
import os
import re
import shutil
import subprocess
from array import array

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _L():
    from smel import _lib
    return _lib.load()


def test_select_refusals():
    L = _L()

    def f(z=16, ldl=64, dt=0, T=4, E=64, K=8, score=0, groups=8, kept=4, best=2, topv=16, topi=16):
        return L.smel_select_experts(z, ldl, dt, T, E, K, score, None, groups, kept, best, 1, 1.0, topv, topi, None, None, None)
    assert f(E=513, ldl=513, groups=1, kept=1) == -2 and b"experts" in L.smel_last_error()
    assert f(K=17) == -2 and f(K=0) == -1 and f(E=0) == -1 and f(T=-1) == -1 and f(T=(1 << 25) + 1) == -2
    assert f(dt=3) == -1 and f(score=2) == -1 and f(ldl=63) == -1 and f(groups=0) == -2 and f(groups=7) == -2 and f(groups=65, E=65 * 2, ldl=130) == -2
    assert f(kept=0) == -1 and f(kept=9) == -1 and f(kept=1, K=9) == -1 and f(best=0) == -1 and f(best=3) == -1
    assert f(z=None) == -1 and f(topv=None) == -1 and f(topi=None) == -1 and f(T=0, z=None) == 0
    b = lambda z=16, T=4, E=64, K=8, score=0, topi=16, d=16, st=None, dz=16, ldd=64: L.smel_select_experts_bwd(  # noqa: E731
        z, 64, 0, T, E, K, score, 1, 1.0, topi, d, st, dz, ldd, None)
    assert b(ldd=63) == -1 and b(z=None) == -1 and b(topi=None) == -1 and b(d=None) == -1 and b(dz=None) == -1
    assert b(score=1) == -1 and b(E=600, ldd=600) == -2 and b(K=17) == -2 and b(T=0, z=None) == 0
    r = lambda x=16, w=16, T=4, H=64, E=8, lg=16: L.smel_router_logits(x, w, T, H, E, lg, None)  # noqa: E731
    assert r(H=72) == -2 and r(E=513) == -2 and r(x=None) == -1 and r(w=None) == -1 and r(lg=None) == -1 and r(T=-1) == -1 and r(T=0, x=None) == 0
    assert r(T=1 << 25) == -2


def _call(**kw):
    from smel import _lib
    c = _lib.Sandwich()
    base = dict(h=16, x=16, s=16, y=16, stats=16, ds=16, dy=16, dh=16, dx=16, rows=4, cols=64, x_stride=64, h_stride=64, eps=1e-6, scale_value=1.0,
                pre=1)
    for k, v in {**base, **kw}.items():
        setattr(c, k, v)
    return c


def test_sandwich_refusals():
    L = _L()
    f = lambda **kw: L.smel_sandwich_fwd(ctypes.byref(_call(**kw)), None)  # noqa: E731
    b = lambda ws=None, n=0, **kw: L.smel_sandwich_bwd(ctypes.byref(_call(**kw)), ws, n, None)  # noqa: E731
    for g in (f, b):
        assert g(rows=-1) == -1 and g(cols=0) == -1 and g(cols=16385, x_stride=1 << 20, h_stride=1 << 20) == -2
        assert g(x_stride=63) == -1 and g(h_stride=63) == -1 and g(dtype=3) == -1 and g(dtype=0, wtype=1) == -1 and g(dtype=2, wtype=0) == -1
        assert g(gate_kind=4) == -1 and g(gate_kind=1) == -1 and g(gate_kind=2, gate=16, gate_type=1) == -1
        assert g(scale=16, scale_type=1) == -1 and g(x=None) == -1
    assert f(h=None) == -1 and f(s=None) == -1 and f(y=None) == -1
    assert f(rows=0, x=None) == 0
    assert b(s=None) == -1 and b(stats=None) == -1 and b(dscale=16, h=None) == -1
    assert L.smel_sandwich_fwd(None, None) == -1 and L.smel_sandwich_bwd(None, None, 0, None) == -1
    need = lambda **kw: L.smel_sandwich_bwd_ws_floats(ctypes.byref(_call(**kw)))  # noqa: E731
    assert need() == 0 and need(rows=0, dw1=16) == 0 and need(cols=0) == 0
    one = need(dw1=16)
    assert one > 0 and need(dw1=16, dw2=16, dgate=16, gate=16, gate_kind=1) == 3 * one and need(dgate=16, gate=16, gate_kind=3) == 0
    assert b(dw1=16) == -1 and b(dw1=16, ws=16, n=one - 1) == -1 and b"workspace" in L.smel_last_error() and b(dw1=16, ws=20, n=one) == -1


def test_clip_refusals():
    L = _L()

    def f(*jobs, ws=16, n=None, most=1.0, eps=1e-6, kind=0, norm=16):
        a = array("q", [v for j in jobs for v in j])
        at = a.buffer_info()[0]
        need = L.smel_clip_ws(at, len(jobs))
        return need, L.smel_clip_grads(at, len(jobs), kind, most, eps, norm, ws, need if n is None else n, None)
    ok = (4096, 8192, 100, 1)
    assert f((4096, 8192, -1, 1)) == (-1, -1) and f((4096, 8192, 4, 3)) == (-1, -1) and f((0, 8192, 4, 1)) == (-1, -1)
    assert f((4098, 8192, 4, 1)) == (-1, -1) and f((4097, 8192, 4, 0)) == (-1, -1) and f((4096, 8192, 1 << 40, 1))[1] == -2
    assert f((4096, 8193, 4, 0))[1] == -1 and f((4096, 0, 4, 1))[1] == -1
    assert f(ok, most=-1.0)[1] == -1 and f(ok, most=float("nan"))[1] == -1 and f(ok, eps=-1.0)[1] == -1 and f(ok, kind=2)[1] == -1
    assert f(ok, norm=None)[1] == -1 and f(ok, ws=None)[1] == -1 and f(ok, ws=24)[1] == -1
    need, rc = f(ok, n=8)
    assert need == 16 and rc == -1 and b"workspace" in L.smel_last_error()
    # overlaps: (in, out, n, fp32)
    for a, b in (((4096, 4096, 100, 1), (4096, 4096, 100, 1)), ((4096, 8192, 100, 1), (8192, 16384, 10, 1)), ((4096, 4096, 100, 1), (4492, 4492, 9, 1)),
                 ((4096, 8192, 100, 1), (40960, 8188, 2, 1)), ((4096, 4100, 10, 1), (40960, 8192, 1, 1)), ((4096, 4096, 100, 1), (4200, 8192, 1, 1)),
                 ((4096, 8192, 1000, 1), (4100, 8200, 1, 1))):
        for jobs in ((a, b), (b, a)):
            assert f(*jobs)[1] == -1 and b"overlap" in L.smel_last_error(), jobs
    assert L.smel_clip_ws(None, 0) == 8 and L.smel_clip_ws(None, 1) == -1


def test_layouts_match_headers(tmp_path):
    """smel_sandwich has the C compiler's offsets, smel_clip_job the binding's order of 8-byte fields."""
    from smel import _lib, lora
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "smel_clip.h")).read(), flags=re.S)
    body = re.search(r"typedef struct smel_clip_job \{(.*?)\} smel_clip_job;", src, re.S).group(1)
    fields = []
    for line in body.split(";"):
        if line.strip():
            m = re.fullmatch(r"\s*(?:const\s+)?(void\s*\*|int64_t)\s*(.+?)\s*", line, re.S)
            assert m, line
            fields += [f.strip() for f in m.group(2).split(",")]
    assert tuple(fields) == lora._CLIP_JOB
    cxx = shutil.which("g++")
    if cxx is None or not os.path.exists("/opt/rocm/include/hip/hip_runtime.h"):
        pytest.skip("no host compiler / HIP headers")
    names = [n for n, _ in _lib.Sandwich._fields_]
    prog = '#include <stddef.h>\n#include <stdio.h>\n#include "smel_norm.h"\nint main() {\n' + \
        "".join(f'printf("{n} %zu\\n", offsetof(smel_sandwich, {n}));\n' for n in names) + 'printf("size %zu\\n", sizeof(smel_sandwich));\nreturn 0; }\n'
    (tmp_path / "p.cpp").write_text(prog)
    subprocess.run([cxx, "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), str(tmp_path / "p.cpp"), "-o",
                    str(tmp_path / "p")], check=True, capture_output=True)
    got = dict(line.split() for line in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(got.pop("size")) == ctypes.sizeof(_lib.Sandwich)
    assert {k: int(v) for k, v in got.items()} == {n: getattr(_lib.Sandwich, n).offset for n in names}


def test_python_refusals():
    from smel.lora import clip_grads, clip_grads_, grad_norm
    from smel.moe import route_grouped, select_experts
    from smel.norm import post_rmsnorm, sandwich_rmsnorm
    x, w = torch.zeros(4, 8), torch.ones(8)
    for bad in (lambda: select_experts(x, 2), lambda: route_grouped(x, x, 2), lambda: post_rmsnorm(x, x, w, 1e-6),
                lambda: sandwich_rmsnorm(x, x, w, w, 1e-6), lambda: clip_grads([x], 1.0), lambda: clip_grads_([x], 1.0), lambda: grad_norm([x])):
        with pytest.raises(ValueError, match="GPU"):
            bad()
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads([x], -1.0)
    with pytest.raises(ValueError, match="norm_type"):
        grad_norm([x], 1.0)
    with pytest.raises(ValueError, match="gate_act"):
        post_rmsnorm(x, x, w, 1e-6, gate_act="relu")
    assert clip_grads([], 1.0)[0] == []


def test_flat():
    """Which tensors are taken as they lie in memory."""
    from smel.lora import _flat
    t = torch.zeros(4, 6, 5)
    for yes in (t, t.permute(2, 0, 1), t.transpose(0, 1), t[1], t[2, 3], t[:1], torch.zeros(()), torch.zeros(0, 3)):
        assert _flat(yes), (yes.shape, yes.stride())
    for no in (t[:, 1:], t[..., ::2], t[:1].expand(3, 6, 5), t[:, :, :1]):
        assert not _flat(no), (no.shape, no.stride())
