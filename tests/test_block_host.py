"""Host-side checks of the recurrence and the residual norm that need no GPU: exported symbols, plain-C headers, argument errors that are reported
before anything is launched, workspace arithmetic, the Python surface's refusals."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import nanoplm_amd as npa
from nanoplm_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = {"nplm_recurrence": _lib.RECURRENCE_SYMBOLS, "nplm_resnorm": _lib.RESNORM_SYMBOLS}
A = 0x10000   # a fake, well-aligned, never dereferenced device address


def _declared(name):
    return set(re.findall(rf"\b({name}_[a-z_]+)\s*\(", open(os.path.join(ROOT, "include", name + ".h")).read())) - {name + "_bytes"}


@pytest.mark.parametrize("name", HEADERS)
def test_library_exports_every_declared_symbol(name):
    assert _declared(name) == set(HEADERS[name])
    lib = ctypes.CDLL(_lib.LIB_PATH)
    assert all(hasattr(lib, s) for s in HEADERS[name])


@pytest.mark.parametrize("name", HEADERS)
def test_header_is_plain_c_and_links(name, tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    src, exe = tmp_path / "abi.c", tmp_path / "abi"
    src.write_text(f'#include "{name}.h"\ntypedef void (*fn)(void);\nint main(void) {{ fn all[] = {{'
                   + ", ".join(f"(fn){s}" for s in sorted(HEADERS[name])) + "}; return all[0] == 0; }\n")
    libdir = os.path.dirname(_lib.LIB_PATH)
    cc = subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe),
                         "-L", libdir, "-l:" + os.path.basename(_lib.LIB_PATH), "-Wl,-rpath," + libdir, "-Wl,-rpath-link,/opt/rocm/lib"],
                        capture_output=True, text=True)
    assert cc.returncode == 0, cc.stderr
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def _fwd(x=A, xs=64, g=A, gs=128, cu=A, decay=A, scale=8.0, h0=A, y=A, state=A, carries=A, T=100, C=64, S=2, act=1, wd=1, flags=0, ws=A, wsb=1 << 40):
    return _lib.load().nplm_recurrence_fwd(x, xs, g, gs, cu, decay, scale, h0, y, state, carries, ws, wsb, T, C, S, act, wd, flags, None)


def _bwd(x=A, xs=64, g=A, gs=128, dy=A, ds=64, cu=A, decay=A, scale=8.0, carries=A, dx=A, dg=A, dd=A, dh=A, T=100, C=64, S=2, act=1, wd=1, flags=0,
         ws=A, wsb=1 << 40):
    return _lib.load().nplm_recurrence_bwd(x, xs, g, gs, dy, ds, cu, decay, scale, A, A, carries, dx, dg, dd, dh, ws, wsb, T, C, S, act, wd, flags, None)


def _step(x=A, xs=64, g=A, gs=128, decay=A, scale=8.0, state=A, out=A, slots=A, y=A, B=4, C=64, N=8, act=1, wd=1):
    return _lib.load().nplm_recurrence_step(x, xs, g, gs, decay, scale, state, out, slots, y, B, C, N, act, wd, None)


def test_recurrence_argument_errors():
    for f in (_fwd, _bwd):
        assert f(x=None) == -1 and f(g=None) == -1 and f(cu=None) == -1 and f(decay=None) == -1
        assert f(T=-1) == -2 and f(C=0) == -2 and f(S=-1) == -2 and f(T=2 ** 31) == -2
        assert f(xs=63) == -2 and f(gs=127) == -2 and f(xs=1 << 41) == -2
        assert f(scale=0.0) == -2 and f(scale=-1.0) == -2 and f(scale=float("nan")) == -2 and f(scale=float("inf")) == -2
        assert f(act=2) == -4 and f(wd=5) == -4
        assert f(x=A + 1) == -5 and f(g=A + 1) == -5 and f(decay=A + 1) == -5 and f(cu=A + 2) == -5 and f(carries=A + 2) == -5
        assert f(flags=8) == -9
    assert _fwd(y=None) == -1 and _fwd(state=A + 2) == -5 and _fwd(flags=2) == -9
    assert _fwd(T=0, state=None) == 0 and _fwd(T=0, S=0) == 0
    assert _bwd(dy=None) == -1 and _bwd(dx=None) == -1 and _bwd(dg=None) == -1 and _bwd(dd=None) == -1 and _bwd(carries=None) == -1
    assert _bwd(ds=60) == -2 and _bwd(dh=A + 2) == -5 and _bwd(dd=A + 2) == -5


def test_sizes_that_no_launch_can_count():
    for act, most in ((0, 2 ** 29), (1, 2 ** 30)):
        for f, size in ((_fwd, "fwd"), (_bwd, "bwd")):
            need = getattr(_lib.load(), f"nplm_recurrence_{size}_workspace_bytes")
            assert f(T=most + 1, act=act) == -2 and need(most + 1, 64, 2, act) == 0
            assert f(T=most // 8 + 1, C=1024, act=act, xs=1024, gs=2048, **({"ds": 1024} if f is _bwd else {})) == -2
            assert need(most - 4096, 64, 2, act) > 0 and f(T=most - 4096, act=act, ws=None) == -6
    assert _step(B=2 ** 24, N=2 ** 25) == -2


def test_step_argument_errors():
    assert _step(x=None) == -1 and _step(g=None) == -1 and _step(decay=None) == -1 and _step(state=None) == -1 and _step(out=None) == -1
    assert _step(B=-1) == -2 and _step(C=0) == -2 and _step(N=-1) == -2 and _step(slots=None, B=9) == -2 and _step(xs=10) == -2 and _step(scale=0.0) == -2
    assert _step(act=3) == -4 and _step(x=A + 1) == -5 and _step(slots=A + 1) == -5 and _step(state=A + 2) == -5
    assert _step(B=0, x=None) == 0


def _rn_fwd(u=A, us=64, g=A, gs=64, r=A, rs=64, p=(A, A, A, A, A), out=A, normed=A, stats=A, T=10, C=64, act=1, st=1, wd=1, flags=0):
    return _lib.load().nplm_resnorm_fwd(u, us, g, gs, r, rs, *p, 1e-5, out, normed, stats, T, C, act, st, wd, flags, None)


def _rn_bwd(u=A, us=64, g=A, gs=64, r=A, rs=64, do=A, dos=64, dn=A, dns=64, stats=A, p=(A, A, A, A), du=A, dg=A, dr=A, grads=(A,) * 5, ws=A, wsb=1 << 40, T=10,
            C=64, act=1, st=1, wd=1, flags=0):
    return _lib.load().nplm_resnorm_bwd(u, us, g, gs, r, rs, do, dos, dn, dns, stats, *p, du, dg, dr, *grads, ws, wsb, T, C, act, st, wd, flags, None)


def test_resnorm_argument_errors():
    for f in (_rn_fwd, _rn_bwd):
        assert f(u=None) == -1 and f(r=None) == -1
        assert f(T=-1) == -2 and f(C=0) == -2 and f(T=2 ** 31) == -2 and f(us=63) == -2 and f(rs=1) == -2 and f(gs=0) == -2
        assert f(act=2) == -4 and f(st=7) == -4 and f(wd=3) == -4 and f(act=0, st=1) == -4
        assert f(u=A + 1) == -5 and f(r=A + 1) == -5 and f(g=A + 1) == -5 and f(stats=A + 8) == -5
        assert f(flags=4) == -9 and f(C=16385, us=16385, rs=16385, gs=16385) == -10
    assert _rn_fwd(out=None) == -1 and _rn_fwd(p=(None, A, A, A, A)) == -1 and _rn_fwd(p=(A, A, A, None, A)) == -1
    assert _rn_fwd(p=(A, A, A, None, None)) == -1 and _rn_fwd(flags=2) == -9 and _rn_fwd(T=0) == 0
    assert _rn_bwd(du=None) == -1 and _rn_bwd(dg=None) == -1 and _rn_bwd(dr=None) == -1 and _rn_bwd(stats=None) == -1
    assert _rn_bwd(p=(None, None, A, A)) == -1 and _rn_bwd(p=(A, A, A, None)) == -1 and _rn_bwd(p=(A, A, None, A)) == -1
    assert _rn_bwd(ws=None) == -6 and _rn_bwd(ws=A + 64) == -6 and _rn_bwd(wsb=100) == -6


def test_workspace_bytes():
    lib = _lib.load()
    assert lib.nplm_resnorm_bwd_workspace_bytes(0, 64) == 0 and lib.nplm_resnorm_bwd_workspace_bytes(10, 16385) == 0
    for T, C in ((1, 1), (1000, 64), (131072, 1024), (2 ** 31 - 2 ** 20 - 1, 768), (70000, 16384)):
        n = lib.nplm_resnorm_bwd_workspace_bytes(T, C)
        assert n > 0 and n % 256 == 0


# ---- Python surface -----------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, gates, decay, cu = torch.randn(5, 4), torch.randn(5, 8), torch.randn(4), torch.tensor([0, 5], dtype=torch.int32)
    for call in (lambda: npa.varlen_recurrence(x, gates, cu, decay), lambda: npa.VarlenRecurrence(4)(x, gates, cu),
                 lambda: npa.recurrence_step(x, gates, decay, torch.zeros(5, 4)), lambda: npa.residual_norm(x, x), lambda: npa.ResidualNorm(4)(x, x)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_modules_and_their_parameters():
    m = npa.VarlenRecurrence(64, scale=4.0)
    kept = torch.exp(-4.0 * torch.nn.functional.softplus(m.decay.detach().double()))
    assert m.decay.dim() == 1 and float(kept.min()) >= 0.899 and float(kept.max()) <= 0.9991
    assert npa.VarlenRecurrence(8, dtype=torch.bfloat16).decay.dtype == torch.bfloat16
    with pytest.raises(ValueError):
        npa.VarlenRecurrence(8, scale=0.0)
    with pytest.raises(RuntimeError, match="no next token"):
        npa.VarlenRecurrence(4, reverse=True).step(torch.zeros(1, 4), torch.zeros(1, 8), torch.zeros(1, 4))
    names = lambda **k: {n for n, _ in npa.ResidualNorm(8, **k).named_parameters()}
    assert names() == {"post_weight", "pre_weight"}
    assert names(bias=True, scale_init=0.0) == {"post_weight", "post_bias", "scale", "pre_weight", "pre_bias"}
    assert names(post=False, pre=False, scale_init=1.0, bias=True) == {"scale"}
    for bad in (dict(norm="batch"), dict(channels=0), dict(channels=16385)):
        with pytest.raises(ValueError):
            npa.ResidualNorm(**{"channels": 8, **bad})


def test_refusals_that_come_before_the_device_is_looked_at():
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="2-D"):
        npa.varlen_recurrence(torch.zeros(5), torch.zeros(5, 8), cu, torch.zeros(4))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        npa.varlen_recurrence(torch.zeros(5, 4, dtype=torch.float16), torch.zeros(5, 8), cu, torch.zeros(4))
    with pytest.raises(ValueError, match="2-D"):
        npa.residual_norm(torch.zeros(5), torch.zeros(5))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        npa.residual_norm(torch.zeros(5, 4, dtype=torch.float16), torch.zeros(5, 4))
