"""Host-side checks of linear attention and the layer norm that need no GPU: exported symbols, plain-C headers, argument errors that are reported before anything is
launched, which rows a block gets, workspace arithmetic, the Python surface's refusals."""
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
HEADERS = {"nplm_linattn": _lib.LINATTN_SYMBOLS, "nplm_layernorm": _lib.LAYERNORM_SYMBOLS}
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


# ---- which rows a block gets --------------------------------------------------------------------------------------------------------------
def _segments(cu, T, L):
    cu, lib = torch.tensor(cu, dtype=torch.int32), _lib.load()
    S = cu.numel() - 1
    out = torch.full((T // L + S + 2 + T // L, 6), -99, dtype=torch.int64)
    places = lib.nplm_linattn_debug_segments(cu.data_ptr(), S, T, L, out.data_ptr())
    assert places == T // L + S + 2
    return out[:places].tolist(), out[places:].tolist()


def _cases():
    g = torch.Generator().manual_seed(0)
    yield [0], 0, 64
    yield [0], 200, 64
    yield [5, 5, 130], 200, 64
    for L in (64, 128, 320, 2048):
        for kind in range(6):
            lens = torch.randint(0, (3, 70, 700, 5000, 2, 130)[kind], ((300, 40, 20, 6, 500, 1)[kind],), generator=g).tolist()
            cu = torch.tensor([0, *lens]).cumsum(0)
            lead, tail = ((0, 0), (37, 0), (0, 900))[kind % 3]
            yield (cu + lead).tolist(), int(cu[-1]) + lead + tail, L


@pytest.mark.parametrize("cu,T,L", list(_cases()))
def test_every_row_is_in_one_segment_and_every_boundary_is_found(cu, T, L):
    places, bounds = _segments(cu, T, L)
    edges = [0, *cu, T]
    want = {(e - 1, lo, hi, p0, min(L, hi - lo - p0)) for e, (lo, hi) in enumerate(zip(edges[:-1], edges[1:])) for p0 in range(0, hi - lo, L)}
    got = [tuple(p[:5]) for p in places if p[4] > 0]
    assert len(got) == len(set(got)) and set(got) == want
    # an empty sequence of cu has one place that says so, for its state
    empty = [p[0] for p in places if p[4] == 0 and p[3] == 0 and p[2] <= p[1] and 0 <= p[0] < len(cu) - 1]
    assert sorted(empty) == [s for s, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])) if lo == hi]
    later = {(p[0], p[3]): p for p in places if p[4] > 0 and p[3] > 0}
    found = {(b[0], b[3]): (i, b) for i, b in enumerate(bounds, 1) if b[4] > 0}
    assert set(found) == set(later) and len(found) == sum(b[4] > 0 for b in bounds)
    for key, (i, b) in found.items():
        assert b[5] == i == later[key][5] and b[:5] == later[key][:5]


def test_cu_that_makes_no_sense_leads_nowhere_outside():
    g = torch.Generator().manual_seed(1)
    for T in (1, 100, 1000):
        for S in (1, 2, 65, 300):
            cu = torch.randint(-T, 2 * T, (S + 1,), generator=g).tolist()
            places, bounds = _segments(cu, T, 64)
            for i, (seq, lo, hi, p0, n, bound) in enumerate(places + bounds):
                assert -1 <= seq <= S and 0 <= lo <= T and 0 <= hi <= T and 0 <= n <= 64
                if n:
                    assert p0 >= 0 and lo + p0 + n <= hi and bound <= T // 64
                if n and i >= len(places):
                    assert p0 >= 64                              # (the segment in front of a boundary is there, too)


def test_segments_are_as_short_as_fit_the_chip_at_once():
    rows = _lib.load().nplm_linattn_debug_segment_rows
    assert rows(131072, 16, 490) == 2048 and rows(65536, 16, 1) == 2048 and rows(20011, 8, 1) == 320 and rows(129, 1, 1) == 64 and rows(10 ** 6, 1, 512) == 2048
    assert rows(128, 1, 1) == 2048 and rows(2048, 9, 16) == 2048 and rows(2048, 9, 15) == 64       # (small batches of short sequences: whole)
    for T in (1, 1000, 30000, 10 ** 6, 2 ** 31 - 2 ** 20 - 1):
        for H in (1, 7, 64, 2 ** 14):
            for S in (0, 1, 100, 10000):
                L = rows(T, H, S)
                assert L % 64 == 0 and 64 <= L <= 2048
                if 64 < L < 2048:
                    assert (T / L + S) * H <= 512 < (T / (L - 64) + S) * H


# ---- the C ABI's argument errors ------------------------------------------------------------------------------------------------------------
def _fwd(q=A, qr=64, qh=32, k=A, v=A, vr=32, cu=A, g=A, gr=2, gh=1, scale=1.0, h0=A, o=A, state=A, bounds=A, bb=1 << 40, T=300, H=2, S=2, dk=32, dv=16, act=1, gd=1, flags=0):
    return _lib.load().nplm_linattn_fwd(q, qr, qh, k, 64, 32, v, vr, 16, cu, g, gr, gh, scale, h0, o, state, bounds, bb, T, H, S, dk, dv, act, gd, flags, None)


def _bwd(q=A, qr=64, qh=32, k=A, v=A, vr=32, do=A, cu=A, g=A, gr=2, gh=1, scale=1.0, h0=A, state=A, ds=A, bounds=A, bb=1 << 40, dq=A, dko=A, dvo=A, dg=A, dh=A, ws=A,
         wsb=1 << 40, T=300, H=2, S=2, dk=32, dv=16, act=1, gd=1, flags=0):
    return _lib.load().nplm_linattn_bwd(q, qr, qh, k, 64, 32, v, vr, 16, do, 32, 16, cu, g, gr, gh, scale, h0, state, ds, bounds, bb, dq, dko, dvo, dg, dh, ws, wsb,
                                        T, H, S, dk, dv, act, gd, flags, None)


def _step(q=A, k=A, v=A, g=A, gr=2, scale=1.0, state=A, out=A, slots=A, o=A, B=4, H=2, N=8, dk=32, dv=16, act=1, gd=1, flags=0):
    return _lib.load().nplm_linattn_step(q, 64, 32, k, 64, 32, v, 32, 16, g, gr, 1, scale, state, out, slots, o, B, H, N, dk, dv, act, gd, flags, None)


def test_linattn_argument_errors():
    for f in (_fwd, _bwd):
        assert f(q=None) == -1 and f(k=None) == -1 and f(v=None) == -1 and f(cu=None) == -1 and f(g=None) == -1
        assert f(T=-1) == -2 and f(H=0) == -2 and f(S=-1) == -2 and f(dk=0) == -2 and f(dv=0) == -2 and f(T=2 ** 31) == -2
        assert f(qr=-1) == -2 and f(qh=-8) == -2 and f(gr=-1) == -2 and f(vr=1 << 37) == -2
        assert f(scale=float("nan")) == -2 and f(scale=float("inf")) == -2 and f(scale=-float("inf")) == -2
        assert f(act=2) == -4 and f(gd=5) == -4 and f(dk=129) == -10 and f(dv=129) == -10
        assert f(q=A + 1) == -5 and f(g=A + 1) == -5 and f(cu=A + 2) == -5 and f(h0=A + 2) == -5 and f(state=A + 2) == -5
        assert f(flags=4) == -9 and f(bounds=None) == -6 and f(bounds=A + 64) == -6 and f(bb=8) == -6
        assert f(H=2 ** 22) == -2 and f(S=2 ** 23) == -2
    assert _fwd(o=None) == -1 and _fwd(o=A + 2) == -5 and _fwd(T=0, state=None) == 0
    assert _bwd(do=None) == -1 and _bwd(dq=None) == -1 and _bwd(dko=None) == -1 and _bwd(dvo=None) == -1 and _bwd(state=None) == -1
    assert _bwd(dq=A + 4) == -5 and _bwd(dg=A + 1) == -5 and _bwd(dh=A + 2) == -5 and _bwd(ds=A + 1) == -5
    assert _bwd(ws=None) == -6 and _bwd(ws=A + 128) == -6 and _bwd(wsb=100) == -6


def test_linattn_step_argument_errors():
    assert _step(q=None) == -1 and _step(k=None) == -1 and _step(v=None) == -1 and _step(g=None) == -1 and _step(state=None) == -1 and _step(out=None) == -1 and _step(o=None) == -1
    assert _step(B=-1) == -2 and _step(H=0) == -2 and _step(N=-1) == -2 and _step(N=2 ** 31) == -2 and _step(slots=None, B=9) == -2 and _step(B=2 ** 16 + 1, N=2 ** 20) == -2
    assert _step(slots=None, B=2 ** 23, N=2 ** 24) == -2 and _step(gr=-1) == -2 and _step(scale=float("nan")) == -2
    assert _step(act=3) == -4 and _step(q=A + 1) == -5 and _step(slots=A + 1) == -5 and _step(state=A + 2) == -5 and _step(dk=129) == -10 and _step(flags=1) == -9
    assert _step(B=0, q=None) == 0


def _ln_fwd(x=A, xs=64, gate=A, gs=64, w=A, b=A, y=A, T=10, C=64, heads=2, act=1, wd=1, flags=0):
    return _lib.load().nplm_layernorm_fwd(x, xs, gate, gs, w, b, 1e-5, y, T, C, heads, act, wd, flags, None)


def _ln_bwd(x=A, xs=64, gate=A, gs=64, dy=A, ds=64, w=A, b=A, dx=A, dgate=A, dw=A, db=A, ws=A, wsb=1 << 40, T=10, C=64, heads=2, act=1, wd=1, flags=0):
    return _lib.load().nplm_layernorm_bwd(x, xs, gate, gs, dy, ds, w, b, 1e-5, dx, dgate, dw, db, ws, wsb, T, C, heads, act, wd, flags, None)


def test_layernorm_argument_errors():
    for f in (_ln_fwd, _ln_bwd):
        assert f(x=None) == -1 and f(w=None) == -1
        assert f(T=-1) == -2 and f(C=0) == -2 and f(heads=0) == -2 and f(heads=3) == -2 and f(T=2 ** 31) == -2 and f(xs=63) == -2 and f(gs=0) == -2
        assert f(act=2) == -4 and f(wd=7) == -4
        assert f(x=A + 1) == -5 and f(gate=A + 1) == -5 and f(w=A + 1) == -5 and f(b=A + 1) == -5
        assert f(C=1 << 16, heads=1 << 16, xs=1 << 16, gs=1 << 16, **({"ds": 1 << 16} if f is _ln_bwd else {})) == -10
        assert f(flags=8) == -9 and f(C=16385, heads=1, xs=16385, gs=16385, **({"ds": 16385} if f is _ln_bwd else {})) == -10
    assert _ln_fwd(y=None) == -1 and _ln_fwd(flags=2) == -9 and _ln_fwd(T=0, x=None) == 0
    assert _ln_bwd(dy=None) == -1 and _ln_bwd(dx=None) == -1 and _ln_bwd(dgate=None) == -1 and _ln_bwd(ds=1) == -2
    assert _ln_bwd(ws=None) == -6 and _ln_bwd(ws=A + 64) == -6 and _ln_bwd(wsb=100) == -6 and _ln_bwd(dw=A + 2) == -5


def test_workspace_bytes():
    lib = _lib.load()
    assert lib.nplm_layernorm_bwd_workspace_bytes(0, 64, 1) == 0 and lib.nplm_layernorm_bwd_workspace_bytes(10, 64, 3) == 0
    for T, C, heads in ((1, 1, 1), (1000, 64, 4), (131072, 1024, 16), (2 ** 31 - 2 ** 20 - 1, 768, 1), (70000, 16384, 1)):
        n = lib.nplm_layernorm_bwd_workspace_bytes(T, C, heads)
        assert n > 0 and n % 256 == 0
    assert lib.nplm_linattn_bounds_bytes(128, 2, 1, 64, 64, 1) == 0 and lib.nplm_linattn_bounds_bytes(129, 2, 1, 64, 64, 1) > 0
    assert lib.nplm_linattn_bounds_bytes(65, 2, 1, 129, 64, 1) == 0 and lib.nplm_linattn_bwd_workspace_bytes(65, 0, 1, 64, 64, 1) == 0
    for args in ((100, 2, 3, 64, 128, 1), (131072, 16, 490, 64, 64, 1), (10 ** 6, 4, 1, 128, 128, 0)):
        b, w = lib.nplm_linattn_bounds_bytes(*args), lib.nplm_linattn_bwd_workspace_bytes(*args)
        assert b % 256 == 0 and w % 256 == 0 and w > b


# ---- Python surface -----------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    q, v, g, cu = torch.randn(5, 2, 4), torch.randn(5, 2, 3), torch.randn(2), torch.tensor([0, 5], dtype=torch.int32)
    for call in (lambda: npa.varlen_linear_attention(q, q, v, cu, g), lambda: npa.VarlenLinearAttention(2)(q, q, v, cu),
                 lambda: npa.linear_attention_step(q, q, v, g, torch.zeros(5, 2, 4, 3)), lambda: npa.layer_norm(q[:, 0]), lambda: npa.LayerNorm(4)(q[:, 0])):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_modules_and_their_parameters():
    m = npa.VarlenLinearAttention(8)
    kept = torch.sigmoid(m.decay.detach().double())
    assert m.decay.shape == (8,) and abs(float(kept[0]) - (1 - 2 ** -5)) < 1e-6 and abs(float(kept[-1]) - (1 - 2 ** -9)) < 1e-6
    assert m.log_decay().shape == (8,) and m.log_decay(torch.zeros(3, 8)).shape == (3, 8) and bool((m.log_decay() < 0).all())
    assert npa.VarlenLinearAttention(1, dtype=torch.bfloat16).decay.dtype == torch.bfloat16
    for bad in (dict(heads=0), dict(heads=2, scale=float("nan"))):
        with pytest.raises(ValueError):
            npa.VarlenLinearAttention(**bad)
    with pytest.raises(RuntimeError, match="no next token"):
        npa.VarlenLinearAttention(2, reverse=True).step(*(torch.zeros(1, 2, 4),) * 3, torch.zeros(1, 2, 4, 4))
    shapes = lambda **k: {n: tuple(t.shape) for n, t in npa.LayerNorm(12, **k).named_parameters()}
    assert shapes() == {"weight": (12,)} and shapes(bias=True, heads=3, shared=True) == {"weight": (4,), "bias": (4,)}
    for bad in (dict(norm="batch"), dict(heads=5), dict(heads=0), dict(channels=0), dict(channels=16385)):
        with pytest.raises(ValueError):
            npa.LayerNorm(**{"channels": 12, **bad})


def test_refusals_that_come_before_the_device_is_looked_at():
    q, cu = torch.zeros(5, 2, 4), torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="3-D"):
        npa.varlen_linear_attention(q[0], q, q, cu, torch.zeros(2))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        npa.varlen_linear_attention(q.half(), q, q, cu, torch.zeros(2))
    with pytest.raises(ValueError, match="3-D"):
        npa.linear_attention_step(q[0], q, q, torch.zeros(2), torch.zeros(5, 2, 4, 4))
    with pytest.raises(ValueError, match="2-D"):
        npa.layer_norm(q)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        npa.layer_norm(q[0].half())


def test_recorded_calls_are_registered_ops(monkeypatch):
    """With fake tensors, whose outputs are known by shape and dtype alone, under the recorder of torch.fx."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setattr(_lib, "load_node", lambda: _lib._NoNode)
    z = lambda *s, d=torch.float32: torch.empty(*s, dtype=d, device="cuda")
    inputs = lambda: (z(300, 2, 4), z(300, 2, 6), z(3, d=torch.int32), z(300, 2), z(2, 2, 4, 6), z(300, 2, 4, 6), z(6))

    def f(q, v, cu, g, h0, table, w):
        o, state = npa.varlen_linear_attention(q, q, v, cu, g, initial_state=h0, return_state=True)
        y = npa.layer_norm(o.flatten(1), w, gate=v.flatten(1), heads=2, norm="rms")
        return y, state, npa.linear_attention_step(q, q, v, g, table), npa.linear_attention_step(q, q, v, g, table, out_state=table + 1)
    with FakeTensorMode(allow_non_fake_inputs=True):
        assert [tuple(t.shape) for t in f(*inputs())] == [(300, 12), (2, 2, 4, 6), (300, 2, 6), (300, 2, 6)]
        graph = make_fx(f, tracing_mode="fake")(*inputs()).graph
    names = [str(n.target).split(".")[1] for n in graph.nodes if n.op == "call_function" and str(n.target).startswith("nanoplm_amd.")]
    assert names == ["varlen_linear_attention_fwd", "layer_norm_fwd", "linear_attention_step", "linear_attention_step_to"]


def test_bounds_of_the_registered_op_are_enough():
    """The op's fake has no value of S to ask the library with: what it takes must cover all of them, and not much more where it matters."""
    from nanoplm_amd import linattn
    for T in (0, 1, 64, 129, 2048, 2049, 5003, 20011, 32768, 131072, 10 ** 6, 2 ** 27):
        for H in (1, 3, 7, 16, 64, 511, 512, 513, 3000):
            for dk, dv in ((1, 1), (64, 128), (91, 91)):
                most = linattn._most_bounds_bytes(T, H, dk, dv)
                for S in (0, 1, 2, 5, 31, 100, 490, 513, 4000):
                    assert linattn._bounds_bytes(T, H, S, dk, dv, 1) <= most, (T, H, S, dk, dv)
                assert most <= (512 + H * (T // 2048 + 1)) * (dk * dv + 1) * 4 + 512


def test_fakes_keep_symbolic_sizes(monkeypatch):
    """Rows and sequences of a packed batch change from step to step: a compiled model must not be made for one of each."""
    from torch._dynamo.source import ConstantSource
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext
    monkeypatch.setattr(_lib, "load_node", lambda: _lib._NoNode)
    env = ShapeEnv()
    size = lambda n, name: env.create_symintnode(env.create_symbol(n, ConstantSource(name), dynamic_dim=DimDynamic.DYNAMIC), hint=n, source=ConstantSource(name))
    with FakeTensorMode(shape_env=env, allow_non_fake_inputs=True):
        T, S = size(3001, "T"), size(6, "S")
        z = lambda *s, d=torch.float32: torch.empty(*s, dtype=d, device="cuda")
        q, v, g, cu, h0 = z(T, 2, 4), z(T, 2, 6), z(T, 2), z(S + 1, d=torch.int32), z(S, 2, 4, 6)
        o, state, bounds = npa.varlen_linear_attention_fwd_op(q, q, v, cu, g, h0, None, False, True)
        npa.varlen_linear_attention_bwd_op(q, q, v, o, cu, g, bounds, h0, state, state, None, False, True, True)
        npa.layer_norm_bwd_op(v.flatten(1), z(6), None, v.flatten(1), o.flatten(1), 2, "rms", 1e-5, True)
    assert not env.replacements, env.replacements
    assert not any("Eq" in str(guard.expr) for guard in env.guards), [str(guard.expr) for guard in env.guards]
    assert all(isinstance(t.shape[0], torch.SymInt) for t in (o, state, bounds))


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(monkeypatch, grad):
    """Refused, not dropped: the derivative would read as zero."""
    import torch.autograd.forward_ad as forward_ad
    monkeypatch.setattr(_lib, "load_node", lambda: _lib._NoNode)
    q, v, g, cu, table = torch.randn(5, 2, 4), torch.randn(5, 2, 3), -torch.ones(5, 2), torch.tensor([0, 5], dtype=torch.int32), torch.zeros(5, 2, 4, 3)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: npa.varlen_linear_attention(dual(q), q, v, cu, g), lambda: npa.varlen_linear_attention(q, q, v, cu, dual(g)),
                     lambda: npa.varlen_linear_attention(q, q, v, cu, g, initial_state=dual(table[:1])), lambda: npa.linear_attention_step(q, q, dual(v), g, table),
                     lambda: npa.linear_attention_step(q, q, v, g, dual(table)), lambda: npa.layer_norm(dual(q[:, 0])), lambda: npa.layer_norm(q[:, 0], dual(q[0, 0]))):
            with pytest.raises(NotImplementedError):
                call()
