"""Forms of call of the recurrence, its step and the residual norm, on the CPU: the Python route drives a stand-in for the library that fills every output it is
given with what it read (so that a tensor that nothing filled, or that was read the wrong way, shows)."""
import contextlib
import ctypes
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nanoplm_amd as npa
from nanoplm_amd import _lib, recurrence, resnorm


def _at(address, n):
    return torch.frombuffer((ctypes.c_float * n).from_address(address), dtype=torch.float32)


class _HostLib:
    """y = x, state = 3, the step's new states = 2 x; stream = u + residual, normed = u. All tensors fp32, [T, C] contiguous."""
    nplm_recurrence_fwd_workspace_bytes = nplm_resnorm_bwd_workspace_bytes = staticmethod(lambda *a: 0)

    def nplm_recurrence_fwd(self, x, xs, gates, gs, cu, decay, scale, initial, y, state, carries, ws, wsb, T, C, S, *rest):
        _at(y, T * C).copy_(_at(x, T * C))
        if state is not None:
            _at(state, S * C).fill_(3.0)
        return 0

    def nplm_recurrence_step(self, x, xs, gates, gs, decay, scale, state, out_state, slots, y, B, C, N, *rest):
        _at(y, B * C).copy_(_at(x, B * C))
        _at(out_state, B * C).copy_(2 * _at(x, B * C))
        return 0

    def nplm_resnorm_fwd(self, u, us, gate, gs, residual, rs, pw, pb, scale, qw, qb, eps, out, normed, stats, T, C, *rest):
        _at(out, T * C).copy_(_at(u, T * C) + _at(residual, T * C))
        if normed is not None:
            _at(normed, T * C).copy_(_at(u, T * C))
        return 0


@pytest.fixture
def host(monkeypatch):
    lib = _HostLib()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "load_node", lambda: _lib._NoNode)
    for module in (recurrence, resnorm):
        monkeypatch.setattr(module, "_launch_on", lambda t: contextlib.nullcontext(SimpleNamespace(stream=None)))
    monkeypatch.setattr(recurrence, "_check_rows", lambda x, gates, decay, name: tuple(x.shape))
    monkeypatch.setattr(recurrence, "_check", lambda x, gates, cu, *rest: (*x.shape, cu.numel() - 1))
    monkeypatch.setattr(resnorm, "_check", lambda u, *rest: tuple(u.shape))
    return lib


CU = torch.tensor([0, 4], dtype=torch.int32)


def _calls(x):
    """Every function on inputs made of x [4, 3]: its outputs."""
    gates, decay = torch.cat([x, x], 1), torch.zeros(3)
    return {"recurrence": lambda: npa.varlen_recurrence(x, gates, CU, decay, return_state=True),
            "step": lambda: (npa.recurrence_step(x, gates, decay, torch.zeros(4, 3)),),
            "norm": lambda: npa.residual_norm(x, x, pre_weight=torch.ones(3))}


def test_the_stand_in_answers(host):
    x = torch.randn(4, 3)
    calls = {k: f() for k, f in _calls(x).items()}
    assert torch.equal(calls["recurrence"][0], x) and bool((calls["recurrence"][1] == 3).all())
    assert torch.equal(calls["step"][0], x) and torch.equal(calls["norm"][0], 2 * x) and torch.equal(calls["norm"][1], x)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["recurrence", "step", "norm"])
def test_forward_mode_is_refused(host, name, grad):
    """A tangent is refused, not dropped: the derivative would read as zero."""
    x, t = torch.randn(4, 3), torch.randn(4, 3)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError):
            _calls(forward_ad.make_dual(x, t))[name]()
        _calls(x)[name]()                                # (a level alone is none)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda x: _calls(x)[name]()[0], (x,), (t,))


@pytest.mark.parametrize("which", ["gates", "decay", "state", "out_state"])
def test_every_tangent_of_a_step_is_refused(host, which):
    args = dict(x=torch.randn(4, 3), gates=torch.randn(4, 6), decay=torch.zeros(3), state=torch.zeros(4, 3), out_state=torch.zeros(4, 3))
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            npa.recurrence_step(**args)


def test_a_frozen_call_on_the_python_route_keeps_nothing_for_a_backward(host, monkeypatch):
    seen = []
    for module, name, what in ((recurrence, "varlen_recurrence_fwd", "want_carries"), (resnorm, "residual_norm_fwd", "want_stats")):
        raw = getattr(module, name)
        monkeypatch.setattr(module, name, lambda *a, raw=raw, what=what, **k: seen.append(k[what]) or raw(*a, **k))
    for x in (torch.randn(4, 3), torch.randn(4, 3, requires_grad=True)):
        _calls(x)["recurrence"](), _calls(x)["norm"]()
    assert seen == [False, False, True, True]


def _fake_inputs():
    z = lambda *s, d=torch.float32: torch.empty(*s, dtype=d, device="cuda")
    return z(4, 3), z(4, 6), z(3, d=torch.int32), z(3), z(2, 3), z(4, 3), z(9, 3)


def test_recorded_calls_are_registered_ops():
    """Where something records operations, it has to see the call itself: the library's launch is invisible to it. With fake tensors, whose outputs are known
    by shape and dtype alone, under the recorder of torch.fx."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x, gates, cu, decay, h0, gate, table):
        y, state = npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0, return_state=True)
        stream, normed = npa.residual_norm(y, x, gate, pre_weight=decay)
        (last, none) = npa.residual_norm(normed, stream)
        assert none is None
        return last, state, npa.recurrence_step(x, gates, decay, table), npa.recurrence_step(x, gates, decay, table, out_state=table + 1)
    with FakeTensorMode(allow_non_fake_inputs=True):
        out = f(*_fake_inputs())
        assert [tuple(t.shape) for t in out] == [(4, 3), (2, 3), (4, 3), (4, 3)]
        graph = make_fx(f, tracing_mode="fake")(*_fake_inputs()).graph
    names = [str(n.target).split(".")[1] for n in graph.nodes if n.op == "call_function" and str(n.target).startswith("nanoplm_amd.")]
    assert names == ["varlen_recurrence_fwd", "residual_norm_fwd", "residual_norm_fwd", "recurrence_step", "recurrence_step_to"]


def test_recorded_calls_refuse_what_others_refuse():
    """A registered op without a rule for it would drop a tangent, and let a gradient through a step only to fail in the backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, gates, cu, decay, h0, gate, table = _fake_inputs()
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            for call in (lambda: npa.varlen_recurrence(dual, gates, cu, decay), lambda: npa.residual_norm(x, dual), lambda: npa.recurrence_step(dual, gates, decay, table)):
                with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                    call()
        with pytest.raises(RuntimeError, match="no gradient"):
            npa.recurrence_step(x.requires_grad_(), gates, decay, table)


def test_views_that_negate_their_values_are_read_as_they_say(host):
    """(x.conj().imag is one: its memory holds the other sign.)"""
    x = torch.randn(4, 3)
    neg = torch._neg_view(-x)
    assert neg.is_neg() and torch.equal(neg, x)
    for name, call in _calls(neg).items():
        assert all(torch.equal(a, b) for a, b in zip(call(), _calls(x)[name]())), name
    for grad in (torch.enable_grad, torch.no_grad):
        with grad():
            assert torch.equal(npa.varlen_recurrence(neg, torch.zeros(4, 6), CU, torch.zeros(3)), x)
    for which in ("state", "out_state"):
        tables = {"state": torch.zeros(4, 3), "out_state": torch.zeros(4, 3)}
        tables[which] = torch._neg_view(tables[which])
        with pytest.raises(ValueError, match="contiguous float32 table"):
            npa.recurrence_step(x, torch.zeros(4, 6), torch.zeros(3), **tables)


def test_tables_of_a_step_are_one_or_apart(host):
    x, gates, decay = torch.ones(4, 3), torch.zeros(4, 6), torch.zeros(3)
    both = torch.zeros(9, 3)
    for state, out in ((both[:5], both[1:6]), (both[4:], both[:5])):
        with pytest.raises(ValueError, match="shares some of its memory"):
            npa.recurrence_step(x, gates, decay, state, out_state=out)
    assert not bool(both.any())
    npa.recurrence_step(x, gates, decay, both[:4], out_state=both[4:8])
    assert not bool(both[:4].any()) and bool((both[4:8] == 2).all()) and not bool(both[8:].any())
    npa.recurrence_step(x, gates, decay, both[:4], out_state=both.view(-1)[:12].view(4, 3))
    assert bool((both[:8] == 2).all())


@pytest.mark.parametrize("C", [16, 64, 768, 1024, 2050, 4096, 16384])
def test_no_lane_adds_up_more_rows_than_fp32_is_good_for(C):
    """The workspace has five sums a channel and block: no more than 4096 rows a lane, whatever the number of rows."""
    lib = _lib.load()
    lanes = 8
    while lanes * (8 if C <= 8192 else 16) < C:
        lanes *= 2
    rows = max(256 // lanes, 1)
    for T in (1, 5000, 131072, 2200000, 2 ** 31 - 2 ** 20 - 1):
        blocks = lib.nplm_resnorm_bwd_workspace_bytes(T, C) // (5 * 4 * C)
        steps = -(-T // rows)
        assert blocks >= 1 and -(-steps // blocks) <= 4096, (T, blocks)


def test_a_module_steps_under_no_grad(host):
    m, x, table = npa.VarlenRecurrence(3), torch.randn(4, 3), torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match="call it under torch.no_grad"):
        m.step(x, torch.zeros(4, 6), table)
    assert not bool(table.any())
    with torch.no_grad():
        assert torch.equal(m.step(x, torch.zeros(4, 6), table), x) and torch.equal(table, 2 * x)


def test_rows_that_name_slots_are_bounded(host):
    """Each of them looks through all of them: millions would hold the GPU for hours."""
    n = 2 ** 18 + 1
    big = torch.empty(n, 3)
    with pytest.raises(ValueError, match="at most 262144 rows"):
        npa.recurrence_step(big, torch.empty(n, 6), torch.zeros(3), torch.empty(n, 3), torch.zeros(n, dtype=torch.int32))
    npa.recurrence_step(big, torch.empty(n, 6), torch.zeros(3), torch.empty(n, 3))


def test_the_library_bounds_rows_that_name_slots():
    lib, at = _lib.load(), 0x10000                     # (an address that nothing reads: refused before a launch)
    step = lambda B, slots: lib.nplm_recurrence_step(at, 64, at, 128, at, 8.0, at, at, slots, at, B, 64, 2 ** 25, 1, 1, None)
    assert step(2 ** 18 + 1, at) == -2 and step(2 ** 24, None) == -2
