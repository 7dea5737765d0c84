"""Forms of call of the recurrence, its step and the residual norm that the block's own tests do not make: forward mode, recorded calls, negated views, tables that share memory, second derivatives."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nanoplm_amd as npa

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _inputs(T=300, C=70, act=F32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s, d=act: torch.randn(*s, device="cuda", generator=g).to(d)
    return dict(x=n(T, C), gates=n(T, 2 * C), cu=torch.tensor([0, 100, 100, T], dtype=torch.int32, device="cuda"), decay=n(C, d=F32) - 4, h0=n(3, C, d=F32),
                gate=n(T, C), weight=n(C, d=F32), table=n(T + 5, C, d=F32))


def _calls(i, table=None):
    table = i["table"].clone() if table is None else table
    return {"recurrence": lambda: npa.varlen_recurrence(i["x"], i["gates"], i["cu"], i["decay"], initial_state=i["h0"], return_state=True),
            "norm": lambda: npa.residual_norm(i["x"], i["x"], i["gate"], pre_weight=i["weight"]),
            "step": lambda: (npa.recurrence_step(i["x"], i["gates"], i["decay"], table),)}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["recurrence", "norm", "step"])
def test_forward_mode_is_refused(name, grad):
    i = _inputs()
    for which in ("x", "gates", "decay", "h0", "gate", "weight"):
        used = {"recurrence": ("x", "gates", "decay", "h0"), "norm": ("x", "gate", "weight"), "step": ("x", "gates", "decay")}[name]
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            call = _calls({**i, which: forward_ad.make_dual(i[which], torch.ones_like(i[which]))})[name]
            if which in used:
                with pytest.raises(NotImplementedError):
                    call()
            else:
                call()
    want = _calls(i)[name]()
    with forward_ad.dual_level():
        got = _calls(i)[name]()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def _recordable(i):
    """(name, function of tensors, its arguments): every form whose launches nothing but a registered op shows to a recorder."""
    slots = torch.arange(len(i["x"]), dtype=torch.int32, device="cuda").flip(0)
    return {"recurrence": (lambda x, g, d: npa.varlen_recurrence(x, g, i["cu"], d), (i["x"], i["gates"], i["decay"])),
            "states": (lambda x, g, d, h: npa.varlen_recurrence(x, g, i["cu"], d, initial_state=h, reverse=True, return_state=True),
                       (i["x"], i["gates"], i["decay"], i["h0"])),
            "norm": (lambda u, r, g, w: npa.residual_norm(u, r, g, pre_weight=w, norm="rms"), (i["x"], i["x"], i["gate"], i["weight"])),
            "stream": (lambda u, r: npa.residual_norm(u, r)[0], (i["x"], i["x"])),
            "step": (lambda x, g, d, t: npa.recurrence_step(x, g, d, t, slots), (i["x"], i["gates"], i["decay"], i["table"])),
            "step_to": (lambda x, g, d, t, o: npa.recurrence_step(x, g, d, t, out_state=o), (i["x"], i["gates"], i["decay"], i["table"], i["table"] * 2))}


def _listed(out):
    return list(out) if isinstance(out, tuple) else [out]


@pytest.mark.parametrize("record", ["jit.trace", "make_fx"])
@pytest.mark.parametrize("name", ["recurrence", "states", "norm", "stream", "step", "step_to"])
def test_a_recorded_call_follows_the_inputs_of_the_replay(name, record):
    """Recorded with one set of inputs and replayed with others, outputs and changed tables are the eager call's."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, example = _recordable(_inputs())[name]
    example = tuple(t.clone() for t in example)
    recorded = torch.jit.trace(f, example, check_trace=False) if record == "jit.trace" else make_fx(f)(*example)
    for seed in (1, 2):
        args = _recordable({**_inputs(seed=seed), "cu": _inputs()["cu"]})[name][1]
        mine, its = tuple(t.clone() for t in args), tuple(t.clone() for t in args)
        want, got = _listed(f(*mine)), _listed(recorded(*its))
        torch.full((1 << 20,), float("nan"), device="cuda")          # (what a block that nothing filled may hold)
        assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a, b) for a, b in zip(mine, its))


@pytest.mark.parametrize("name", ["states", "norm"])
def test_a_recorded_call_is_differentiable(name):
    f, example = _recordable(_inputs())[name]
    leaves = [t.clone().requires_grad_() for t in example]
    traced = torch.jit.trace(f, tuple(leaves), check_trace=False)
    results = []
    for call in (f, traced):
        outs = _listed(call(*leaves))
        results.append(outs + list(torch.autograd.grad(sum((o * o).sum() for o in outs), leaves)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_views_that_negate_their_values_are_read_as_they_say():
    i = _inputs(act=BF16)
    for which in ("x", "gates", "decay", "h0", "gate", "weight"):
        neg = {**i, which: torch._neg_view(-i[which])}
        for name, call in _calls(neg).items():
            assert all(torch.equal(a, b) for a, b in zip(call(), _calls(i)[name]())), (which, name)
    dy = torch.randn(300, 70, device="cuda").bfloat16()
    leaves = [i[k].clone().requires_grad_() for k in ("x", "gates", "decay", "h0")]
    grads = [torch.autograd.grad(npa.varlen_recurrence(leaves[0], leaves[1], i["cu"], leaves[2], initial_state=leaves[3]), leaves, d)
             for d in (dy, torch._neg_view(-dy))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    raw = [npa.varlen_recurrence_bwd(i["x"], i["gates"], d, i["cu"], i["decay"], npa.varlen_recurrence_fwd(
        i["x"], i["gates"], i["cu"], i["decay"], want_carries=True)[2]) for d in (dy, torch._neg_view(-dy))]
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(*raw))


def test_tables_of_a_step_are_one_or_apart():
    i, both = _inputs(), torch.randn(700, 70, device="cuda")
    old = both.clone()
    for state, out in ((both[:310], both[1:311]), (both[300:], both[:400])):
        with pytest.raises(ValueError, match="shares some of its memory"):
            npa.recurrence_step(i["x"], i["gates"], i["decay"], state, out_state=out)
    assert torch.equal(both, old)
    y = npa.recurrence_step(i["x"], i["gates"], i["decay"], both[:350], out_state=both[350:])
    assert torch.equal(both[:350], old[:350]) and torch.equal(both[650:], old[650:])
    assert torch.equal(y, npa.recurrence_step(i["x"], i["gates"], i["decay"], both[:350], out_state=both.view(-1)[:350 * 70].view(350, 70)))
    assert torch.equal(both[:300], both[350:650])


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["recurrence", "norm"])
def test_the_first_derivative_under_create_graph_and_no_second(name, native):
    i = _inputs()
    x, decay = i["x"].requires_grad_(), i["decay"].requires_grad_()
    call = {("recurrence", True): lambda: npa.varlen_recurrence(x, i["gates"], i["cu"], decay),
            ("recurrence", False): lambda: npa.VarlenRecurrenceFunction.apply(x, i["gates"], i["cu"], decay)[0],
            ("norm", True): lambda: npa.residual_norm(x, x, scale=decay)[0],
            ("norm", False): lambda: npa.ResidualNormFunction.apply(x, x, None, None, None, decay, None, None, "layer", 1e-5)[0]}[name, native]
    want = torch.autograd.grad(call().square().sum(), [x, decay])
    got = torch.autograd.grad(call().square().sum(), [x, decay], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and got[0].requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula" if native else "once_differentiable"):
        got[0].sum().backward()


def test_a_module_steps_under_no_grad():
    i, m = _inputs(), npa.VarlenRecurrence(70).cuda()
    table = i["table"].clone()
    with pytest.raises(RuntimeError, match="call it under torch.no_grad"):
        m.step(i["x"], i["gates"], table)
    assert torch.equal(table, i["table"])
    with torch.no_grad():
        y = m.step(i["x"], i["gates"], table)
    assert torch.equal(y, table[:300])


@pytest.mark.parametrize("kind", ["once", "four times", "by halves"])
def test_thousands_of_rows_that_name_slots(kind):
    """Rows of one slot in their order, whatever lies between: the same as steps of one row of each slot, one step after the other, bit for bit."""
    B, C, N = 6001, 70, 9000
    g = torch.Generator("cuda").manual_seed(1)
    x, gates, decay, table = (torch.randn(*s, device="cuda", generator=g) for s in ((B, C), (B, 2 * C), (C,), (N, C)))
    slots = torch.randperm(N, device="cuda", generator=g)[:B].int()
    if kind == "four times":
        slots = slots[torch.arange(B, device="cuda") % 1501]
    elif kind == "by halves":
        slots[3000:] = slots[:3001].flip(0)
    slots[7::97] = -1
    want_table, want = table.clone(), torch.zeros(B, C, device="cuda")
    seen, turns = {}, []
    for b, s in enumerate(slots.tolist()):             # (row b is its slot's turn-th)
        turns.append(seen.get(s, 0) if s >= 0 else -1)
        seen[s] = seen.get(s, 0) + 1
    turns = torch.tensor(turns, device="cuda")
    for turn in range(int(turns.max()) + 1):
        rows = (turns == turn).nonzero()[:, 0]
        want[rows] = npa.recurrence_step(x[rows], gates[rows], decay, want_table, slots[rows])
    for out in (None, table.clone()):
        state = table.clone()
        y = npa.recurrence_step(x, gates, decay, state, slots, out_state=out)
        assert torch.equal(y, want) and torch.equal(state if out is None else out, want_table)
        assert out is None or torch.equal(state, table)


def test_the_usage_example_runs_as_it_stands():
    import os
    import re
    source = re.search(r"```python\n(.*?)```", open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read(), re.S)[1]
    T, C = 1000, 1024
    b = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    names = dict(x=b(T, C).requires_grad_(), dy=b(T, C), z=b(T, 2 * C), u=b(T, C), gates=b(T, 2 * C), gate=b(T, C), norm=torch.nn.LayerNorm(C).cuda().bfloat16(),
                 cu_seqlens=torch.tensor([0, 400, T], dtype=torch.int32, device="cuda"), u_t=b(2, C), gates_t=b(2, 2 * C), states=torch.zeros(9, C, device="cuda"),
                 slots=torch.tensor([3, 1], dtype=torch.int32, device="cuda"))
    exec(source, names)
    assert names["y"].shape == (2, C) and names["normed"].shape == (T, C) and names["state"].shape == (2, C) and bool(names["states"][3].any())
