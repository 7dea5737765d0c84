"""The packed recurrent block: pre-norm conv, gated linear recurrence and residual norm as a layer uses them together; refusals on device tensors."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import nanoplm_amd as npa
from tests import recurrence_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


class Block(nn.Module):
    """normed rows -> projection -> short conv -> gates -> recurrence (both directions) -> gated norm, residual and the next block's norm."""

    def __init__(self, C):
        super().__init__()
        self.proj, self.to_gates = nn.Linear(C, 2 * C, bias=False), nn.Linear(C, 2 * C)
        self.conv = npa.VarlenDWConv1d(C, 5, residual=True)
        self.left, self.right = npa.VarlenRecurrence(C), npa.VarlenRecurrence(C, reverse=True)
        self.join = npa.ResidualNorm(C, norm="rms", scale_init=0.5)

    def forward(self, stream, normed, cu):
        x, gate = self.proj(normed).chunk(2, dim=-1)
        x = self.conv(x, cu)
        gates = self.to_gates(x)
        return self.join(self.left(x, gates, cu) + self.right(x, gates, cu), stream, gate)


def _reference(block, stream, normed, cu, lens):
    """The same in fp64 on the CPU, differentiable."""
    C = normed.shape[1]
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in block.named_parameters()}
    s, x0 = stream.detach().cpu().double().requires_grad_(), normed.detach().cpu().double().requires_grad_()
    x, gate = (x0 @ p["proj.weight"].t()).chunk(2, dim=-1)
    rows = []
    for part in x.split(lens):
        y = F.conv1d(part.t()[None], p["conv.weight"][:, None], p["conv.bias"], padding=2, groups=C)[0].t() if part.shape[0] else part
        rows.append(part + y)
    x = torch.cat(rows)
    gates = x @ p["to_gates.weight"].t() + p["to_gates.bias"]
    u = torch.zeros_like(x)
    for name, reverse in (("left", False), ("right", True)):
        k = R.coefficients(x, gates, p[f"{name}.decay"], 8.0)
        out = [None] * x.shape[0]
        for lo, hi, _ in R.sequences(cu.cpu(), x.shape[0]):
            h = torch.zeros(C, dtype=torch.float64)
            for t in range(hi - 1, lo - 1, -1) if reverse else range(lo, hi):
                h = k["a"][t] * h + k["b"][t]
                out[t] = h
        u = u + torch.stack(out)
    rms = lambda a: a / torch.sqrt((a * a).mean(1, keepdim=True) + 1e-5)
    new = s + p["join.scale"] * rms(u) * p["join.post_weight"] * F.silu(gate)
    return (new, rms(new) * p["join.pre_weight"]), [s, x0] + list(p.values())


def test_a_block_and_its_gradients():
    """fp32 against fp64. Each of the eight steps in either direction leaves at most about 32 roundings of 2^-24 (2e-6) on its terms, and none gains
    more than a few times: 1e-4 of a tensor's norm."""
    torch.manual_seed(0)
    C, lens = 48, [70, 0, 1, 130, 64, 5]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    T = sum(lens)
    block = Block(C).cuda()
    stream, normed = torch.randn(T, C, device="cuda", requires_grad=True), torch.randn(T, C, device="cuda", requires_grad=True)
    d = [torch.randn(T, C, device="cuda") for _ in range(2)]
    want, leaves = _reference(block, stream, normed, cu, lens)
    wgrads = torch.autograd.grad(want, leaves, [t.cpu().double() for t in d])
    out = block(stream, normed, cu)
    grads = torch.autograd.grad(out, [stream, normed] + list(block.parameters()), d)
    for name, a, b in zip(["stream", "normed", "d stream", "d normed"] + [n for n, _ in block.named_parameters()], list(out) + list(grads), list(want) + list(wgrads)):
        off = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 1e-4, (name, off)


def test_two_blocks_under_autocast_compiled_and_replayed():
    """bf16 branches on an fp32 stream, two blocks chained through (stream, normed): eager, compiled, and captured with its backward into a graph."""
    torch.manual_seed(1)
    C, lens = 128, [300, 17, 0, 500, 207]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    T = sum(lens)
    blocks = nn.ModuleList([Block(C), Block(C)]).cuda()
    stream, normed = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda")
    params = list(blocks.parameters())

    def step(stream, normed):
        with torch.autocast("cuda", BF16, cache_enabled=False):
            for b in blocks:
                stream, normed = b(stream, normed, cu)
        assert stream.dtype == F32
        loss = stream.square().mean() + normed.float().square().mean()
        return [loss.detach(), stream.detach()] + list(torch.autograd.grad(loss, params))
    want = [t.clone() for t in step(stream, normed)]
    assert all(bool(torch.isfinite(t).all()) for t in want)
    got = torch.compile(step, dynamic=False, backend="aot_eager")(stream, normed)
    assert all(torch.equal(a, b) for a, b in zip(want[:2], got[:2]))
    del got
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(stream, normed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(stream, normed)
    for k in range(3):
        stream.normal_()
        graph.replay()
        torch.cuda.synchronize()
        # the stream, which no library sum over blocks had a part in
        assert torch.equal(step(stream, normed)[1], outs[1]), k


def test_two_calls_at_once_on_two_streams():
    g = torch.Generator("cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    T, C = 5000, 256
    cu = torch.tensor([0, 100, 4700, T], dtype=torch.int32).cuda()
    ins = [[n(T, C), n(T, 2 * C), n(C), n(T, C)] for _ in range(2)]

    def call(x, gates, decay, dy):
        y, _, carries = npa.varlen_recurrence_fwd(x, gates, cu, decay, want_carries=True)
        out = npa.varlen_recurrence_bwd(x, gates, dy, cu, decay, carries)
        stream, normed, stats = npa.residual_norm_fwd(y, x, dy, decay, pre_weight=decay, want_stats=True)
        return [y, *out[:3], stream, normed, *[t for t in npa.residual_norm_bwd(y, x, dy, decay, None, None, decay, stats, dy, x) if t is not None]]
    want = [call(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, i in zip(streams, ins):
            with torch.cuda.stream(s):
                got.append(call(*i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_recurrence_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    cu = torch.tensor([0, 5], dtype=torch.int32).cuda()
    good = dict(x=z(5, 4), gates=z(5, 8), cu_seqlens=cu, decay=z(4))
    npa.varlen_recurrence(**good)
    for bad, err in [(dict(gates=z(5, 7)), ValueError), (dict(gates=z(4, 8)), ValueError), (dict(gates=z(5, 8, d=BF16)), TypeError), (dict(decay=z(5)), ValueError),
                     (dict(decay=z(4, d=torch.float16)), TypeError), (dict(cu_seqlens=cu.long()), TypeError), (dict(cu_seqlens=cu[:0]), TypeError),
                     (dict(cu_seqlens=cu.cpu()), RuntimeError), (dict(gates=z(5, 8).cpu()), RuntimeError), (dict(decay=z(4).cpu()), RuntimeError),
                     (dict(x=z(5, 0), gates=z(5, 0), decay=z(0)), ValueError), (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError),
                     (dict(initial_state=z(2, 4)), ValueError), (dict(initial_state=z(1, 4, d=BF16)), ValueError),
                     (dict(initial_state=z(1, 4).cpu()), RuntimeError)]:
        with pytest.raises(err):
            npa.varlen_recurrence(**{**good, **bad})
    _, _, carries = npa.varlen_recurrence_fwd(**good, want_carries=True)
    args = (good["x"], good["gates"], z(5, 4), cu, good["decay"])
    npa.varlen_recurrence_bwd(*args, carries)
    for a, c, k in ((args, None, {}), (args, carries[:, :3], {}), (args, carries, dict(dstate=z(3, 4))), (args[:2] + (z(5, 4, d=BF16),) + args[3:], carries, {})):
        with pytest.raises(ValueError):
            npa.varlen_recurrence_bwd(*a, c, **k)


def test_a_step_is_a_change_that_autograd_sees():
    z = lambda *s: torch.randn(*s, device="cuda")
    x, gates, decay, table = z(3, 70), z(3, 140), z(70) - 4, z(5, 70)
    cu = torch.tensor([0, 1, 2, 2, 2, 3], dtype=torch.int32, device="cuda")
    for route in (lambda: npa.recurrence_step(x, gates, decay, table, slots), lambda: npa.recurrence_step(x, gates.t().contiguous().t(), decay, table, slots)):
        slots = torch.tensor([0, 4, 2], dtype=torch.int32, device="cuda")
        leaf = x.clone().requires_grad_()
        y = npa.varlen_recurrence(leaf, gates, cu, decay, initial_state=table)
        before = table._version
        route()
        assert table._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        t = table.clone()
        npa.recurrence_step(x, gates, decay, t, slots)
    npa.recurrence_step(x, gates, decay, t, slots)


@pytest.mark.parametrize("apart", [False, True])
def test_a_step_in_a_compiled_model(apart):
    z = lambda *s: torch.randn(*s, device="cuda")
    x, gates, decay = z(3, 70), z(3, 140), z(70) - 4
    slots = torch.tensor([0, 4, -1], dtype=torch.int32, device="cuda")

    def f(x, gates, table, other):
        y = npa.recurrence_step(x * 2, gates, decay, table, slots, out_state=other if apart else None)
        y = y + npa.recurrence_step(x, gates, decay, table, slots, out_state=other if apart else table)
        return y, table.sum(), other.sum()
    a, b = z(5, 70), z(5, 70)
    a2, b2 = a.clone(), b.clone()
    with torch.no_grad():
        want = f(x, gates, a, b)
        got = torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")(x, gates, a2, b2)
        assert all(torch.equal(p, q) for p, q in zip(want, got)) and torch.equal(a, a2) and torch.equal(b, b2)
        torch.library.opcheck(npa.recurrence.recurrence_step_op, (x, gates, decay, a, slots, 8.0))
        torch.library.opcheck(npa.recurrence.recurrence_step_to_op, (x, gates, decay, a, None if apart else slots, 8.0, b))


def test_step_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(x=z(5, 4), gates=z(5, 8), decay=z(4), state=z(6, 4), slots=z(5, d=torch.int32))
    npa.recurrence_step(**good)
    for bad, err in [(dict(state=z(6, 5)), ValueError), (dict(state=z(6, 4, d=BF16)), ValueError), (dict(state=z(4, 6).t()), ValueError),
                     (dict(out_state=z(5, 4)), ValueError), (dict(slots=z(5, d=torch.int64)), TypeError), (dict(slots=z(4, d=torch.int32)), TypeError),
                     (dict(slots=None, state=z(4, 4)), ValueError), (dict(slots=z(5, d=torch.int32).cpu()), RuntimeError), (dict(state=z(6, 4).cpu()), RuntimeError),
                     (dict(x=z(5, 4).requires_grad_()), RuntimeError)]:
        with pytest.raises(err):
            npa.recurrence_step(**{**good, **bad})
    with torch.no_grad():
        npa.recurrence_step(**{**good, "x": z(5, 4).requires_grad_()})
    assert npa.recurrence_step(z(0, 4), z(0, 8), z(4), z(6, 4)).shape == (0, 4)


def test_residual_norm_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(u=z(5, 4), residual=z(5, 4), gate=z(5, 4), post_weight=z(4), pre_weight=z(4))
    npa.residual_norm(**good)
    for bad, err in [(dict(residual=z(5, 5)), ValueError), (dict(residual=z(5, 4, d=BF16)), TypeError), (dict(gate=z(4, 4)), ValueError),
                     (dict(gate=z(5, 4, d=BF16)), ValueError), (dict(post_weight=z(5)), ValueError), (dict(scale=z(4, d=torch.float16)), TypeError),
                     (dict(post_weight=None, post_bias=z(4)), ValueError), (dict(pre_weight=None, pre_bias=z(4)), ValueError), (dict(norm="none"), ValueError),
                     (dict(eps=-1.0), ValueError), (dict(scale=z(4).cpu()), RuntimeError), (dict(residual=z(5, 4).cpu()), RuntimeError),
                     (dict(u=z(2, 16385), residual=z(2, 16385), gate=None, post_weight=None, pre_weight=None), ValueError)]:
        with pytest.raises(err):
            npa.residual_norm(**{**good, **bad})


# ---- native nodes and the Python Functions ------------------------------------------------------------------------------------------------
def _recurrence_leaves(act, par, states, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s, d=act: torch.randn(*s, device="cuda", generator=g).to(d).requires_grad_()
    T, C, S = 700, 96, 4
    cu = torch.tensor([0, 200, 200, 650, T], dtype=torch.int32).cuda()
    return [n(T, C), n(T, 2 * C), n(C, d=par)], cu, n(S, C, d=F32) if states else None


@pytest.mark.parametrize("act,par", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("states,reverse", [(True, False), (False, True)])
def test_native_recurrence_gives_the_bits_of_the_function(act, par, states, reverse):
    (x, gates, decay), cu, h0 = _recurrence_leaves(act, par, states)
    assert npa._lib.load_node().__name__ == "nanoplm_amd._node"
    leaves = [t for t in (x, gates, decay, h0) if t is not None]
    results = []
    for native in (True, False):
        if native:
            y, state = npa.varlen_recurrence(x, gates, cu, decay, scale=4.0, initial_state=h0, reverse=reverse, return_state=True)
            assert "nanoplm_amd::VarlenRecurrence" in y.grad_fn.name()
        else:
            y, state = npa.VarlenRecurrenceFunction.apply(x, gates, cu, decay, h0, 4.0, reverse, True)
        results.append([y, state, *torch.autograd.grad((y.float() * 1.5).sum() + state.square().sum(), leaves)])
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*results))
    with torch.no_grad():
        y, none = npa.varlen_recurrence(x, gates, cu, decay, scale=4.0, initial_state=h0, reverse=reverse), None
    assert torch.equal(y, results[0][0]) and not y.requires_grad


@pytest.mark.parametrize("act,st,par", [(F32, F32, F32), (BF16, F32, BF16), (BF16, BF16, F32)])
@pytest.mark.parametrize("parts", ["gate post_weight post_bias scale pre_weight pre_bias", "scale pre_weight", "gate post_weight", ""])
def test_native_residual_norm_gives_the_bits_of_the_function(act, st, par, parts):
    g = torch.Generator("cuda").manual_seed(0)
    n = lambda *s, d: torch.randn(*s, device="cuda", generator=g).to(d).requires_grad_()
    T, C = 130, 136
    u, residual = n(T, C, d=act), n(T, C, d=st)
    names = ("gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
    rest = [n(T, C, d=act) if k == "gate" else n(C, d=par) for k in names]
    rest = [t if k in parts.split() else None for k, t in zip(names, rest)]
    leaves = [t for t in (u, residual, *rest) if t is not None]
    results = []
    for call in (lambda: npa.residual_norm(u, residual, *rest, norm="rms", eps=1e-4), lambda: npa.ResidualNormFunction.apply(u, residual, *rest, "rms", 1e-4)):
        stream, normed = call()
        loss = stream.float().square().sum() + (0 if normed is None else (normed.float() * 0.3).sum())
        results.append([t for t in (stream, normed) if t is not None] + list(torch.autograd.grad(loss, leaves)))
    assert len(results[0]) == len(results[1]) and all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*results))
    # parameters in two dtypes, some frozen
    if rest[3] is not None:
        mixed = [t if i != 3 else t.detach().to(BF16 if par == F32 else F32) for i, t in enumerate(rest)]
        a, b = npa.residual_norm(u, residual, *mixed), npa.ResidualNormFunction.apply(u, residual, *mixed, "layer", 1e-5)
        assert torch.equal(a[0], b[0])
        (ga,), (gb,) = (torch.autograd.grad(o[0].float().sum(), [u]) for o in (a, b))
        assert torch.equal(ga, gb)


def test_other_forms_of_call_take_the_python_route():
    from torch.utils._python_dispatch import TorchDispatchMode
    (x, gates, decay), cu, h0 = _recurrence_leaves(F32, F32, True)
    want = npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0)

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Watch():
        assert torch.equal(npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0), want)
        res = npa.residual_norm(x, x, scale=decay)
    assert torch.equal(res[0], npa.residual_norm(x, x, scale=decay)[0])
    # what saved-tensor hooks give back
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        y = npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0)
        stream, normed = npa.residual_norm(x, x, scale=decay, pre_weight=decay)
    g1 = torch.autograd.grad(y.sum(), [x, gates, decay, h0])
    g2 = torch.autograd.grad(want.sum(), [x, gates, decay, h0])
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))
    torch.autograd.grad(stream.sum() + normed.sum(), [x, decay])
    # strided, expanded and transposed gradients
    y = npa.varlen_recurrence(x, gates, cu, decay)
    a = torch.autograd.grad(y, [x], torch.ones(1, device="cuda").expand(700, 96), retain_graph=True)[0]
    b = torch.autograd.grad(y, [x], torch.ones(96, 700, device="cuda").t(), retain_graph=True)[0]
    assert torch.equal(a, b) and torch.equal(a, torch.autograd.grad(y, [x], torch.ones(700, 96, device="cuda"))[0])


def test_second_derivatives_are_refused():
    (x, gates, decay), cu, _ = _recurrence_leaves(F32, F32, False)
    for out in (npa.varlen_recurrence(x, gates, cu, decay), npa.VarlenRecurrenceFunction.apply(x, gates, cu, decay)[0],
                npa.residual_norm(x, x, scale=decay)[0], npa.ResidualNormFunction.apply(x, x, None, None, None, decay, None, None, "layer", 1e-5)[0]):
        with pytest.raises((RuntimeError, NotImplementedError)):
            (dx,) = torch.autograd.grad(out.square().sum(), [x], create_graph=True)
            torch.autograd.grad(dx.sum(), [decay])


def test_checkpointing_and_threads():
    from concurrent.futures import ThreadPoolExecutor
    from torch.utils.checkpoint import checkpoint
    (x, gates, decay), cu, h0 = _recurrence_leaves(BF16, F32, True)

    def f(x, gates):
        y = npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0)
        return npa.residual_norm(y, x, pre_weight=decay)[1]
    want = torch.autograd.grad(f(x, gates).float().sum(), [x, gates, decay])
    got = torch.autograd.grad(checkpoint(f, x, gates, use_reentrant=False).float().sum(), [x, gates, decay])
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    def job(_):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            out = torch.autograd.grad(f(x, gates).float().sum(), [x, gates, decay])
        s.synchronize()
        return out
    with ThreadPoolExecutor(4) as pool:
        for out in pool.map(job, range(8)):
            assert all(torch.equal(a, b) for a, b in zip(want, out))
