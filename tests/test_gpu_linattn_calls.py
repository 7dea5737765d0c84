"""Forms of call of linear attention, its step and the layer norm: refusals, forward mode, recorded calls, negated views, tables that share memory, second derivatives,
strides beyond a buffer's, graphs beside each other; and the operators one behind the other, as a block has them."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nanoplm_amd as npa

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
T, H, K, V = 300, 2, 24, 20


def _inputs(act=F32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s, d=act: torch.randn(*s, device="cuda", generator=g).to(d)
    return dict(q=n(T, H, K), k=n(T, H, K), v=n(T, H, V), g=-n(T, H, d=F32).abs(), cu=torch.tensor([0, 100, 100, T], dtype=torch.int32, device="cuda"),
                h0=n(3, H, K, V, d=F32), table=n(T + 5, H, K, V, d=F32), x=n(T, 70), gate=n(T, 70), weight=n(35, d=F32), bias=n(35, d=F32))


def _calls(i, table=None):
    table = i["table"].clone() if table is None else table
    return {"attention": lambda: npa.varlen_linear_attention(i["q"], i["k"], i["v"], i["cu"], i["g"], initial_state=i["h0"], return_state=True),
            "norm": lambda: (npa.layer_norm(i["x"], i["weight"], i["bias"], gate=i["gate"], heads=2),),
            "step": lambda: (npa.linear_attention_step(i["q"], i["k"], i["v"], i["g"], table),)}


USED = {"attention": ("q", "k", "v", "g", "h0"), "norm": ("x", "gate", "weight", "bias"), "step": ("q", "k", "v", "g")}


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_attention_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    cu = torch.tensor([0, 5], dtype=torch.int32).cuda()
    good = dict(q=z(5, 2, 4), k=z(5, 2, 4), v=z(5, 2, 3), cu_seqlens=cu, log_decay=z(2))
    npa.varlen_linear_attention(**good)
    for bad, err in [(dict(k=z(5, 2, 3)), ValueError), (dict(v=z(4, 2, 3)), ValueError), (dict(v=z(5, 1, 3)), ValueError), (dict(v=z(5, 2, 3, d=BF16)), TypeError),
                     (dict(log_decay=z(3)), ValueError), (dict(log_decay=z(5, 1)), ValueError), (dict(log_decay=z(2, d=BF16)), TypeError),
                     (dict(cu_seqlens=cu.long()), TypeError), (dict(cu_seqlens=cu[:0]), TypeError), (dict(cu_seqlens=cu.cpu()), RuntimeError),
                     (dict(k=z(5, 2, 4).cpu()), RuntimeError), (dict(log_decay=z(2).cpu()), RuntimeError), (dict(v=z(5, 2, 0)), ValueError), (dict(v=z(5, 2, 129)), ValueError),
                     (dict(q=z(5, 2, 129), k=z(5, 2, 129)), ValueError), (dict(q=z(5, 0, 4), k=z(5, 0, 4), v=z(5, 0, 3), log_decay=z(0)), ValueError),
                     (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError), (dict(initial_state=z(2, 2, 4, 3)), ValueError),
                     (dict(initial_state=z(1, 2, 4, 3, d=BF16)), ValueError), (dict(initial_state=z(1, 2, 4, 3).cpu()), RuntimeError)]:
        with pytest.raises(err):
            npa.varlen_linear_attention(**{**good, **bad})
    args = [z(300, 2, 4), z(300, 2, 4), z(300, 2, 3), z(300, 2, 3), cu * 60, z(2)]
    _, state, bounds = npa.varlen_linear_attention_fwd(*args[:3], *args[4:], want_state=True)
    assert bounds.numel() > 0
    npa.varlen_linear_attention_bwd(*args, bounds, state=state, dstate=state)
    for a, b, k in ((args, bounds[:-1], {}), (args, bounds.cpu(), {}), (args, None, {}), (args, bounds, dict(dstate=state)), (args, bounds, dict(state=z(2, 2, 4, 3))),
                    (args[:3] + [z(300, 2, 3, d=BF16)] + args[4:], bounds, {})):
        with pytest.raises(ValueError):
            npa.varlen_linear_attention_bwd(*a, b, **k)


def test_bounds_of_the_op_serve_the_raw_backward_and_others_do_not():
    r = torch.Generator().manual_seed(2)
    q, v, g = torch.randn(300, 2, 16, generator=r).cuda(), torch.randn(300, 2, 12, generator=r).cuda(), -torch.rand(300, 2, generator=r).cuda()
    cu = torch.tensor([0, 300], dtype=torch.int32).cuda()
    o, _, bounds = npa.varlen_linear_attention_fwd(q, q, v, cu, g)
    same, _, more = npa.varlen_linear_attention_fwd_op(q, q, v, cu, g, None, None, False, False)
    assert torch.equal(o, same) and 0 < bounds.numel() < more.numel()
    want, got = (npa.varlen_linear_attention_bwd(q, q, v, v, cu, g, b)[:4] for b in (bounds, more))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for other in (more[:-1], torch.cat((bounds, bounds[:256])), torch.cat((more, more[:1]))):
        with pytest.raises(ValueError, match="bounds"):
            npa.varlen_linear_attention_bwd(q, q, v, v, cu, g, other)


def test_step_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(q=z(5, 2, 4), k=z(5, 2, 4), v=z(5, 2, 3), log_decay=z(5, 2), state=z(6, 2, 4, 3), slots=z(5, d=torch.int32))
    npa.linear_attention_step(**good)
    for bad, err in [(dict(state=z(6, 2, 4, 4)), ValueError), (dict(state=z(6, 2, 4, 3, d=BF16)), ValueError), (dict(state=z(6, 2, 3, 4).transpose(2, 3)), ValueError),
                     (dict(out_state=z(5, 2, 4, 3)), ValueError), (dict(slots=z(5, d=torch.int64)), TypeError), (dict(slots=z(4, d=torch.int32)), TypeError),
                     (dict(slots=None, state=z(4, 2, 4, 3)), ValueError), (dict(slots=z(5, d=torch.int32).cpu()), RuntimeError),
                     (dict(state=z(6, 2, 4, 3).cpu()), RuntimeError), (dict(q=z(5, 2, 4).requires_grad_()), RuntimeError), (dict(log_decay=z(6, 2)), ValueError),
                     (dict(scale=float("inf")), ValueError)]:
        with pytest.raises(err):
            npa.linear_attention_step(**{**good, **bad})
    many = (1 << 16) + 1
    with pytest.raises(ValueError, match="at most 65536 rows"):
        npa.linear_attention_step(z(many, 1, 1), z(many, 1, 1), z(many, 1, 1), z(1), z(3, 1, 1, 1), z(many, d=torch.int32))
    npa.linear_attention_step(z(many, 1, 1), z(many, 1, 1), z(many, 1, 1), z(1), z(many, 1, 1, 1))
    with torch.no_grad():
        npa.linear_attention_step(**{**good, "q": z(5, 2, 4).requires_grad_()})
    assert npa.linear_attention_step(z(0, 2, 4), z(0, 2, 4), z(0, 2, 3), z(2), z(6, 2, 4, 3)).shape == (0, 2, 3)


def test_norm_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(x=z(5, 8), weight=z(8), bias=z(8), gate=z(5, 8))
    npa.layer_norm(**good)
    for bad, err in [(dict(weight=z(7)), ValueError), (dict(bias=z(4), heads=2), ValueError), (dict(weight=None), ValueError), (dict(gate=z(5, 7)), ValueError),
                     (dict(gate=z(5, 8, d=BF16)), ValueError), (dict(heads=3), ValueError), (dict(heads=0), ValueError), (dict(norm="batch"), ValueError),
                     (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError), (dict(weight=z(8).cpu()), RuntimeError), (dict(weight=z(8, d=torch.float16)), TypeError),
                     (dict(x=z(5, 0), gate=None, weight=None, bias=None), ValueError)]:
        with pytest.raises(err):
            npa.layer_norm(**{**good, **bad})
    for x, heads in ((z(1, 16385), 1), (z(1, 65536), 65536)):
        with pytest.raises(ValueError, match="groups"):
            npa.layer_norm(x, heads=heads)
    assert bool(npa.layer_norm(torch.randn(2, 65535, device="cuda"), heads=65535).eq(0).all())       # (groups of one)


# ---- ways of calling --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["attention", "norm", "step"])
def test_forward_mode_is_refused(name, grad):
    i = _inputs()
    for which in sorted(set(sum(USED.values(), ()))):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            call = _calls({**i, which: forward_ad.make_dual(i[which], torch.ones_like(i[which]))})[name]
            if which in USED[name]:
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
    slots = torch.arange(T, dtype=torch.int32, device="cuda").flip(0)
    rows = i["q"], i["k"], i["v"]
    return {"attention": (lambda q, k, v, g: npa.varlen_linear_attention(q, k, v, i["cu"], g), (*rows, i["g"])),
            "states": (lambda q, k, v, g, h: npa.varlen_linear_attention(q, k, v, i["cu"], g, scale=0.5, initial_state=h, reverse=True, return_state=True),
                       (*rows, i["g"], i["h0"])),
            "norm": (lambda x, w, b, g: npa.layer_norm(x, w, b, gate=g, heads=2, norm="rms"), (i["x"], i["weight"], i["bias"], i["gate"])),
            "plain norm": (lambda x: npa.layer_norm(x), (i["x"],)),
            "step": (lambda q, k, v, g, t: npa.linear_attention_step(q, k, v, g, t, slots), (*rows, i["g"], i["table"])),
            "step_to": (lambda q, k, v, g, t, o: npa.linear_attention_step(q, k, v, g, t, out_state=o), (*rows, i["g"], i["table"], i["table"] * 2))}


def _listed(out):
    return list(out) if isinstance(out, tuple) else [out]


@pytest.mark.parametrize("record", ["jit.trace", "make_fx"])
@pytest.mark.parametrize("name", ["attention", "states", "norm", "plain norm", "step", "step_to"])
def test_a_recorded_call_follows_the_inputs_of_the_replay(name, record):
    """Recorded with one set of inputs and replayed with others, outputs and changed tables are the eager call's."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, example = _recordable(_inputs())[name]
    example = tuple(t.clone() for t in example)
    recorded = torch.jit.trace(f, example, check_trace=False) if record == "jit.trace" else make_fx(f)(*example)
    for seed in (1, 2):
        args = _recordable(_inputs(seed=seed))[name][1]
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
    for which in sorted(set(sum(USED.values(), ()))):
        neg = {**i, which: torch._neg_view(-i[which])}
        for name, call in _calls(neg).items():
            assert all(torch.equal(a, b) for a, b in zip(call(), _calls(i)[name]())), (which, name)
    do, dy = torch.randn(T, H, V, device="cuda").bfloat16(), torch.randn(T, 70, device="cuda").bfloat16()
    leaves = [i[n].clone().requires_grad_() for n in USED["attention"]]
    grads = [torch.autograd.grad(npa.varlen_linear_attention(*leaves[:3], i["cu"], leaves[3], initial_state=leaves[4]), leaves, d) for d in (do, torch._neg_view(-do))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    leaves = [i[n].clone().requires_grad_() for n in USED["norm"]]
    grads = [torch.autograd.grad(npa.layer_norm(leaves[0], *leaves[2:], gate=leaves[1], heads=2), leaves, d) for d in (dy, torch._neg_view(-dy))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_tables_of_a_step_are_one_or_apart():
    i, both = _inputs(), torch.randn(700, H, K, V, device="cuda")
    old = both.clone()
    args = i["q"], i["k"], i["v"], i["g"]
    for state, out in ((both[:310], both[1:311]), (both[300:], both[:400])):
        with pytest.raises(ValueError, match="shares some of its memory"):
            npa.linear_attention_step(*args, state, out_state=out)
    assert torch.equal(both, old)
    o = npa.linear_attention_step(*args, both[:350], out_state=both[350:])
    assert torch.equal(both[:350], old[:350]) and torch.equal(both[650:], old[650:])
    assert torch.equal(o, npa.linear_attention_step(*args, both[:350], out_state=both.view(-1)[:350 * H * K * V].view(350, H, K, V)))
    assert torch.equal(both[:300], both[350:650])


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", ["attention", "norm"])
def test_the_first_derivative_under_create_graph_and_no_second(name, native):
    i = _inputs()
    a, b = (i["q"], i["g"]) if name == "attention" else (i["x"], i["weight"])
    a.requires_grad_(), b.requires_grad_()
    call = {("attention", True): lambda: npa.varlen_linear_attention(a, i["k"], i["v"], i["cu"], b),
            ("attention", False): lambda: npa.VarlenLinearAttentionFunction.apply(a, i["k"], i["v"], i["cu"], b)[0],
            ("norm", True): lambda: npa.layer_norm(a, b, heads=2),
            ("norm", False): lambda: npa.LayerNormFunction.apply(a, b, None, None, 2, "layer", 1e-5)}[name, native]
    want = torch.autograd.grad(call().square().sum(), [a, b])
    got = torch.autograd.grad(call().square().sum(), [a, b], create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and got[0].requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula" if native else "once_differentiable"):
        got[0].sum().backward()


def test_a_module_steps_under_no_grad():
    i, m = _inputs(), npa.VarlenLinearAttention(H).cuda()
    table = i["table"].clone()
    with pytest.raises(RuntimeError, match="call it under torch.no_grad"):
        m.step(i["q"], i["k"], i["v"], table)
    assert torch.equal(table, i["table"])
    with torch.no_grad():
        m.step(i["q"], i["k"], i["v"], table)
    assert not torch.equal(table[:T], i["table"][:T]) and torch.equal(table[T:], i["table"][T:])


def test_a_step_is_a_change_that_autograd_sees():
    i = _inputs()
    cu = torch.arange(T + 1, dtype=torch.int32, device="cuda")
    args = i["q"], i["k"], i["v"], i["g"]
    for route in (lambda t: npa.linear_attention_step(*args, t), lambda t: npa.linear_attention_step(torch._neg_view(-i["q"]), *args[1:], t)):
        table = i["table"][:T].clone()
        leaf = i["q"].clone().requires_grad_()
        o = npa.varlen_linear_attention(leaf, *args[1:3], cu, args[3], initial_state=table)
        before = table._version
        route(table)
        assert table._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.sum().backward()
    with torch.inference_mode():
        t = i["table"].clone()
        npa.linear_attention_step(*args, t)
    npa.linear_attention_step(*args, t)


@pytest.mark.parametrize("apart", [False, True])
def test_a_step_in_a_compiled_model(apart):
    i = _inputs()
    slots = torch.arange(T, dtype=torch.int32, device="cuda") - 1

    def f(q, table, other):
        o = npa.linear_attention_step(q * 2, i["k"], i["v"], i["g"], table, slots, out_state=other if apart else None)
        o = o + npa.linear_attention_step(q, i["k"], i["v"], i["g"], table, slots, out_state=other if apart else table)
        return o, table.sum(), other.sum()
    a, b = i["table"].clone(), i["table"] * 2
    a2, b2 = a.clone(), b.clone()
    with torch.no_grad():
        want = f(i["q"], a, b)
        got = torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")(i["q"], a2, b2)
        assert all(torch.equal(p, q) for p, q in zip(want, got)) and torch.equal(a, a2) and torch.equal(b, b2)
        torch.library.opcheck(npa.linear_attention_step_op, (i["q"], i["k"], i["v"], i["g"], a, slots, 0.5))
        torch.library.opcheck(npa.linear_attention_step_to_op, (i["q"], i["k"], i["v"], i["g"], a, None if apart else slots, 0.5, b))


def test_one_compiled_model_for_packed_batches_of_all_sizes():
    """Rows and sequences both change from batch to batch: nothing is compiled after the first one, and the results are those of the calls by themselves."""
    from torch._dynamo.testing import CompileCounterWithBackend
    counter = CompileCounterWithBackend("aot_eager")

    def f(q, k, v, cu, g, w):
        return npa.layer_norm(npa.varlen_linear_attention(q * 1.0, k, v, cu, g).flatten(1), w, heads=2)
    compiled = torch.compile(f, dynamic=True, fullgraph=True, backend=counter)
    graphs = []
    for seed, lens in enumerate(([300, 20], [64, 1, 700, 9, 30], [2500, 0, 10], [40] * 31)):
        r = torch.Generator().manual_seed(seed)
        T = sum(lens)
        make = lambda *s: torch.randn(*s, generator=r).cuda()
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        leaves = [t.requires_grad_() for t in (make(T, 2, 16), make(T, 2, 16), make(T, 2, 12), -make(T, 2).abs(), make(24))]
        dy = make(T, 24)
        want, got = (call(*leaves[:3], cu, *leaves[3:]) for call in (f, compiled))
        assert torch.equal(want, got)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(want, leaves, dy), torch.autograd.grad(got, leaves, dy)))
        graphs.append(counter.frame_count)
    assert len(set(graphs)) == 1, graphs


def test_one_tensor_as_queries_keys_and_values():
    i = _inputs()
    x = i["q"].clone().requires_grad_()
    (got,) = torch.autograd.grad(npa.varlen_linear_attention(x, x, x, i["cu"], i["g"]).square().sum(), [x])
    three = [i["q"].clone().requires_grad_() for _ in range(3)]
    apart = torch.autograd.grad(npa.varlen_linear_attention(*three, i["cu"], i["g"]).square().sum(), three)
    assert torch.allclose(got, sum(apart), rtol=0, atol=4 * 2.0 ** -24 * float(sum(t.abs() for t in apart).max()))      # (two additions, in whatever order)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("reverse", [False, True])
def test_rows_too_far_apart_for_one_buffer(act, reverse):
    """Rows of 2^24 bytes: a segment of them is more than a buffer's offsets hold, and the results are those of rows that lie side by side."""
    n, K, V = 70, 64, 64
    wide = torch.empty(n, (1 << 24) // (2 if act == BF16 else 4), dtype=act, device="cuda")
    g = torch.Generator("cuda").manual_seed(0)
    far = [wide[:, j * H * 64:(j + 1) * H * 64].view(n, H, 64).normal_(generator=g) for j in range(4)]
    near = [t.contiguous() for t in far]
    cu = torch.tensor([0, 30, n], dtype=torch.int32, device="cuda")
    log_decay = -torch.rand(n, H, device="cuda", generator=g)
    results = []
    for q, k, v, do in (far, near):
        o, state, bounds = npa.varlen_linear_attention_fwd(q, k, v, cu, log_decay, reverse=reverse, want_state=True)
        results.append([o, state, *npa.varlen_linear_attention_bwd(q, k, v, do, cu, log_decay, bounds, reverse=reverse)[:4]])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("B,H,K,V,N", [(6001, 2, 8, 12, 1500), (6001, 1, 5, 7, 6000), (600, 8, 128, 128, 200)])
def test_rows_that_name_one_slot_are_its_tokens_in_order(B, H, K, V, N):
    """The same as steps of one row of each slot, one step after the other, bit for bit; the last size's states are more than the caches hold."""
    g = torch.Generator("cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v, log_decay, table = n(B, H, K), n(B, H, K), n(B, H, V), -n(B, H).abs(), n(N, H, K, V)
    slots = torch.randint(0, N, (B,), device="cuda", generator=g).int()
    slots[7::97] = -1
    seen, turns = {}, []
    for s in slots.tolist():                           # (row b is its slot's turn-th)
        turns.append(seen.get(s, 0) if s >= 0 else -1)
        seen[s] = seen.get(s, 0) + 1
    turns = torch.tensor(turns, device="cuda")
    want_table, want = table.clone(), torch.zeros(B, H, V, device="cuda")
    for turn in range(int(turns.max()) + 1):
        now = turns == turn
        o = npa.linear_attention_step(q, k, v, log_decay, want_table, torch.where(now, slots, -1))
        want[now] = o[now]
        assert not bool(o[~now].any())
    for out in (None, table.clone()):
        state = table.clone()
        o = npa.linear_attention_step(q, k, v, log_decay, state, slots, out_state=out)
        assert torch.equal(o, want) and torch.equal(state if out is None else out, want_table)
        assert out is None or torch.equal(state, table)


def test_two_graphs_replayed_beside_each_other():
    """Each of two captured training steps has workspaces of its own: replayed on two streams at once they give what they give alone."""
    def make(seed, reverse):
        i = {n: t.clone() for n, t in _inputs(BF16, seed).items()}
        g = torch.Generator("cuda").manual_seed(seed)
        do = torch.randn(T, H, V, device="cuda", generator=g).bfloat16()
        cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
        leaves = [i[n].requires_grad_() for n in ("q", "k", "v", "g", "x", "weight")]

        def step():
            o = npa.varlen_linear_attention(*leaves[:3], cu, leaves[3], reverse=reverse)
            y = npa.layer_norm(leaves[4], leaves[5], heads=2)
            return list(torch.autograd.grad([o, y], leaves, [do, leaves[4].detach()]))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        return graph, outs, want, step                # (step has the inputs, which the graph reads)
    made = [make(1, False), make(2, True)]
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for (graph, *_), stream in zip(made, streams):
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for _, outs, want, _ in made:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()


# ---- together ---------------------------------------------------------------------------------------------------------------------------
def _silu(x):
    return x * torch.sigmoid(x)


def _norm(x, w, eps, rms=False):
    m = 0 if rms else x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps) * w


def _block_plain(p, x, lens, H, d):
    """In 64 bits, by differentiable elementary operations."""
    y = _norm(x, p["norm"], 1e-5)
    z = y @ p["in"]
    q, k, v, gate, rate = z[:, :H * d], z[:, H * d:2 * H * d], z[:, 2 * H * d:3 * H * d], z[:, 3 * H * d:4 * H * d], z[:, 4 * H * d:]
    k_taps, rows, lo = p["conv"], [], 0
    for n in lens:                                     # the conv of the values, each sequence by itself
        u = torch.nn.functional.pad(v[lo:lo + n], (0, 0, 1, 1))
        rows.append(sum(u[j:j + n] * k_taps[:, j] for j in range(3)))
        lo += n
    v = torch.cat(rows)
    g = torch.nn.functional.logsigmoid(p["decay"] + rate)
    out, lo = [], 0
    for n in lens:
        s = torch.zeros(H, d, d, dtype=x.dtype)
        for t in range(lo, lo + n):
            s = torch.exp(g[t])[:, None, None] * s + k[t].view(H, d, 1) * v[t].view(H, 1, d)
            out.append(d ** -0.5 * (q[t].view(H, 1, d) @ s).view(H * d))
        lo += n
    o = torch.stack(out)
    o = _norm(o.view(-1, H, d), p["head"], 1e-5, rms=True).view(-1, H * d) * _silu(gate)
    stream = x + o @ p["out"]
    return stream, _norm(stream, p["next"], 1e-5)


def test_a_block_of_the_operators_together():
    """Norm, projection, conv, linear attention, gated norm of the heads, residual norm: outputs and every gradient against 64 bits. fp32,
    off by at most 6 operators x sums of 64 x 2^-24 x 4 for the norms' divisions: 1e-4 of a tensor's 2-norm."""
    H, d, C, lens = 3, 16, 40, [50, 1, 70, 29]
    T = sum(lens)
    g = torch.Generator().manual_seed(0)
    n = lambda *s, std=1.0, m=0.0: torch.randn(*s, generator=g) * std + m
    params = {"norm": n(C, std=0.1, m=1.0), "in": n(C, 4 * H * d + H, std=C ** -0.5), "conv": n(H * d, 3, std=0.5), "decay": n(H, m=3.0), "head": n(d, std=0.1, m=1.0),
              "out": n(H * d, C, std=(H * d) ** -0.5), "next": n(C, std=0.1, m=1.0)}
    x, ds, dn = n(T, C), n(T, C), n(T, C)
    plain = {k: t.double().requires_grad_() for k, t in params.items()}
    x64 = x.double().requires_grad_()
    outs = _block_plain(plain, x64, lens, H, d)
    want = list(outs) + list(torch.autograd.grad(outs, [x64, *plain.values()], [ds.double(), dn.double()]))

    p = {k: t.cuda().requires_grad_() for k, t in params.items()}
    xc = x.cuda().requires_grad_()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    norm = npa.LayerNorm(d * H, heads=H, norm="rms", shared=True).cuda()
    attention = npa.VarlenLinearAttention(H).cuda()
    with torch.no_grad():
        norm.weight.copy_(p["head"]), attention.decay.copy_(p["decay"])
    z = npa.layer_norm(xc, p["norm"]) @ p["in"]
    q, k, v, gate, rate = z.split([H * d, H * d, H * d, H * d, H], 1)
    v = npa.varlen_dwconv(v.contiguous(), cu, p["conv"])
    heads = lambda t: t.unflatten(1, (H, d))
    o = attention(heads(q), heads(k), heads(v), cu, rate)
    o = norm(o.flatten(1), gate)
    outs = npa.residual_norm(o @ p["out"], xc, pre_weight=p["next"])
    leaves = [xc, p["norm"], p["in"], p["conv"], attention.decay, norm.weight, p["out"], p["next"]]
    got = list(outs) + list(torch.autograd.grad(outs, leaves, [ds.cuda(), dn.cuda()]))
    for name, a, b in zip(["stream", "normed", "x", *params], got, want):
        off = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 1e-4, (name, off)


def test_the_usage_example_runs_as_it_stands():
    import os
    import re
    readme = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read()
    source = next(s for s in re.findall(r"```python\n(.*?)```", readme, re.S) if "VarlenLinearAttention" in s)
    rows = 500
    b = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    names = dict(qkvg=b(rows, 4096), rates=torch.randn(rows, 16, device="cuda"), cu_seqlens=torch.tensor([0, 200, rows], dtype=torch.int32, device="cuda"), q_t=b(2, 16, 64),
                 k_t=b(2, 16, 64), v_t=b(2, 16, 64), rates_t=torch.randn(2, 16, device="cuda"), states=torch.zeros(9, 16, 64, 64, device="cuda"),
                 slots=torch.tensor([3, 1], dtype=torch.int32, device="cuda"))
    exec(source, names)
    assert names["y"].shape == (rows, 1024) and names["state"].shape == (2, 16, 64, 64) and names["o_t"].shape == (2, 16, 64) and bool(names["states"][3].any())
