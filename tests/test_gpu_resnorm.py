"""The residual norm against the definition in 64 bits (resnorm_ref.py), through the public entry points."""
import pytest
import torch

import nanoplm_amd as npa
from tests import resnorm_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("u", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
ALL = "g p pb s q qb"


def _inputs(T, C, act, st, par, parts, seed=0):
    """On the CPU, by name; what ``parts`` does not list is None. dstream and dnormed come last."""
    g = torch.Generator().manual_seed(seed * 100 + T * 3 + C)
    parts = parts.split()
    n = lambda *s, d=act, std=1.0, m=0.0: (torch.randn(*s, generator=g) * std + m).to(d)
    opt = lambda part, t: t if part in parts else None
    return {"u": n(T, C, m=0.5), "residual": n(T, C, d=st, std=3.0, m=-1.0), "gate": opt("g", n(T, C, std=2.0)), "post_weight": opt("p", n(C, d=par, m=1.0)),
            "post_bias": opt("pb", n(C, d=par)), "scale": opt("s", n(C, d=par)), "pre_weight": opt("q", n(C, d=par, m=1.0)),
            "pre_bias": opt("qb", n(C, d=par))}, n(T, C, d=st), opt("q", n(T, C))


def _check(ins, ds, dy, norm, eps=1e-5, shifted=()):
    leaves = {k: None if t is None else t.cuda() for k, t in ins.items()}
    for k in shifted:                     # an element off the alignment that vectors want
        leaves[k] = torch.empty(leaves[k].numel() + 1, dtype=leaves[k].dtype, device="cuda")[1:].view(leaves[k].shape).copy_(leaves[k])
    leaves = {k: None if t is None else t.requires_grad_() for k, t in leaves.items()}
    stream, normed = npa.residual_norm(*leaves.values(), norm=norm, eps=eps)
    want = R.run(*ins.values(), norm, eps, ds, dy)
    R.assert_within(stream, want["stream"], "stream")
    assert stream.dtype == ins["residual"].dtype and (normed is None) == (ins["pre_weight"] is None)
    if normed is not None:
        assert normed.dtype == ins["u"].dtype
        R.assert_within(normed, want["normed"], "normed")
    there = [k for k, t in leaves.items() if t is not None]
    outs = [stream] + ([] if normed is None else [normed])
    grads = torch.autograd.grad(outs, [leaves[k] for k in there], [ds.cuda()] + ([] if normed is None else [dy.cuda()]))
    for k, grad in zip(there, grads):
        assert grad.dtype == ins[k].dtype
        R.assert_within(grad, want["d" + k], "d" + k)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act,st,par", [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (BF16, F32, BF16)])
@pytest.mark.parametrize("T,C", [(1, 1), (3, 2), (5, 7), (9, 8), (33, 64), (70, 129), (64, 200), (17, 256), (40, 511), (600, 512), (31, 768), (20, 1000),
                                 (13, 1001), (50, 1024), (9, 1032), (11, 2048), (7, 4095), (5, 8192), (3, 16384)])
def test_whole_operator(T, C, act, st, par, norm):
    _check(*_inputs(T, C, act, st, par, ALL), norm)


@pytest.mark.parametrize("T,C", [(50, 4), (9, 212), (33, 1004), (4, 8212)])          # fp32 vectors of 4 that are no vectors of 8
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_channels_in_fours(T, C, norm):
    for act, st in ((F32, F32), (BF16, F32)):
        _check(*_inputs(T, C, act, st, F32, ALL, 3), norm)


@pytest.mark.parametrize("shifted", ["u", "residual", "gate", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias"])
def test_one_tensor_that_no_vector_load_takes(shifted):
    for act, st, par in ((BF16, BF16, BF16), (F32, F32, F32), (BF16, F32, F32)):
        _check(*_inputs(2100, 64, act, st, par, ALL, 4), "layer", shifted=[shifted])


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("parts", ["", "g", "p", "s", "q", "p pb", "q qb", "g p s q", "g s", "p q", "s q qb", "g p pb"])
@pytest.mark.parametrize("C", [72, 333])
def test_parts(C, parts, norm):
    _check(*_inputs(45, C, BF16, F32, F32, parts), norm)
    _check(*_inputs(45, C, F32, F32, F32, parts), norm)


def test_many_rows():
    """More rows than one block each takes once, gradients of parameters from every block."""
    for T, C in ((20011, 64), (5003, 300), (2500, 1024)):
        _check(*_inputs(T, C, BF16, F32, F32, ALL, 1), "layer")


def test_mixed_parameter_dtypes_and_column_slices():
    ins, ds, dy = _inputs(50, 96, BF16, F32, BF16, ALL)
    ins["pre_weight"] = ins["pre_weight"].float()
    _check(ins, ds, dy, "layer")
    for off in (0, 3, 8):
        wide = torch.randn(50, off + 2 * 96 + 8, dtype=F32).to(BF16).cuda()
        wide[:, off:off + 96], wide[:, off + 96:off + 192] = ins["u"].cuda(), ins["gate"].cuda()
        rest = [None if t is None else t.cuda() for t in list(ins.values())[3:]]
        wide_x = torch.empty(50, 100, device="cuda")
        wide_x[:, 1:97] = ins["residual"].cuda()
        a = npa.residual_norm_fwd(ins["u"].cuda(), ins["residual"].cuda(), ins["gate"].cuda(), *rest, want_stats=True)
        b = npa.residual_norm_fwd(wide[:, off:off + 96], wide_x[:, 1:97], wide[:, off + 96:off + 192], *rest, want_stats=True)
        want = R.run(*ins.values(), "layer", 1e-5, ds, dy)
        for got in (a, b):
            R.assert_within(got[0], want["stream"], "stream")
            R.assert_within(got[1], want["normed"], "normed")
        dst = ds.cuda().t().contiguous().t()
        g = npa.residual_norm_bwd(wide[:, off:off + 96], wide_x[:, 1:97], wide[:, off + 96:off + 192], *rest[:4], b[2], dst, dy.cuda(), pre_bias=True)
        for name, t in zip(("du", "dresidual", "dgate", "dpost_weight", "dpost_bias", "dscale", "dpre_weight", "dpre_bias"), g):
            R.assert_within(t, want[name], name)


def test_one_gradient_alone():
    """Only one of the two outputs is used; frozen parameters."""
    ins, ds, dy = _inputs(30, 128, F32, F32, F32, ALL)
    for which in (0, 1):
        leaves = {k: t.cuda().requires_grad_() for k, t in ins.items()}
        out = npa.residual_norm(*leaves.values())[which]
        grads = torch.autograd.grad(out, list(leaves.values()), (ds, dy)[which].cuda(), allow_unused=True)
        want = R.run(*ins.values(), "layer", 1e-5, ds if which == 0 else None, dy if which == 1 else None)
        for k, g in zip(leaves, grads):
            R.assert_within(g, want["d" + k], "d" + k)
    u = ins["u"].cuda().requires_grad_()
    rest = [t.cuda() for t in list(ins.values())[1:]]
    stream, normed = npa.residual_norm(u, *rest)
    (g,) = torch.autograd.grad([stream, normed], [u], [ds.cuda(), dy.cuda()])
    R.assert_within(g, R.run(*ins.values(), "layer", 1e-5, ds, dy)["du"], "du")


def test_gradients_agree_with_differences():
    ins, ds, dy = _inputs(12, 40, F32, F32, F32, ALL)
    leaves = {k: t.cuda().requires_grad_() for k, t in ins.items()}
    grads = torch.autograd.grad(npa.residual_norm(*leaves.values()), list(leaves.values()), [ds.cuda(), dy.cuda()])
    g = torch.Generator().manual_seed(1)
    for k, grad in zip(ins, grads):
        d = torch.randn(ins[k].shape, generator=g).double()

        def value(eps):
            moved = {n: t.double() + eps * d if n == k else t.double() for n, t in ins.items()}
            out = R.run(*moved.values(), "layer", 1e-5)
            return float((out["stream"][0] * ds.double()).sum() + (out["normed"][0] * dy.double()).sum())
        want = (value(1e-5) - value(-1e-5)) / 2e-5
        terms = grad.cpu().double() * d
        assert abs(float(terms.sum()) - want) <= 1e-4 * float(terms.abs().sum()), k


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_rows_keep_to_themselves_and_constant_rows_are_finite(norm):
    ins, ds, dy = _inputs(40, 136, F32, F32, F32, ALL)
    ins["u"][7], ins["residual"][7] = 0.0, 0.0                 # nothing to normalise: eps alone
    ins["u"][8] = 5.0
    _check(ins, ds, dy, norm)
    c = lambda t: t.cuda()
    clean = npa.residual_norm_fwd(*map(c, ins.values()), norm=norm, want_stats=True)
    gc = npa.residual_norm_bwd(*map(c, list(ins.values())[:7]), clean[2], c(ds), c(dy), norm=norm)
    ins["u"][3, 5], ins["gate"][4, 0], ins["residual"][5, 100] = float("nan"), float("inf"), float("-inf")
    dirty = npa.residual_norm_fwd(*map(c, ins.values()), norm=norm, want_stats=True)
    gd = npa.residual_norm_bwd(*map(c, list(ins.values())[:7]), dirty[2], c(ds), c(dy), norm=norm)
    keep = torch.tensor([t for t in range(40) if t not in (3, 4, 5)]).cuda()
    for a, b in list(zip(clean[:2], dirty[:2])) + list(zip(gc[:3], gd[:3])):
        assert torch.equal(a[keep], b[keep])


def test_far_from_zero():
    """Rows whose mean is a thousand times their spread: the variance comes from differences to the mean."""
    ins, ds, dy = _inputs(20, 256, F32, F32, F32, ALL)
    ins["u"] += 1000.0
    ins["residual"] += 3000.0
    _check(ins, ds, dy, "layer")


def test_results_repeat_bit_for_bit_and_empty_batches():
    ins, ds, dy = _inputs(3000, 264, BF16, F32, BF16, ALL)
    c = [t.cuda() for t in ins.values()]
    fwd = npa.residual_norm_fwd(*c, want_stats=True)
    first = npa.residual_norm_bwd(*c[:7], fwd[2], ds.cuda(), dy.cuda(), pre_bias=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, npa.residual_norm_bwd(*c[:7], fwd[2], ds.cuda(), dy.cuda(), pre_bias=True)))
    half = npa.residual_norm_bwd(*c[:7], fwd[2], ds.cuda(), dy.cuda(), pre_bias=True, grads_bf16=True)
    assert all(torch.equal(a.bfloat16(), b) for a, b in zip(first[3:], half[3:]))
    empty = [t[:0] if t.dim() == 2 else t for t in c]
    out = npa.residual_norm_fwd(*empty, want_stats=True)
    assert out[0].shape == (0, 264) and out[1].shape == (0, 264)
    grads = npa.residual_norm_bwd(*empty[:7], out[2], ds.cuda()[:0], dy.cuda()[:0], pre_bias=True)
    assert all(not bool(g.any()) for g in grads[3:])


def test_custom_ops_pass_opcheck_and_compile_without_graph_breaks():
    for parts in (ALL, "p s", "g q"):
        ins, ds, dy = _inputs(40, 64, BF16, F32, F32, parts)
        leaves = [None if t is None else t.cuda().requires_grad_() for t in ins.values()]
        torch.library.opcheck(npa.residual_norm_fwd_op, tuple(leaves) + ("layer", 1e-5),
                              test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))

        def f(*a):
            stream, normed = npa.residual_norm(a[0] * 1.0, *a[1:])
            return (stream * 2.0,) if normed is None else (stream * 2.0, normed)
        there = [t for t in leaves if t is not None]
        douts = [ds.cuda()] + ([] if dy is None else [dy.cuda()])
        eager = f(*leaves)
        g1 = torch.autograd.grad(eager, there, douts)
        got = torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")(*leaves)
        g2 = torch.autograd.grad(got, there, douts)
        assert all(torch.equal(a, b) for a, b in zip(list(eager) + list(g1), list(got) + list(g2)))


def test_side_stream_and_graph_replay():
    ins, ds, dy = _inputs(700, 192, BF16, F32, F32, ALL)
    leaves = [t.cuda().requires_grad_() for t in ins.values()]
    ds, dy = ds.cuda(), dy.cuda()

    def step():
        outs = npa.residual_norm(*leaves)
        grads = torch.autograd.grad(outs, leaves, [ds, dy])
        return [o.detach() for o in outs] + list(grads)        # (no eager graph of the leaves may live while the step is captured)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        with torch.no_grad():
            leaves[0].mul_(0.5 + k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, got)), k


def test_offsets_beyond_four_gib():
    T, C = 600000, 4096                              # 4.9 GB in bf16
    u = torch.zeros(T, C, dtype=BF16, device="cuda")
    x = torch.zeros(T, C, dtype=BF16, device="cuda")
    ds = torch.zeros(T, C, dtype=BF16, device="cuda")
    ins, d, dy = _inputs(10, C, BF16, BF16, F32, "p q")
    u[-10:], x[-10:], ds[-10:] = ins["u"].cuda(), ins["residual"].cuda(), d.cuda()
    pw, qw = ins["post_weight"].cuda(), ins["pre_weight"].cuda()
    stream, normed, stats = npa.residual_norm_fwd(u, x, None, pw, None, None, qw, want_stats=True)
    want = R.run(*ins.values(), "layer", 1e-5, d, None)
    R.assert_within(stream[-10:], want["stream"], "stream")
    R.assert_within(normed[-10:], want["normed"], "normed")
    assert not bool(stream[:-10].any())
    del stream, normed
    du, dx, *_ = npa.residual_norm_bwd(u, x, None, pw, None, None, qw, stats, ds, None)
    R.assert_within(du[-10:], want["du"], "du")
    R.assert_within(dx[-10:], want["dresidual"], "dresidual")


def test_module():
    m = npa.ResidualNorm(96, norm="rms", bias=True, scale_init=0.5).cuda()
    ins, ds, dy = _inputs(20, 96, BF16, F32, F32, "g")
    stream, normed = m(ins["u"].cuda(), ins["residual"].cuda(), ins["gate"].cuda())
    p = {k: (None if getattr(m, k) is None else getattr(m, k).detach().cpu()) for k in NAMES[3:]}
    want = R.run(ins["u"], ins["residual"], ins["gate"], *p.values(), "rms", m.eps)
    R.assert_within(stream, want["stream"], "stream")
    R.assert_within(normed, want["normed"], "normed")
    (stream.sum() + normed.float().square().sum()).backward()
    assert all(q.grad is not None for q in m.parameters())
    last = npa.ResidualNorm(96, post=False, pre=False)
    assert len(list(last.parameters())) == 0
