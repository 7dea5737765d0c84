"""The layer norm over rows and heads against the definition in 64 bits, through the public entry points. The bounds are resnorm_ref.py's: the residual norm of u with
a gate and nothing to add to is this norm, head by head."""
import pytest
import torch

import nanoplm_amd as npa
from tests import resnorm_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _inputs(T, C, heads, act, par, gated=True, biased=True, shared=False, seed=0):
    g = torch.Generator().manual_seed(seed * 100 + T * 3 + C)
    n = lambda *s, d=act, std=1.0, m=0.0: (torch.randn(*s, generator=g) * std + m).to(d)
    P = C // heads if shared else C
    return {"x": n(T, C, m=0.5), "weight": n(P, d=par, m=1.0), "bias": n(P, d=par) if biased else None, "gate": n(T, C, std=2.0) if gated else None}, n(T, C)


def _want(ins, dy, heads, norm, eps):
    """{name: (value, bound)}: each head as rows of its own."""
    T, C = ins["x"].shape
    n = C // heads
    out = {}
    part = lambda t, h: None if t is None else t[..., h * n:(h + 1) * n] if t.shape[-1] == C else t
    got = [R.run(part(ins["x"], h), torch.zeros(T, n), part(ins["gate"], h), part(ins["weight"], h), part(ins["bias"], h), None, None, None, norm, eps,
                 part(dy, h)) for h in range(heads)]
    for name, theirs in (("y", "stream"), ("x", "du"), ("gate", "dgate"), ("weight", "dpost_weight"), ("bias", "dpost_bias")):
        if theirs not in got[0]:
            continue
        if name in ("weight", "bias") and ins["weight"].shape[0] != C:        # one for all heads: a lane, a block's groups, fp64
            out[name] = tuple(sum(g[theirs][i] for g in got) for i in range(2))
        else:
            out[name] = tuple(torch.cat([g[theirs][i] for g in got], -1) for i in range(2))
    return out


def _check(ins, dy, heads, norm, eps=1e-5, shifted=()):
    leaves = {k: None if t is None else t.cuda() for k, t in ins.items()}
    for k in shifted:                     # an element off the alignment that vectors want
        leaves[k] = torch.empty(leaves[k].numel() + 1, dtype=leaves[k].dtype, device="cuda")[1:].view(leaves[k].shape).copy_(leaves[k])
    leaves = {k: None if t is None else t.requires_grad_() for k, t in leaves.items()}
    y = npa.layer_norm(leaves["x"], leaves["weight"], leaves["bias"], gate=leaves["gate"], heads=heads, norm=norm, eps=eps)
    want = _want(ins, dy, heads, norm, eps)
    assert y.dtype == ins["x"].dtype
    R.assert_within(y, want["y"], "y")
    there = [k for k, t in leaves.items() if t is not None]
    for k, grad in zip(there, torch.autograd.grad(y, [leaves[k] for k in there], dy.cuda())):
        assert grad.dtype == ins[k].dtype and grad.shape == ins[k].shape
        R.assert_within(grad, want[k], "d" + k)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act,par", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("T,C", [(1, 1), (3, 2), (5, 7), (9, 8), (33, 64), (70, 129), (64, 200), (17, 256), (40, 511), (600, 512), (31, 520), (31, 768), (20, 1000),
                                 (13, 1001), (50, 1024), (9, 1032), (11, 2048), (7, 4095), (5, 8192), (3, 16384)])
def test_whole_rows(T, C, act, par, norm):
    _check(*_inputs(T, C, 1, act, par), 1, norm)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act,par", [(F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("T,C,heads", [(1, 16, 2), (9, 192, 3), (70, 1024, 16), (33, 768, 12), (5, 1001, 11), (20, 320, 5), (6, 2560, 40), (3, 24, 24), (150, 64, 32),
                                       (4, 2100, 2), (11, 8200, 4), (300, 96, 8), (2, 4096, 64), (3, 640, 80), (40, 96, 3), (70, 1024, 64), (7, 217, 7), (500, 1024, 32)])
def test_heads(T, C, heads, act, par, norm, shared):
    _check(*_inputs(T, C, heads, act, par, shared=shared), heads, norm)


@pytest.mark.parametrize("gated,biased", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_parts(norm, gated, biased):
    for heads in (1, 3):
        for act in (F32, BF16):
            _check(*_inputs(45, 72, heads, act, F32, gated, biased), heads, norm)
            _check(*_inputs(45, 333, heads, act, F32, gated, biased), heads, norm)


@pytest.mark.parametrize("shifted", ["x", "gate", "weight", "bias"])
def test_one_tensor_that_no_vector_load_takes(shifted):
    for act in (BF16, F32):
        _check(*_inputs(900, 128, 2, act, act, seed=4), 2, "layer", shifted=[shifted])


def test_many_rows():
    """More rows than one block each takes once, gradients of parameters from every block."""
    for T, C, heads, shared in ((20011, 64, 4, True), (20011, 64, 4, False), (5003, 300, 1, False), (2500, 1024, 16, True), (3001, 2048, 1, False)):
        _check(*_inputs(T, C, heads, BF16, F32, shared=shared, seed=1), heads, "layer")


def test_without_parameters():
    ins, dy = _inputs(40, 96, 3, F32, F32, False, False)
    ones = torch.ones(96)
    x = ins["x"].cuda().requires_grad_()
    y = npa.layer_norm(x, heads=3)
    (dx,) = torch.autograd.grad(y, x, dy.cuda())
    want = _want({**ins, "weight": ones}, dy, 3, "layer", 1e-5)
    R.assert_within(y, want["y"], "y")
    R.assert_within(dx, want["x"], "dx")


def test_column_slices_mixed_parameters_and_other_strides():
    ins, dy = _inputs(50, 96, 2, BF16, BF16)
    ins["weight"] = ins["weight"].float()
    _check(ins, dy, 2, "layer")
    for off in (0, 3, 8):
        wide = torch.randn(50, off + 2 * 96 + 8).to(BF16).cuda()
        x, gate = wide[:, off:off + 96].copy_(ins["x"].cuda()), wide[:, off + 96:off + 192].copy_(ins["gate"].cuda())
        want = _want(ins, dy, 2, "rms", 1e-5)
        w, b = ins["weight"].cuda(), ins["bias"].cuda()
        R.assert_within(npa.layer_norm_fwd(x, w, b, gate, heads=2, norm="rms"), want["y"], "y")
        got = npa.layer_norm_bwd(x, w, b, gate, dy.cuda().t().contiguous().t(), heads=2, norm="rms")
        for name, t in zip(("x", "gate", "weight", "bias"), got):
            R.assert_within(t, want[name], name)


def test_rows_with_nan_stay_alone_and_constant_rows():
    ins, dy = _inputs(40, 64, 2, F32, F32, seed=2)
    ins["x"][7, 3], ins["gate"][9, 40], ins["x"][11] = float("nan"), float("inf"), 1.5
    args = lambda: [None if t is None else t.cuda() for t in ins.values()]
    y = npa.layer_norm(*args()[:3], gate=args()[3], heads=2)
    got = npa.layer_norm_bwd(*args(), dy.cuda(), heads=2)
    clean, _ = _inputs(40, 64, 2, F32, F32, seed=2)
    clean["x"][11] = 1.5
    want = _want(clean, dy, 2, "layer", 1e-5)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[7, 9]] = False
    for t, name in ((y, "y"), (got[0], "x"), (got[1], "gate")):
        R.assert_within(t[keep.cuda()], tuple(v[keep] for v in want[name]), name)
    assert bool(torch.isnan(y[7, :32]).all()) and bool(torch.isfinite(y[7, 32:]).all()) and bool(torch.isnan(got[2][:32]).all())


def test_empty_batches_and_frozen_parameters():
    w = torch.ones(8, device="cuda", requires_grad=True)
    b = torch.zeros(8, device="cuda", requires_grad=True)
    y = npa.layer_norm(torch.zeros(0, 8, device="cuda"), w, b)
    assert y.shape == (0, 8)
    y.sum().backward()
    assert not bool(w.grad.any()) and not bool(b.grad.any())
    ins, dy = _inputs(30, 128, 1, F32, F32)
    x = ins["x"].cuda().requires_grad_()
    (dx,) = torch.autograd.grad(npa.layer_norm(x, ins["weight"].cuda(), ins["bias"].cuda(), gate=ins["gate"].cuda()), x, dy.cuda())
    R.assert_within(dx, _want(ins, dy, 1, "layer", 1e-5)["x"], "dx")


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T,C,heads,shared", [(1, 1, 1, False), (5, 67, 1, False), (64, 1024, 16, True), (700, 96, 12, False), (33, 2560, 40, True)])
def test_nothing_around_the_outputs_is_written(T, C, heads, shared, act):
    lib = npa._lib.load()
    ins, dy = _inputs(T, C, heads, act, F32, shared=shared)
    c = {k: t.cuda() for k, t in ins.items()}
    dy = dy.cuda()
    dt, P = npa._lib.BF16 if act == BF16 else npa._lib.F32, ins["weight"].numel()
    nw = lib.nplm_layernorm_bwd_workspace_bytes(T, C, heads)
    PAD = 256
    outs = {k: torch.full((n + 2 * PAD,), 77, dtype=d, device="cuda") for k, (n, d) in
            {"y": (T * C, act), "dx": (T * C, act), "dgate": (T * C, act), "dw": (P, F32), "db": (P, F32), "ws": (nw, torch.uint8)}.items()}
    p = {k: t[PAD:].data_ptr() for k, t in outs.items()}
    at = lambda t: t.data_ptr()
    flags = npa._lib.LAYERNORM_SHARED if shared else 0
    tail = (T, C, heads, dt, npa._lib.F32, flags, torch.cuda.current_stream().cuda_stream)
    assert lib.nplm_layernorm_fwd(at(c["x"]), C, at(c["gate"]), C, at(c["weight"]), at(c["bias"]), 1e-5, p["y"], *tail) == 0
    assert lib.nplm_layernorm_bwd(at(c["x"]), C, at(c["gate"]), C, at(dy), C, at(c["weight"]), at(c["bias"]), 1e-5, p["dx"], p["dgate"], p["dw"], p["db"], p["ws"], nw,
                                  *tail) == 0
    torch.cuda.synchronize()
    for k, t in outs.items():
        assert (t[:PAD] == 77).all() and (t[-PAD:] == 77).all(), k
    got = npa.layer_norm_bwd(c["x"], c["weight"], c["bias"], c["gate"], dy, heads=heads)
    for k, t in zip(("dx", "dgate", "dw", "db"), got):
        assert torch.equal(outs[k][PAD:-PAD], t.flatten()), k


def test_gradients_agree_with_differences():
    ins, dy = _inputs(12, 48, 3, F32, F32, shared=True)
    leaves = {k: t.cuda().requires_grad_() for k, t in ins.items()}
    y = npa.layer_norm(leaves["x"], leaves["weight"], leaves["bias"], gate=leaves["gate"], heads=3)
    grads = torch.autograd.grad(y, list(leaves.values()), dy.cuda())
    g = torch.Generator().manual_seed(1)
    for k, grad in zip(ins, grads):
        d = torch.randn(ins[k].shape, generator=g).double()

        def value(eps):
            moved = {n: t.double() + (eps * d if n == k else 0.0) for n, t in ins.items()}
            return float((_want(moved, None, 3, "layer", 1e-5)["y"][0] * dy.double()).sum())
        want = (value(1e-5) - value(-1e-5)) / 2e-5
        mine = grad.cpu().double() * d
        assert abs(float(mine.sum()) - want) <= 1e-4 * float(mine.abs().sum()), k


@pytest.mark.parametrize("par", [F32, BF16])
def test_the_function_is_the_node_and_results_repeat(par):
    ins, dy = _inputs(700, 192, 3, BF16, par)
    results = []
    for call in (lambda l: npa.layer_norm(l["x"], l["weight"], l["bias"], gate=l["gate"], heads=3, norm="rms"),
                 lambda l: npa.LayerNormFunction.apply(l["x"], l["weight"], l["bias"], l["gate"], 3, "rms", 1e-5)) * 2:
        leaves = {k: t.cuda().requires_grad_() for k, t in ins.items()}
        y = call(leaves)
        results.append([y, *torch.autograd.grad(y, list(leaves.values()), dy.cuda())])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


def test_custom_ops_pass_opcheck_and_compile_without_graph_breaks():
    ins, dy = _inputs(50, 96, 3, F32, F32)
    leaves = [t.cuda().requires_grad_() for t in ins.values()]
    torch.library.opcheck(npa.layer_norm_fwd_op, (*leaves, 3, "rms", 1e-5), test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))

    def f(x, w, b, gate):
        return npa.layer_norm(x * 1.0, w, b, gate=gate, heads=3) * 2.0
    results = []
    for call in (f, torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")):
        y = call(*leaves)
        results.append([y, *torch.autograd.grad(y, leaves, dy.cuda())])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_side_stream_and_graph_replay():
    ins, dy = _inputs(700, 256, 4, BF16, F32, shared=True)
    leaves = [t.cuda().requires_grad_() for t in ins.values()]
    first, dy = leaves[0].detach().clone(), dy.cuda()

    def step():
        y = npa.layer_norm(*leaves[:3], gate=leaves[3], heads=4)
        grads = torch.autograd.grad(y, leaves, dy)
        return [y.detach()] + list(grads)
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
    for n in range(4):
        with torch.no_grad():
            leaves[0].copy_(first * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, got)), n


def test_offsets_beyond_four_gib():
    T, C = 140000, 16384                             # 4.6 GB in bf16
    x = torch.empty(T, C, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(0))
    w = torch.ones(64, device="cuda")
    y = npa.layer_norm(x, w, heads=256)
    dx = npa.layer_norm_bwd(x, w, None, None, x, heads=256)[0]
    want = _want({"x": x[-3:].cpu(), "weight": w.cpu(), "bias": None, "gate": None}, x[-3:].cpu(), 256, "layer", 1e-5)
    R.assert_within(y[-3:], want["y"], "y")
    R.assert_within(dx[-3:], want["x"], "dx")
