"""The gated linear recurrence against the definition in 64 bits (recurrence_ref.py), through the public entry points."""
import pytest
import torch

import nanoplm_amd as npa
from tests import recurrence_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _lengths(kind, T, g):
    if kind == "one":
        return [T]
    out, left = [], T
    while left > 0:
        n = {"rows": lambda: 1, "short": lambda: int(torch.randint(0, 9, (), generator=g)),
             "usual": lambda: int(torch.randint(20, 300, (), generator=g)),
             "mixed": lambda: int(torch.randint(0, 4, (), generator=g)) * int(torch.randint(0, 90, (), generator=g))}[kind]()
        out.append(min(n, left))
        left -= out[-1]
    return out + [0, 0]


def _inputs(T, C, kind, act, par, states, seed=0, decay_std=3.0):
    g = torch.Generator().manual_seed(1000 * seed + T * 7 + C)
    lens = _lengths(kind, T, g)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    n = lambda *s, d=act, m=0.0, std=1.0: (torch.randn(*s, generator=g) * std + m).to(d)
    x, gates, dy = n(T, C), n(T, 2 * C, std=2.0), n(T, C)
    decay = n(C, d=par, std=decay_std, m=-3.0)
    S = len(lens)
    h0, ds = (n(S, C, d=F32), n(S, C, d=F32)) if states else (None, None)
    return x, gates, cu, decay, h0, dy, ds


def _run_and_check(x, gates, cu, decay, h0, dy, ds, reverse, scale=8.0):
    leaves = [None if t is None else t.cuda().requires_grad_() for t in (x, gates, decay, h0)]
    gx, gg, gd, gh = leaves
    out = npa.varlen_recurrence(gx, gg, cu.cuda(), gd, scale=scale, initial_state=gh, reverse=reverse, return_state=ds is not None)
    y, state = out if ds is not None else (out, None)
    h, last, k = R.forward(x, gates, cu, decay, scale, h0, reverse)
    R.assert_within(y, h, k["err"], "y")
    if state is not None:
        ends = torch.zeros_like(last)
        for lo, hi, s in R.sequences(cu, x.shape[0]):
            if s is not None:
                ends[s] = k["err"][lo if reverse else hi - 1]
        R.assert_within(state, last, ends, "state")
    outs, douts = ([y, state], [dy.cuda(), ds.cuda()]) if state is not None else ([y], [dy.cuda()])
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], douts)
    want = R.backward(dy, cu, k, scale, ds, reverse)
    C = x.shape[1]
    R.assert_within(grads[0], *want["dx"], "dx")
    R.assert_within(grads[1][:, :C], *want["dr"], "dr")
    R.assert_within(grads[1][:, C:], *want["di"], "di")
    R.assert_within(grads[2], *want["ddecay"], "ddecay")
    if h0 is not None:
        R.assert_within(grads[3], *want["dinitial"], "dinitial")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act,par", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("T,C,kind,states", [
    (1, 1, "one", True), (2, 2, "rows", True), (7, 3, "one", False), (8, 64, "one", True), (9, 65, "short", True), (63, 128, "one", False),
    (64, 130, "mixed", True), (65, 200, "one", True), (129, 64, "usual", False), (200, 96, "short", True), (517, 70, "mixed", True),
    (1000, 33, "one", True), (777, 128, "usual", True), (1100, 16, "rows", True)])
def test_forward_and_gradients(T, C, kind, states, act, par, reverse):
    _run_and_check(*_inputs(T, C, kind, act, par, states), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lens", [
    [9001], [1, 8192, 64, 64, 0, 640], [511, 512, 513, 64, 1, 4096, 3], [4095, 4097, 0, 0, 100], [64] * 70 + [128, 512, 4096 + 64, 63],
    [3, 30, 5000, 2, 2, 2, 700, 1, 4200]])
def test_long_chains(lens, reverse):
    """Sequences that begin and end in, at and across chunks (64 rows), groups of 8 and of 64 chunks."""
    T, C = sum(lens), 20
    g = torch.Generator().manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=g)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    # slow decays, so that what lies thousands of rows back still counts
    _run_and_check(n(T, C), n(T, 2 * C), cu, n(C) - 8.0, n(len(lens), C), n(T, C), n(len(lens), C), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("C", [65, 70, 129])
@pytest.mark.parametrize("act", [F32, BF16])
def test_two_channels_a_lane(act, C, reverse):
    """Wide slices, with an odd channel or without: boundaries in, at and across chunks, groups of chunks and the state behind 64 of them."""
    lens = [3, 30, 4700, 2, 2, 700, 0, 1, 128, 64, 900]
    T, S = sum(lens), len(lens)
    g = torch.Generator().manual_seed(C)
    n = lambda *s: torch.randn(*s, generator=g)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    _run_and_check(n(T, C).to(act), n(T, 2 * C).to(act), cu, n(C) - 8.0, n(S, C), n(T, C).to(act), n(S, C), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("C", [1, 3, 64, 70])
@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("unit", [32, 64, 128])
def test_sequences_of_whole_chunks(unit, act, C, reverse):
    """Sequences that end with a chunk and cover it, at all places of a group and of a state's 64 chunks."""
    g = torch.Generator().manual_seed(unit + C)
    lens = (torch.randint(1, 13, (60,), generator=g) * unit).tolist()
    T, S = sum(lens), len(lens)
    n = lambda *s: torch.randn(*s, generator=g)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    _run_and_check(n(T, C).to(act), n(T, 2 * C).to(act), cu, n(C) - 8.0, n(S, C), n(T, C).to(act), n(S, C), reverse)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T", [31, 32, 33, 64, 65, 127, 128, 129])
def test_one_chunk_and_a_row_more(T, act):
    for C, reverse in ((40, False), (131, True)):
        _run_and_check(*_inputs(T, C, "mixed", act, F32, True, 7), reverse)


def test_rows_at_any_address():
    """Odd strides and bases: words of two channels that lie across anything."""
    for act, C, off in ((BF16, 97, 1), (BF16, 100, 3), (F32, 67, 1), (F32, 66, 5)):
        x, gates, cu, decay, h0, dy, ds = _inputs(600, C, "mixed", act, F32, True, 9)
        wide = torch.randn(600, off + 4 * C + 1).to(act).cuda()
        parts = wide[:, off:off + C], wide[:, off + C:off + 3 * C], wide[:, off + 3 * C:off + 4 * C]
        for p, t in zip(parts, (x, gates, dy)):
            p.copy_(t)
        args = dict(initial_state=h0.cuda())
        a = npa.varlen_recurrence_fwd(x.cuda(), gates.cuda(), cu.cuda(), decay.cuda(), want_carries=True, want_state=True, **args)
        b = npa.varlen_recurrence_fwd(parts[0], parts[1], cu.cuda(), decay.cuda(), want_carries=True, want_state=True, **args)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        ga = npa.varlen_recurrence_bwd(x.cuda(), gates.cuda(), dy.cuda(), cu.cuda(), decay.cuda(), a[2], dstate=ds.cuda(), want_dinitial=True, **args)
        gb = npa.varlen_recurrence_bwd(*parts[:2], parts[2], cu.cuda(), decay.cuda(), a[2], dstate=ds.cuda(), want_dinitial=True, **args)
        assert all(torch.equal(u, v) for u, v in zip(ga, gb))


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T,C", [(1, 1), (5, 67), (64, 65), (700, 129), (700, 64)])
def test_nothing_around_the_outputs_is_written(T, C, act):
    lib = npa._lib.load()
    x, gates, cu, decay, h0, dy, ds = [t.cuda() for t in _inputs(T, C, "mixed", act, F32, True, 11)]
    S, chunks, dt = h0.shape[0], -(-T // 32), npa._lib.BF16 if act == BF16 else npa._lib.F32
    at = lambda t: None if t is None else t.data_ptr()
    sizes = {"y": (T * C, act), "state": (S * C, F32), "carries": (chunks * C, F32), "dx": (T * C, act), "dgates": (2 * T * C, act), "ddecay": (C, F32),
             "dinitial": (S * C, F32)}
    fw, bw = lib.nplm_recurrence_fwd_workspace_bytes(T, C, S, dt), lib.nplm_recurrence_bwd_workspace_bytes(T, C, S, dt)
    sizes["fw"], sizes["bw"] = (fw, torch.uint8), (bw, torch.uint8)
    PAD = 256
    outs = {k: torch.full((n + 2 * PAD,), 77, dtype=d, device="cuda") for k, (n, d) in sizes.items()}
    o = {k: at(t[PAD:]) for k, t in outs.items()}
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.nplm_recurrence_fwd(at(x), C, at(gates), 2 * C, at(cu), at(decay), 8.0, at(h0), o["y"], o["state"], o["carries"], o["fw"] if fw else None, fw,
                                   T, C, S, dt, npa._lib.F32, 0, stream) == 0
    assert lib.nplm_recurrence_bwd(at(x), C, at(gates), 2 * C, at(dy), C, at(cu), at(decay), 8.0, at(h0), at(ds), o["carries"], o["dx"], o["dgates"],
                                   o["ddecay"], o["dinitial"], o["bw"] if bw else None, bw, T, C, S, dt, npa._lib.F32, 0, stream) == 0
    torch.cuda.synchronize()
    for k, t in outs.items():
        assert (t[:PAD] == 77).all() and (t[-PAD:] == 77).all(), k
    y, state, carries = npa.varlen_recurrence_fwd(x, gates, cu, decay, initial_state=h0, want_state=True, want_carries=True)
    for k, t in (("y", y), ("state", state), ("carries", carries)):
        assert torch.equal(outs[k][PAD:-PAD], t.flatten()), k


@pytest.mark.parametrize("scale,std", [(0.25, 1.0), (8.0, 0.0), (40.0, 4.0)])
def test_scales_and_decays_at_their_ends(scale, std):
    """Decays from e^-40 or so (a state that nothing leaves) to whole forgetting, gates shut and open."""
    x, gates, cu, decay, h0, dy, ds = _inputs(300, 64, "mixed", F32, F32, True, 5, std)
    decay[:8] = torch.linspace(-45, 40, 8)
    gates[:, :16] *= 12
    gates[:, 64:80] *= 12
    _run_and_check(x, gates, cu, decay, h0, dy, ds, False, scale)
    _run_and_check(x, gates, cu, decay, h0, dy, ds, True, scale)


@pytest.mark.parametrize("reverse", [False, True])
def test_nothing_crosses_a_boundary(reverse):
    """A NaN and infinities in one sequence's rows, states and gradients leave the others' bits as they are."""
    x, gates, cu, decay, h0, dy, ds = _inputs(400, 64, "mixed", F32, F32, True, 3)
    S = cu.numel() - 1
    bad = max(range(S), key=lambda s: int(cu[s + 1] - cu[s]))
    lo, hi = int(cu[bad]), int(cu[bad + 1])
    call = lambda *a: _call(*a, reverse)
    clean = call(x, gates, cu, decay, h0, dy, ds)
    x2, g2, h2, dy2, ds2 = (t.clone() for t in (x, gates, h0, dy, ds))
    x2[lo], x2[hi - 1], g2[(lo + hi) // 2, ::3] = float("nan"), float("inf"), float("nan")
    h2[bad], dy2[lo:hi, ::2], ds2[bad] = float("inf"), float("nan"), float("nan")
    dirty = call(x2, g2, cu, decay, h2, dy2, ds2)
    rows = torch.ones(400, dtype=torch.bool)
    rows[lo:hi] = False
    seqs = torch.arange(S) != bad
    for name, a, b in zip(("y", "state", "dx", "dgates", "dinitial"), clean, dirty):
        keep = rows if a.shape[0] == 400 else seqs
        assert torch.equal(a[keep], b[keep]), name


def _call(x, gates, cu, decay, h0, dy, ds, reverse):
    c = lambda t: t.cuda()
    y, state, carries = npa.varlen_recurrence_fwd(c(x), c(gates), c(cu), c(decay), initial_state=c(h0), reverse=reverse, want_state=True,
                                                  want_carries=True)
    dx, dgates, _, dinitial = npa.varlen_recurrence_bwd(c(x), c(gates), c(dy), c(cu), c(decay), carries, initial_state=c(h0), dstate=c(ds),
                                                        reverse=reverse, want_dinitial=True)
    return [t.cpu() for t in (y, state, dx, dgates, dinitial)]


@pytest.mark.parametrize("reverse", [False, True])
def test_rows_outside_cu_are_sequences_of_their_own(reverse):
    x, gates, _, decay, _, dy, _ = _inputs(150, 40, "one", F32, F32, False)
    for cu in ([10, 30, 30, 140], [0], [150], [5], [0, 150], [70, 70]):
        cu = torch.tensor(cu, dtype=torch.int32)
        S = cu.numel() - 1
        g = torch.Generator().manual_seed(S)
        _run_and_check(x, gates, cu, decay, torch.randn(S, 40, generator=g), dy, torch.randn(S, 40, generator=g), reverse)


def test_thousands_of_sequences_and_runs_of_empty_ones():
    x, gates, _, decay, _, dy, _ = _inputs(600, 16, "one", F32, F32, False)
    for lens in ([0] * 5000 + [100] + [0] * 70 + [200, 1, 1] + [0] * 130 + [298] + [0] * 9000, [1] * 600 + [0] * 300, [0, 0, 0] * 2000 + [600]):
        cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
        S = len(lens)
        g = torch.Generator().manual_seed(S)
        for reverse in (False, True):
            _run_and_check(x, gates, cu, decay, torch.randn(S, 16, generator=g), dy, torch.randn(S, 16, generator=g), reverse)


@pytest.mark.parametrize("act", [F32, BF16])
def test_column_slices_and_other_strides(act):
    """x and gates as column slices of one wider projection, at offsets that are not aligned to anything, and a transposed dy."""
    for C, off, pad in ((64, 0, 0), (64, 1, 5), (33, 2, 0), (128, 8, 8)):
        x, gates, cu, decay, h0, dy, ds = _inputs(130, C, "mixed", act, F32, True)
        wide = torch.randn(130, off + 3 * C + pad).to(act).cuda()
        wide[:, off:off + C], wide[:, off + C:off + 3 * C] = x.cuda(), gates.cuda()
        sx, sg = wide[:, off:off + C], wide[:, off + C:off + 3 * C]
        dyt = dy.cuda().t().contiguous().t()
        args = dict(initial_state=h0.cuda())
        a = npa.varlen_recurrence_fwd(x.cuda(), gates.cuda(), cu.cuda(), decay.cuda(), want_carries=True, want_state=True, **args)
        b = npa.varlen_recurrence_fwd(sx, sg, cu.cuda(), decay.cuda(), want_carries=True, want_state=True, **args)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        ga = npa.varlen_recurrence_bwd(x.cuda(), gates.cuda(), dy.cuda(), cu.cuda(), decay.cuda(), a[2], dstate=ds.cuda(), want_dinitial=True, **args)
        gb = npa.varlen_recurrence_bwd(sx, sg, dyt, cu.cuda(), decay.cuda(), a[2], dstate=ds.cuda(), want_dinitial=True, **args)
        assert all(torch.equal(u, v) for u, v in zip(ga, gb))


def test_gradients_agree_with_differences():
    """The directional derivative of a weighted sum of the outputs, by central differences of the fp64 definition at the kernel's inputs."""
    x, gates, cu, decay, h0, dy, ds = _inputs(90, 24, "mixed", F32, F32, True)
    leaves = [t.cuda().requires_grad_() for t in (x, gates, decay, h0)]
    y, state = npa.varlen_recurrence(leaves[0], leaves[1], cu.cuda(), leaves[2], initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad([y, state], leaves, [dy.cuda(), ds.cuda()])
    g = torch.Generator().manual_seed(1)
    for i, t in enumerate((x, gates, decay, h0)):
        d = torch.randn(t.shape, generator=g)

        def value(eps):
            args = [u.double() for u in (x, gates, decay, h0)]
            args[i] = args[i] + eps * d.double()
            h, last, _ = R.forward(args[0], args[1], cu, args[2], 8.0, args[3])
            return float((h * dy.double()).sum() + (last * ds.double()).sum())
        want = (value(1e-5) - value(-1e-5)) / 2e-5
        got = float((grads[i].cpu().double() * d.double()).sum())
        size = float((grads[i].cpu().double() * d.double()).abs().sum())
        assert abs(got - want) <= 1e-4 * size, (i, got, want)


@pytest.mark.parametrize("reverse", [False, True])
def test_a_sequence_in_pieces_is_the_sequence(reverse):
    x, gates, _, decay, _, dy, _ = _inputs(500, 72, "one", F32, F32, False)
    x, gates, decay = x.cuda(), gates.cuda(), decay.cuda()
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32).cuda()
    h0 = torch.randn(1, 72).cuda()
    y, state = npa.varlen_recurrence(x, gates, cu(500), decay, initial_state=h0, reverse=reverse, return_state=True)
    parts, s = [], h0
    bounds = [0, 1, 64, 200, 333, 500]
    spans = list(zip(bounds[:-1], bounds[1:]))
    for a, b in reversed(spans) if reverse else spans:
        part, s = npa.varlen_recurrence(x[a:b], gates[a:b], cu(b - a), decay, initial_state=s, reverse=reverse, return_state=True)
        parts.append(part)
    whole = torch.cat(parts[::-1] if reverse else parts)
    h, _, k = R.forward(x.cpu(), gates.cpu(), [0, 500], decay.cpu(), 8.0, h0.cpu(), reverse)
    R.assert_within(whole, h, k["err"], "pieces")
    R.assert_within(y, h, k["err"], "whole")
    assert float((s - state).abs().max()) <= 2 * float(k["err"].max())


def test_results_repeat_bit_for_bit():
    x, gates, cu, decay, h0, dy, ds = _inputs(4000, 128, "mixed", BF16, BF16, True)
    first = _call(x, gates, cu, decay, h0, dy, ds, False)
    for _ in range(3):
        again = _call(x, gates, cu, decay, h0, dy, ds, False)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_empty_batches():
    z = lambda *s: torch.zeros(*s, device="cuda", requires_grad=True)
    x, gates, decay, h0 = z(0, 8), z(0, 16), z(8), torch.randn(3, 8, device="cuda", requires_grad=True)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    y, state = npa.varlen_recurrence(x, gates, cu, decay, initial_state=h0, return_state=True)
    assert y.shape == (0, 8) and torch.equal(state, h0)
    ds = torch.randn(3, 8, device="cuda")
    dx, dgates, ddecay, dh = torch.autograd.grad([y, state], [x, gates, decay, h0], [torch.zeros_like(y), ds])
    assert dx.shape == (0, 8) and dgates.shape == (0, 16) and torch.equal(ddecay, torch.zeros(8, device="cuda")) and torch.equal(dh, ds)
    y, state = npa.varlen_recurrence(x, gates, cu, decay, return_state=True)
    assert torch.equal(state, torch.zeros(3, 8, device="cuda"))


# ---- single tokens ----------------------------------------------------------------------------------------------------------------------
def _step_ref(x, gates, decay, state, slots, scale=8.0):
    k = R.coefficients(x, gates, decay, scale)
    table, y = state.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    err = torch.zeros_like(table)
    bound = torch.zeros_like(y)
    for b, s in enumerate(slots):
        if 0 <= s < table.shape[0]:
            e = k["a"][b] * err[s] + k["da"][b] * table[s].abs() + k["eb"][b] * k["b"][b].abs()
            big = k["a"][b] * table[s].abs() + k["b"][b].abs()
            table[s] = k["a"][b] * table[s] + k["b"][b]
            err[s] = e + 3 * R.U * big
            y[b], bound[b] = table[s], err[s]
    return y, bound, table, err


@pytest.mark.parametrize("act,par", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("B,C,N,slots", [
    (1, 1, 1, None), (1, 1024, 8, [5]), (3, 257, 3, None), (5, 64, 9, [8, 0, 3, -1, 7]), (6, 300, 4, [2, 2, 0, 2, 0, 99]), (4, 31, 2, [-1, -7, 2, 5]),
    (300, 65, 500, "mixed")])
def test_step(B, C, N, slots, act, par):
    g = torch.Generator().manual_seed(B + C)
    x, gates = torch.randn(B, C, generator=g).to(act), torch.randn(B, 2 * C, generator=g).to(act)
    decay, state = (torch.randn(C, generator=g) - 3).to(par), torch.randn(N, C, generator=g)
    if slots == "mixed":
        slots = torch.randint(-30, 530, (B,), generator=g).tolist()
    named = list(range(B)) if slots is None else slots
    y64, by, t64, bt = _step_ref(x, gates, decay, state, named)
    table, other = state.cuda(), torch.full((N, C), -3.0, device="cuda")
    ids = None if slots is None else torch.tensor(slots, dtype=torch.int32).cuda()
    y2 = npa.recurrence_step(x.cuda(), gates.cuda(), decay.cuda(), table, ids, out_state=other)
    assert torch.equal(table.cpu(), state)                      # the old states stay
    y = npa.recurrence_step(x.cuda(), gates.cuda(), decay.cuda(), table, ids)
    R.assert_within(y, y64, by, "y")
    R.assert_within(table, t64, bt, "state")
    assert torch.equal(y, y2)
    touched = sorted({s for s in named if 0 <= s < N})
    rest = [s for s in range(N) if s not in touched]
    assert torch.equal(other[touched], table[touched]) and bool((other[rest] == -3.0).all()) and torch.equal(table[rest].cpu(), state[rest])


def test_steps_continue_a_prompt():
    """A packed prompt of three sequences, then their next tokens one by one through a table of states, against the sequences run whole."""
    C, lens, more = 80, [50, 1, 130], 4
    g = torch.Generator().manual_seed(2)
    m = npa.VarlenRecurrence(C).cuda()
    parts = [(torch.randn(n + more, C, generator=g), torch.randn(n + more, 2 * C, generator=g)) for n in lens]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    cat = lambda k, f: torch.cat([f(p[k], n) for p, n in zip(parts, lens)]).cuda()
    with torch.no_grad():
        _, state = m(cat(0, lambda t, n: t[:n]), cat(1, lambda t, n: t[:n]), cu, return_state=True)
        table = torch.zeros(10, C, device="cuda")
        slots = torch.tensor([7, 0, 3], dtype=torch.int32).cuda()
        table[slots.long()] = state
        got = [m.step(cat(0, lambda t, n: t[n + j:n + j + 1]), cat(1, lambda t, n: t[n + j:n + j + 1]), table, slots) for j in range(more)]
    for s, (n, (x, gates)) in enumerate(zip(lens, parts)):
        h, _, k = R.forward(x, gates, [0, n + more], m.decay.detach().cpu())
        R.assert_within(torch.stack([y[s] for y in got]), h[n:], k["err"][n:], f"sequence {s}")


# ---- the framework's surfaces -----------------------------------------------------------------------------------------------------------
def test_padded_door_gives_each_sequence_its_packed_results():
    B, L, C = 4, 70, 48
    lens = [70, 1, 33, 0]
    mask = torch.arange(L)[None] < torch.tensor(lens)[:, None]
    m = npa.VarlenRecurrence(C).cuda()
    x, gates = torch.randn(B, L, C, device="cuda"), torch.randn(B, L, 2 * C, device="cuda")
    y = m.forward_padded(x, gates, mask.cuda())
    for b, n in enumerate(lens):
        alone = m(x[b, :n].contiguous(), gates[b, :n].contiguous(), torch.tensor([0, n], dtype=torch.int32).cuda())
        err = R.forward(x[b, :n].cpu(), gates[b, :n].cpu(), [0, n], m.decay.detach().cpu())[2]["err"]
        assert bool(((y[b, :n] - alone).abs().cpu().double() <= 2 * err + 1e-7 * alone.abs().cpu().double()).all())


def test_frozen_inputs_and_missing_gradients():
    x, gates, cu, decay, h0, dy, ds = (t.cuda() for t in _inputs(100, 32, "mixed", F32, F32, True))
    lam = decay.clone().requires_grad_()
    y, state = npa.varlen_recurrence(x, gates, cu, lam, initial_state=h0, return_state=True)
    (state * ds).sum().backward()                               # no gradient reaches y
    want = npa.varlen_recurrence_bwd(x, gates, torch.zeros_like(x), cu, decay, npa.varlen_recurrence_fwd(
        x, gates, cu, decay, initial_state=h0, want_carries=True)[2], initial_state=h0, dstate=ds)[2]
    assert torch.equal(lam.grad, want)
    gx = x.clone().requires_grad_()
    npa.varlen_recurrence(gx, gates, cu, decay).backward(dy)
    assert gx.grad is not None


def test_custom_ops_pass_opcheck_and_compile_without_graph_breaks():
    x, gates, cu, decay, h0, dy, ds = (t.cuda() for t in _inputs(100, 32, "mixed", F32, F32, True))
    ins = tuple(t.requires_grad_() for t in (x, gates)) + (cu, decay.requires_grad_(), h0.requires_grad_(), 8.0, False)
    torch.library.opcheck(npa.varlen_recurrence_fwd_op, ins, test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))

    def f(x, gates, decay, h0):
        y, s = npa.varlen_recurrence(x * 1.0, gates, cu, decay, initial_state=h0, return_state=True)
        return y * 2.0, s
    eager = f(x, gates, decay, h0)
    g1 = torch.autograd.grad(eager, [x, gates, decay, h0], [dy, ds])
    got = torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")(x, gates, decay, h0)
    g2 = torch.autograd.grad(got, [x, gates, decay, h0], [dy, ds])
    assert all(torch.equal(a, b) for a, b in zip(list(eager) + list(g1), list(got) + list(g2)))


def test_side_stream_and_graph_replay():
    x, gates, cu, decay, h0, dy, ds = (t.cuda() for t in _inputs(700, 64, "mixed", BF16, F32, True))
    leaves = [t.clone().requires_grad_() for t in (x, gates, decay, h0)]

    def step():
        y, s = npa.varlen_recurrence(leaves[0], leaves[1], cu, leaves[2], initial_state=leaves[3], return_state=True)
        grads = torch.autograd.grad([y, s], leaves, [dy, ds])
        return [y.detach(), s.detach()] + list(grads)          # (no eager graph of the leaves may live while the step is captured)
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
            leaves[0].copy_(x * (k + 1))
            leaves[3].copy_(h0 * (1 - k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, got)), k


def test_offsets_beyond_four_gib():
    """Rows whose gates begin beyond 4 GiB: the last sequence is what it is alone."""
    T, C = 300000, 4096                              # gates: 4.6 GiB in bf16
    g = torch.Generator("cuda").manual_seed(0)
    gates = torch.empty(T, 2 * C, dtype=BF16, device="cuda").normal_(generator=g)
    x = torch.empty(T, C, dtype=BF16, device="cuda").normal_(generator=g)
    decay = torch.full((C,), -4.0, device="cuda")
    cut = T - 200
    cu = torch.tensor([0, 17, cut, T], dtype=torch.int32).cuda()
    y, _, carries = npa.varlen_recurrence_fwd(x, gates, cu, decay, want_carries=True)
    h, _, k = R.forward(x[cut:].cpu(), gates[cut:].cpu(), [0, 200], decay.cpu())
    R.assert_within(y[cut:], h, k["err"], "y")
    dy = torch.zeros(T, C, dtype=BF16, device="cuda")
    dy[cut:].normal_(generator=g)
    dx, dgates, _, _ = npa.varlen_recurrence_bwd(x, gates, dy, cu, decay, carries)
    want = R.backward(dy[cut:].cpu(), [0, 200], k)
    R.assert_within(dx[cut:], *want["dx"], "dx")
    R.assert_within(dgates[cut:, :C], *want["dr"], "dr")
    R.assert_within(dgates[cut:, C:], *want["di"], "di")
    assert not bool(dx[:cut].any())
