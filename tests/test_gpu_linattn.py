"""Linear attention and its step against the definition in 64 bits (linattn_ref.py), through the public entry points."""
import pytest
import torch

import nanoplm_amd as npa
from tests import linattn_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("q", "k", "v", "log_decay", "initial")


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


def _inputs(lens, H, K, V, act, gdt, rate, states, seed=0, T=None, spread=3.0, mean=3.0):
    T, S = sum(lens) if T is None else T, len(lens)
    g = torch.Generator().manual_seed(1000 * seed + T * 7 + K)
    n = lambda *s, d=act: torch.randn(*s, generator=g).to(d)
    x = {"q": n(T, H, K), "k": n(T, H, K), "v": n(T, H, V)}
    x["log_decay"] = torch.nn.functional.logsigmoid(torch.randn(*((H,) if rate == "head" else (T, H)), generator=g) * spread + mean).to(gdt)
    x["initial"], x["dstate"] = (n(S, H, K, V, d=F32), n(S, H, K, V, d=F32)) if states else (None, None)
    x["do"] = n(T, H, V)
    x["cu"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    return x


def _call(x, reverse, scale, grads=True):
    """Outputs and gradients by name."""
    leaves = {n: None if x[n] is None else x[n].cuda().requires_grad_(grads) for n in NAMES}
    out = npa.varlen_linear_attention(leaves["q"], leaves["k"], leaves["v"], x["cu"].cuda(), leaves["log_decay"], scale=scale, initial_state=leaves["initial"],
                                      reverse=reverse, return_state=x["dstate"] is not None)
    o, state = out if x["dstate"] is not None else (out, None)
    got = {"o": o} if state is None else {"o": o, "state": state}
    if grads:
        there = [n for n in NAMES if leaves[n] is not None]
        douts = [x["do"].cuda()] + ([] if state is None else [x["dstate"].cuda()])
        for n, d in zip(there, torch.autograd.grad(list(got.values()), [leaves[n] for n in there], douts)):
            assert d.dtype == x[n].dtype
            got["d" + n] = d
    return got


def _run_and_check(x, reverse, scale=None, near=True, on="cpu", grads=True):
    got = _call(x, reverse, scale, grads)
    c = lambda t: None if t is None else t.to(on)
    want = R.run(c(x["q"]), c(x["k"]), c(x["v"]), x["cu"], c(x["log_decay"]), x["q"].shape[2] ** -0.5 if scale is None else scale, c(x["initial"]), reverse,
                 c(x["do"]) if grads else None, c(x["dstate"]))
    for n, t in got.items():
        R.assert_within(t, want[n], n, near and n != "dlog_decay")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act,gdt,rate", [(F32, F32, "token"), (F32, F32, "head"), (BF16, BF16, "token"), (BF16, F32, "head"), (BF16, F32, "token")])
@pytest.mark.parametrize("T,H,K,V,kind,states", [
    (1, 1, 1, 1, "one", True), (2, 3, 2, 5, "rows", True), (7, 1, 3, 8, "one", False), (8, 2, 16, 16, "one", True), (31, 1, 32, 32, "short", True),
    (33, 2, 64, 64, "one", False), (64, 2, 33, 65, "mixed", True), (65, 1, 128, 128, "one", True), (129, 2, 64, 128, "usual", False),
    (200, 1, 96, 40, "short", True), (330, 3, 48, 91, "mixed", True), (130, 2, 128, 64, "usual", True), (70, 5, 20, 12, "rows", True)])
def test_forward_and_gradients(T, H, K, V, kind, states, act, gdt, rate, reverse):
    lens = _lengths(kind, T, torch.Generator().manual_seed(T))
    _run_and_check(_inputs(lens, H, K, V, act, gdt, rate, states), reverse)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("lens", [[700], [64, 65, 128, 0, 1, 300, 63, 700], [127, 128, 129, 200], [1, 640, 64, 64, 0, 192, 3], [30, 31, 32, 33, 260, 2, 2, 700]])
def test_sequences_of_several_segments(lens, act, reverse):
    """Segments of 64 rows (few heads): sequences that begin and end in, at and across them, slow decays, so that what lies hundreds of rows back still counts."""
    assert npa._lib.load().nplm_linattn_debug_segment_rows(sum(lens), 2, len(lens)) == 64
    for rate, gdt in (("token", act), ("head", F32)):
        _run_and_check(_inputs(lens, 2, 24, 20, act, gdt, rate, True, spread=1.0, mean=6.0), reverse)
    _run_and_check(_inputs(lens, 2, 24, 20, act, act, "token", False, 1, spread=1.0, mean=6.0), reverse)


@pytest.mark.parametrize("act", [F32, BF16])
def test_segments_of_all_lengths(act):
    rows = npa._lib.load().nplm_linattn_debug_segment_rows
    for lens, L in (([3000, 128, 129, 0, 1, 1100], 128), ([2500, 192, 193, 1, 3000], 192), ([1500, 512, 513, 0, 1024, 2400], 512), ([2048, 2049, 0, 1, 30], 2048)):
        H = next(H for H in range(1, 200) if rows(sum(lens), H, len(lens)) == L)
        for reverse in (False, True):
            _run_and_check(_inputs(lens, H, 6, 5, act, act, "token", True, spread=1.0, mean=7.0), reverse, on="cuda")


@pytest.mark.parametrize("reverse", [False, True])
def test_small_batches_without_boundaries(reverse):
    """Short sequences on the average, one of them of many chunks: no states are kept between forward and backward."""
    lens = [900] + [3] * 9
    assert npa._lib.load().nplm_linattn_bounds_bytes(sum(lens), 2, len(lens), 24, 20, npa._lib.BF16) == 0
    for act in (F32, BF16):
        _run_and_check(_inputs(lens, 2, 24, 20, act, F32, "token", True, spread=1.0, mean=6.0), reverse)


@pytest.mark.parametrize("act", [F32, BF16])
def test_strides_alignments_and_shared_heads(act):
    """Column slices of one projection at any offset, transposed heads, expanded keys and values: bits of contiguous tensors, gradients summed by autograd."""
    for K, V, off in ((64, 64, 0), (64, 64, 1), (40, 56, 8), (33, 21, 3), (128, 64, 4)):
        x = _inputs([70, 0, 90], 3, K, V, act, act, "token", False, 2)
        T, H = 160, 3
        c = {n: x[n].cuda() for n in ("q", "k", "v", "do", "log_decay")}
        wide = torch.randn(T, off + H * (2 * K + V) + 5, device="cuda").to(act)
        views, at = {}, off
        for n, d in (("q", K), ("k", K), ("v", V)):
            views[n] = wide[:, at:at + H * d].view(T, H, d)
            views[n].copy_(c[n])
            at += H * d
        views["do"] = torch.empty(H, T, V, device="cuda", dtype=act).transpose(0, 1).copy_(c["do"])
        views["log_decay"] = torch.empty(H, T, device="cuda", dtype=act).t().copy_(c["log_decay"])
        results = []
        for src in (c, views):
            o, _, bounds = npa.varlen_linear_attention_fwd(src["q"], src["k"], src["v"], x["cu"].cuda(), src["log_decay"])
            results.append([o, *npa.varlen_linear_attention_bwd(src["q"], src["k"], src["v"], src["do"], x["cu"].cuda(), src["log_decay"], bounds)[:4]])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        one = {n: c[n][:, :1].clone().requires_grad_() for n in ("k", "v")}
        q = c["q"].clone().requires_grad_()
        o = npa.varlen_linear_attention(q, one["k"].expand(T, H, K), one["v"].expand(T, H, V), x["cu"].cuda(), c["log_decay"])
        shared = torch.autograd.grad(o, [q, one["k"], one["v"]], views["do"])
        full = {n: t.detach().expand(T, H, -1).contiguous().requires_grad_() for n, t in one.items()}
        o2 = npa.varlen_linear_attention(q, full["k"], full["v"], x["cu"].cuda(), c["log_decay"])
        apart = torch.autograd.grad(o2, [q, full["k"], full["v"]], c["do"])
        assert torch.equal(o, o2) and torch.equal(shared[0], apart[0])
        assert all(torch.equal(s, a.sum(1, keepdim=True)) for s, a in zip(shared[1:], apart[1:]))


def test_a_gradient_that_is_one_number():
    x = _inputs([100], 2, 16, 24, F32, F32, "token", False)
    q = x["q"].cuda().requires_grad_()
    rest = x["k"].cuda(), x["v"].cuda(), x["cu"].cuda(), x["log_decay"].cuda()
    npa.varlen_linear_attention(q, *rest).sum().backward()
    (want,) = torch.autograd.grad(npa.varlen_linear_attention(q, *rest), [q], torch.ones(100, 2, 24, device="cuda"))
    assert torch.equal(q.grad, want)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act", [F32, BF16])
def test_decays_at_their_ends(act, reverse):
    """States that are kept whole, forgotten altogether (-inf and what is 0 in fp32), and every strength beside each other in one chunk."""
    x = _inputs([300, 1, 70], 3, 24, 20, act, F32, "token", True, 4)
    g = x["log_decay"]
    g[:, 0] = 0.0
    g[::7, 1], g[3::11, 1], g[5::13, 1] = -float("inf"), -150.0, -1e30
    g[:, 2] = -torch.rand(371, generator=torch.Generator().manual_seed(0)) * 60
    _run_and_check(x, reverse, near=False)
    x = _inputs([200], 4, 16, 16, act, F32, "head", True, 5)
    x["log_decay"] = torch.tensor([0.0, -float("inf"), -1e-6, -90.0])
    _run_and_check(x, reverse, near=False)


@pytest.mark.parametrize("scale", [0.0, -2.5, 30.0])
def test_scales(scale):
    _run_and_check(_inputs([130, 40], 2, 24, 20, F32, F32, "token", True), False, scale)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act", [F32, BF16])
def test_nothing_crosses_a_boundary(act, reverse):
    """NaN and infinities in one sequence's rows, states, decays and gradients leave the others' bits as they are; within it, rows 64 and more in front of the first."""
    lens = [40, 0, 300, 1, 90, 64]
    x = _inputs(lens, 2, 24, 20, act, F32, "token", True, 3)
    clean = _call(x, reverse, None)
    y = {n: t if t is None else t.clone() for n, t in x.items()}
    lo, hi = 40, 340
    mid = 200
    y["q"][mid], y["k"][mid + 1], y["v"][mid - 1, :, ::3], y["log_decay"][mid, 1] = float("nan"), float("inf"), float("nan"), float("nan")
    y["initial"][2, 0, 3], y["dstate"][2], y["do"][mid, :, 1] = float("inf"), float("nan"), -float("inf")
    dirty = _call(y, reverse, None)
    rows = torch.ones(sum(lens), dtype=torch.bool)
    rows[lo:hi] = False
    seqs = torch.arange(len(lens)) != 2
    for n, a in clean.items():
        keep = rows if a.shape[0] == sum(lens) else seqs
        assert torch.equal(a[keep.cuda()], dirty[n][keep.cuda()]), n
    y["initial"][2] = x["initial"][2]
    far = slice(mid + 66, hi) if reverse else slice(lo, mid - 65)                 # (rows in front, in the walk's order)
    assert torch.equal(_call(y, reverse, None, False)["o"][far], clean["o"][far])


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("K,V", [(24, 30), (64, 64), (40, 128), (128, 64), (128, 128), (91, 91)])
@pytest.mark.parametrize("lens,states", [([70, 200, 130], False), ([70, 200, 130, 0], True)])
def test_what_is_not_finite_reaches_the_rows_behind_it_and_no_others(lens, states, K, V, act, reverse):
    """An infinity or NaN stands behind scores that are masked: all of o and of the last states that does not read it has the very bits that it has without. In segments (three
    sequences of 400 rows) and whole (four)."""
    x = _inputs(lens, 2, K, V, act, F32, "token", states)
    clean = _call(x, reverse, None, False)
    end, h, column = lens[0] + lens[1], 1, 5
    for at, value in ((0, float("nan")), (37, float("inf")), (131, float("-inf")), (170, float("nan")), (199, float("inf"))):
        for bad in ("q", "k", "v", "log_decay"):
            row = lens[0] + at
            y = {**x, bad: x[bad].clone()}
            y[bad][(row, h) if bad == "log_decay" else (row, h, column)] = float("nan") if bad == "log_decay" else value
            got = _call(y, reverse, None, False)
            reached = {n: torch.zeros(t.shape, dtype=torch.bool, device="cuda") for n, t in got.items()}
            rows = slice(row, row + 1) if bad == "q" else slice(lens[0], row + 1) if reverse else slice(row, end)
            reached["o"][rows, h, column if bad == "v" else slice(None)] = True
            if states and bad != "q":
                reached["state"][{"k": (1, h, column), "v": (1, h, slice(None), column), "log_decay": (1, h)}[bad]] = True
            for n, t in got.items():
                assert not torch.isfinite(t[reached[n]]).any(), (n, bad, at)
                assert torch.equal(t[~reached[n]], clean[n][~reached[n]]), (n, bad, at)


@pytest.mark.parametrize("reverse", [False, True])
def test_rows_outside_cu_are_sequences_of_their_own(reverse):
    for cu in ([10, 30, 30, 140], [0], [150], [5], [0, 150], [70, 70]):
        x = _inputs([0] * (len(cu) - 1), 2, 12, 10, F32, F32, "token", True, T=150)
        x["cu"] = torch.tensor(cu, dtype=torch.int32)
        _run_and_check(x, reverse)


def test_thousands_of_sequences_and_runs_of_empty_ones():
    for lens in ([0] * 500 + [100] + [0] * 70 + [200, 1, 1] + [0] * 130 + [98] + [0] * 900, [1] * 300 + [0] * 300, [0, 0, 0] * 300 + [400]):
        for reverse in (False, True):
            _run_and_check(_inputs(lens, 1, 8, 4, F32, F32, "token", True), reverse)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("lens,H,K,V", [([1], 1, 1, 1), ([5, 0, 60], 2, 33, 20), ([300], 2, 64, 128), ([230, 70], 3, 128, 91)])
def test_nothing_around_the_outputs_is_written(lens, H, K, V, act):
    lib, L = npa._lib.load(), npa._lib
    x = _inputs(lens, H, K, V, act, F32, "token", True, 6)
    T, S, dt = sum(lens), len(lens), npa._lib.BF16 if act == BF16 else npa._lib.F32
    x = {n: t.cuda() for n, t in x.items()}
    at = lambda t: t.data_ptr()
    nb, nw = lib.nplm_linattn_bounds_bytes(T, H, S, K, V, dt), lib.nplm_linattn_bwd_workspace_bytes(T, H, S, K, V, dt)
    sizes = {"o": (T * H * V, act), "state": (S * H * K * V, F32), "dq": (T * H * K, act), "dk": (T * H * K, act), "dv": (T * H * V, act), "dlog_decay": (T * H, F32),
             "dinitial": (S * H * K * V, F32), "bounds": (nb, torch.uint8), "work": (nw, torch.uint8)}
    PAD = 256
    outs = {n: torch.full((m + 2 * PAD,), 77, dtype=d, device="cuda") for n, (m, d) in sizes.items()}
    p = {n: at(t[PAD:]) for n, t in outs.items()}
    qkv = (at(x["q"]), H * K, K, at(x["k"]), H * K, K, at(x["v"]), H * V, V)
    rates = (at(x["cu"]), at(x["log_decay"]), H, 1, K ** -0.5, at(x["initial"]))
    tail = (T, H, S, K, V, dt, L.F32, 0, torch.cuda.current_stream().cuda_stream)
    assert lib.nplm_linattn_fwd(*qkv, *rates, p["o"], p["state"], p["bounds"] if nb else None, nb, *tail) == 0
    assert lib.nplm_linattn_bwd(*qkv, at(x["do"]), H * V, V, *rates, p["state"], at(x["dstate"]), p["bounds"] if nb else None, nb, p["dq"], p["dk"], p["dv"],
                                p["dlog_decay"], p["dinitial"], p["work"], nw, *tail) == 0
    torch.cuda.synchronize()
    for n, t in outs.items():
        assert (t[:PAD] == 77).all() and (t[-PAD:] == 77).all(), n
    want = _call({n: t.cpu() for n, t in x.items()}, False, None)
    for n, t in want.items():
        assert torch.equal(outs[n][PAD:-PAD], t.flatten()), n


def test_gradients_agree_with_differences():
    """The directional derivative of a weighted sum of the outputs, by central differences of the fp64 definition at the kernel's inputs."""
    x = _inputs([50, 0, 40], 2, 12, 10, F32, F32, "token", True)
    got = _call(x, False, None)
    g = torch.Generator().manual_seed(1)
    for n in NAMES:
        d = torch.randn(x[n].shape, generator=g)

        def value(eps):
            y = {m: x[m].double() + (eps * d.double() if m == n else 0.0) for m in NAMES}
            out = R.run(y["q"], y["k"], y["v"], x["cu"], y["log_decay"], 12 ** -0.5, y["initial"])
            return float((out["o"][0] * x["do"].double()).sum() + (out["state"][0] * x["dstate"].double()).sum())
        want = (value(1e-5) - value(-1e-5)) / 2e-5
        mine = got["d" + n].cpu().double() * d.double()
        assert abs(float(mine.sum()) - want) <= 1e-4 * float(mine.abs().sum()), (n, float(mine.sum()), want)


@pytest.mark.parametrize("decay", [0.5, 0.97])
@pytest.mark.parametrize("act,H,K,V,kind", [(F32, 32, 64, 64, k) for k in ("even", "state", "first", "growing", "end", "both")] +
                         [(F32, 24, 128, 40, "state"), (BF16, 32, 64, 64, "even"), (BF16, 32, 64, 64, "state"), (BF16, 24, 128, 64, "end"), (BF16, 32, 32, 20, "first")])
def test_one_decay_a_head_is_no_worse_than_the_sum_of_rows(act, H, K, V, kind, decay):
    """The gradient of one decay a head in fp32 has the errors of 2048 rows' sums, and knows what these must come to. Whatever sizes the rows' and the states' terms have, that may not
    make it worse than the sum of the same rows' own gradients (which also have a rounding each): both have the same errors in their rows, so that the rms over
    the heads is compared within 1.5, four times the 1 / sqrt(2 H) that either rms varies by."""
    T, S = 2048, 16                                              # (empty sequences behind: the longest segment there is)
    x = _inputs([T] + [0] * (S - 1), H, K, V, act, F32, "head", True, seed=3)
    x["log_decay"] = torch.full((H,), decay, dtype=torch.float64).log().float()
    x["initial"] *= {"state": 1000.0, "both": 100.0}.get(kind, 0.0)
    x["dstate"] *= {"end": 100.0, "both": 100.0}.get(kind, 0.0)
    if kind == "first":
        x["k"][0] *= 1024.0
    if kind == "growing":
        x["k"] *= torch.linspace(0, 7, T).exp()[:, None, None].to(act)
    c = lambda n: x[n].cuda()
    want = R.run(*(c(n) for n in ("q", "k", "v")), x["cu"], c("log_decay"), K ** -0.5, c("initial"), False, c("do"), c("dstate"))["dlog_decay"][0]
    one = _call(x, False, None)["dlog_decay"].double()
    x["log_decay"] = x["log_decay"].expand(T, H).contiguous()
    rows = _call(x, False, None)["dlog_decay"].double()
    rms = lambda t: float(t.square().mean().sqrt())
    rounding = rms(want) * R.U + rms(rows.norm(dim=0)) * R.U
    assert rms(one - want) <= 1.5 * rms(rows.sum(0) - want) + rounding


@pytest.mark.parametrize("reverse", [False, True])
def test_a_sequence_in_pieces_is_the_sequence(reverse):
    x = _inputs([500], 2, 24, 20, F32, F32, "token", True)
    c = {n: x[n].cuda() for n in ("q", "k", "v", "log_decay")}
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32).cuda()
    parts, s = [], x["initial"].cuda()
    bounds = [0, 1, 64, 200, 333, 500]
    spans = list(zip(bounds[:-1], bounds[1:]))
    for a, b in reversed(spans) if reverse else spans:
        part, s = npa.varlen_linear_attention(c["q"][a:b], c["k"][a:b], c["v"][a:b], cu(b - a), c["log_decay"][a:b], initial_state=s, reverse=reverse, return_state=True)
        parts.append(part)
    want = R.run(x["q"], x["k"], x["v"], [0, 500], x["log_decay"], 24 ** -0.5, x["initial"], reverse)
    R.assert_within(torch.cat(parts[::-1] if reverse else parts), want["o"], "pieces")
    R.assert_within(s, want["state"], "state")


def test_results_repeat_bit_for_bit():
    x = _inputs([1000, 3, 700, 0, 2000], 4, 64, 128, BF16, F32, "head", True)
    first = _call(x, False, None)
    for _ in range(3):
        again = _call(x, False, None)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_empty_batches():
    z = lambda *s: torch.zeros(*s, device="cuda", requires_grad=True)
    q, k, v, h0 = z(0, 2, 8), z(0, 2, 8), z(0, 2, 4), torch.randn(3, 2, 8, 4, device="cuda", requires_grad=True)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    for g in (z(2), z(0, 2)):
        o, state = npa.varlen_linear_attention(q, k, v, cu, g, initial_state=h0, return_state=True)
        assert o.shape == (0, 2, 4) and torch.equal(state, h0)
        ds = torch.randn_like(h0)
        grads = torch.autograd.grad([o, state], [q, k, v, g, h0], [torch.zeros_like(o), ds])
        assert [t.shape for t in grads] == [t.shape for t in (q, k, v, g, h0)] and torch.equal(grads[4], ds) and not bool(grads[3].any())
        assert torch.equal(npa.varlen_linear_attention(q, k, v, cu, g, return_state=True)[1], torch.zeros_like(h0))
    o, state = npa.varlen_linear_attention(z(5, 1, 8), z(5, 1, 8), z(5, 1, 4), cu[:1], z(1), return_state=True)
    assert state.shape == (0, 1, 8, 4) and not bool(o.any())


def test_offsets_beyond_four_gib():
    """Rows that begin beyond 4 GiB of a wide tensor: the last sequence is what it is alone."""
    T, H, d = 140000, 2, 64
    wide = torch.empty(T, 16400, dtype=BF16, device="cuda")                       # 4.6 GB
    g = torch.Generator("cuda").manual_seed(0)
    cut = T - 150
    view = lambda i: wide[:, i * H * d:(i + 1) * H * d].view(T, H, d)
    for i in range(4):
        view(i).normal_(generator=g)
    q, k, v, do = (view(i) for i in range(4))
    log_decay = torch.full((H,), -0.02, device="cuda")
    cu = torch.tensor([0, 17, cut, T], dtype=torch.int32).cuda()
    o, _, bounds = npa.varlen_linear_attention_fwd(q, k, v, cu, log_decay)
    grads = npa.varlen_linear_attention_bwd(q, k, v, do, cu, log_decay, bounds)
    c = lambda t: t[cut:].cpu()
    want = R.run(c(q), c(k), c(v), [0, 150], log_decay.cpu(), d ** -0.5, do=c(do))
    for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        R.assert_within(t[cut:], want[n], n)


# ---- single tokens ----------------------------------------------------------------------------------------------------------------------
def _step_ref(x, state, slots, scale):
    table, err, big = state.double().clone(), torch.zeros(state.shape, dtype=torch.float64), state.double().abs()
    q, k, v = (x[n].double() for n in ("q", "k", "v"))
    g = x["log_decay"].double().expand(q.shape[:2])
    o, bound = torch.zeros(v.shape, dtype=torch.float64), torch.zeros(v.shape, dtype=torch.float64)
    for b, s in enumerate(slots):
        if 0 <= s < table.shape[0]:
            a = torch.exp(g[b])[:, None, None]
            table[s] = a * table[s] + R.outer(k[b], v[b])
            big[s] = a * big[s] + R.outer(k[b], v[b]).abs()
            err[s] = a * err[s] + (R.STATE + 2 * R.U * g[b].abs()[:, None, None]) * big[s]
            o[b] = scale * (q[b][:, None, :] @ table[s])[:, 0]
            bound[b] = abs(scale) * (q[b].abs()[:, None, :] @ (err[s] + R.RESULT * big[s]))[:, 0]
    return (o, bound), (table, err)


@pytest.mark.parametrize("act,gdt,rate", [(F32, F32, "token"), (BF16, BF16, "head"), (BF16, F32, "token"), (F32, F32, "head")])
@pytest.mark.parametrize("B,H,K,V,N,slots", [
    (1, 1, 1, 1, 1, None), (1, 16, 64, 64, 8, [5]), (3, 2, 33, 65, 3, None), (5, 1, 128, 128, 9, [8, 0, 3, -1, 7]), (6, 3, 20, 91, 4, [2, 2, 0, 2, 0, 99]),
    (4, 2, 128, 16, 2, [-1, -7, 2, 5]), (300, 2, 8, 12, 500, "mixed"), (70, 4, 64, 128, 90, "mixed")])
def test_step(B, H, K, V, N, slots, act, gdt, rate):
    x = _inputs([B], H, K, V, act, gdt, rate, False, 8)
    g = torch.Generator().manual_seed(B)
    state = torch.randn(N, H, K, V, generator=g)
    if slots == "mixed":
        slots = torch.randint(-30, N + 30, (B,), generator=g).tolist()
    named = list(range(B)) if slots is None else slots
    want_o, want_table = _step_ref(x, state, named, K ** -0.5)
    args = [x[n].cuda() for n in ("q", "k", "v", "log_decay")]
    table, other = state.cuda(), torch.full(state.shape, -3.0, device="cuda")
    ids = None if slots is None else torch.tensor(slots, dtype=torch.int32).cuda()
    o2 = npa.linear_attention_step(*args, table, ids, out_state=other)
    assert torch.equal(table.cpu(), state)                      # the old states stay
    o = npa.linear_attention_step(*args, table, ids)
    R.assert_within(o, want_o, "o")
    R.assert_within(table, want_table, "state")
    assert torch.equal(o, o2)
    touched = sorted({s for s in named if 0 <= s < N})
    rest = [s for s in range(N) if s not in touched]
    assert torch.equal(other[touched], table[touched]) and bool((other[rest] == -3.0).all()) and torch.equal(table[rest].cpu(), state[rest])


def test_a_step_of_strided_rows_and_of_forgotten_states():
    x = _inputs([6], 3, 40, 24, BF16, F32, "token", False, 9)
    x["log_decay"][::2, 1] = -float("inf")
    state = torch.randn(6, 3, 40, 24)
    wide = torch.randn(6, 3 * (40 + 40 + 24) + 1).bfloat16().cuda()[:, 1:]
    views, at = [], 0
    for n, d in (("q", 40), ("k", 40), ("v", 24)):
        views.append(wide[:, at:at + 3 * d].view(6, 3, d).copy_(x[n].cuda()))
        at += 3 * d
    table = state.cuda()
    o = npa.linear_attention_step(*views, x["log_decay"].t().contiguous().t().cuda(), table)
    want_o, want_table = _step_ref(x, state, range(6), 40 ** -0.5)
    R.assert_within(o, want_o, "o")
    R.assert_within(table, want_table, "state")


def test_a_table_beyond_four_gib():
    N, H, d = 70000, 1, 128
    table = torch.zeros(N, H, d, d, device="cuda")              # 4.6 GB
    x = _inputs([2], H, d, d, BF16, F32, "head", False)
    state = torch.randn(2, H, d, d)
    slots = [N - 1, 40000]
    for s, t in zip(slots, state):
        table[s] = t.cuda()
    o = npa.linear_attention_step(*(x[n].cuda() for n in ("q", "k", "v", "log_decay")), table, torch.tensor(slots, dtype=torch.int32).cuda())
    want_o, want_table = _step_ref(x, state, range(2), d ** -0.5)
    R.assert_within(o, want_o, "o")
    R.assert_within(table[slots], want_table, "state")


def test_steps_continue_a_prompt():
    """A packed prompt of three sequences, then their next tokens one by one through a table of states, against the sequences run whole."""
    H, K, V, lens, more = 2, 40, 24, [50, 1, 130], 4
    g = torch.Generator().manual_seed(2)
    m = npa.VarlenLinearAttention(H).cuda()
    parts = [[torch.randn(n + more, H, d, generator=g) for d in (K, K, V)] + [torch.randn(n + more, H, generator=g)] for n in lens]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    cat = lambda i, f: torch.cat([f(p[i], n) for p, n in zip(parts, lens)]).cuda()
    with torch.no_grad():
        _, state = m(*(cat(i, lambda t, n: t[:n]) for i in range(3)), cu, cat(3, lambda t, n: t[:n]), return_state=True)
        table = torch.zeros(10, H, K, V, device="cuda")
        slots = torch.tensor([7, 0, 3], dtype=torch.int32).cuda()
        table[slots.long()] = state
        got = []
        for j in range(more):
            q, k, v, gates = (cat(i, lambda t, n: t[n + j:n + j + 1]) for i in range(4))
            got.append(m.step(q, k, v, table, slots, gates))
    for s, (n, p) in enumerate(zip(lens, parts)):
        log_decay = torch.nn.functional.logsigmoid(m.decay.detach().cpu() + p[3])
        value, bound = R.run(*p[:3], [0, n + more], log_decay, K ** -0.5)["o"]
        R.assert_within(torch.stack([o[s] for o in got]), (value[n:], bound[n:]), f"sequence {s}")


# ---- the framework's surfaces -----------------------------------------------------------------------------------------------------------
def test_padded_door_gives_each_sequence_its_packed_results():
    B, L, H, d = 4, 70, 2, 16
    lens = [70, 1, 33, 0]
    mask = torch.arange(L)[None] < torch.tensor(lens)[:, None]
    m = npa.VarlenLinearAttention(H).cuda()
    q, k, v = (torch.randn(B, L, H, d, device="cuda") for _ in range(3))
    gates = torch.randn(B, L, H, device="cuda")
    o = m.forward_padded(q, k, v, mask.cuda(), gates)
    assert o.shape == (B, L, H, d)
    for b, n in enumerate(lens):
        c = lambda t: t[b, :n].cpu()
        want = R.run(c(q), c(k), c(v), [0, n], torch.nn.functional.logsigmoid(m.decay.detach().cpu() + c(gates)), d ** -0.5)["o"]
        R.assert_within(o[b, :n], want, f"row {b}")


def test_frozen_inputs_and_missing_gradients():
    x = _inputs([60, 40], 2, 16, 12, F32, F32, "token", True)
    c = {n: t.cuda() for n, t in x.items()}
    args = c["q"], c["k"], c["v"], c["cu"]
    g = c["log_decay"].clone().requires_grad_()
    o, state = npa.varlen_linear_attention(*args, g, initial_state=c["initial"], return_state=True)
    (state * c["dstate"]).sum().backward()                      # no gradient reaches o
    want = R.run(x["q"], x["k"], x["v"], x["cu"], x["log_decay"], 0.25, x["initial"], do=torch.zeros_like(x["do"]), dstate=x["dstate"])
    R.assert_within(g.grad, want["dlog_decay"], "dlog_decay")
    v = c["v"].clone().requires_grad_()
    npa.varlen_linear_attention(c["q"], c["k"], v, c["cu"], c["log_decay"]).backward(c["do"])
    R.assert_within(v.grad, R.run(x["q"], x["k"], x["v"], x["cu"], x["log_decay"], 0.25, do=x["do"])["dv"], "dv")
    h = c["initial"].clone().requires_grad_()
    npa.varlen_linear_attention(*args, c["log_decay"], initial_state=h).backward(c["do"])
    R.assert_within(h.grad, R.run(x["q"], x["k"], x["v"], x["cu"], x["log_decay"], 0.25, x["initial"], do=x["do"])["dinitial"], "dinitial")


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("K,V", [(24, 40), (64, 128), (128, 64), (128, 128), (91, 91)])
@pytest.mark.parametrize("lens", [[150, 0, 70, 1], [700]])
def test_each_set_of_gradients(lens, K, V, act):
    """Frozen log decays and initial states each take kernels of their own."""
    x = _inputs(lens, 2, K, V, act, F32, "head", True, 11)
    want = R.run(x["q"], x["k"], x["v"], x["cu"], x["log_decay"], K ** -0.5, x["initial"], do=x["do"], dstate=x["dstate"])
    c = {n: t.cuda() for n, t in x.items()}
    _, state, bounds = npa.varlen_linear_attention_fwd(c["q"], c["k"], c["v"], c["cu"], c["log_decay"], initial_state=c["initial"], want_state=True)
    for g, h in ((False, False), (False, True), (True, False), (True, True)):
        got = npa.varlen_linear_attention_bwd(c["q"], c["k"], c["v"], c["do"], c["cu"], c["log_decay"], bounds, initial_state=c["initial"], state=state,
                                              dstate=c["dstate"], want_dlog_decay=g, want_dinitial=h)
        assert (got[3] is None) == (not g) and (got[4] is None) == (not h)
        for n, t in zip(("dq", "dk", "dv", "dlog_decay", "dinitial"), got):
            if t is not None:
                R.assert_within(t, want[n], (n, g, h))


@pytest.mark.parametrize("act", [F32, BF16])
def test_rows_shorter_than_a_load_and_just_one(act):
    for K, V in ((4, 4), (3, 8), (8, 1), (1, 9), (7, 7)):
        _run_and_check(_inputs([200, 3], 2, K, V, act, F32, "token", True, 12), False)


def test_other_layouts_of_a_call():
    """One row for all tokens, a decay expanded over the tokens, every second entry of a table of boundaries, channels that are one element of a row, many heads: what the
    same numbers side by side give, bit for bit."""
    x = {n: t.cuda() for n, t in _inputs([70, 60], 2, 16, 24, F32, F32, "head", True, 13).items()}
    T, cu = 130, x["cu"]
    one = x["q"][:1].expand(T, 2, 16)
    rates = x["log_decay"].expand(T, 2)
    wide_cu = torch.stack([cu, cu], 1).flatten()[::2]
    a = npa.varlen_linear_attention(one, x["k"], x["v"], wide_cu, rates)
    assert torch.equal(a, npa.varlen_linear_attention(one.contiguous(), x["k"], x["v"], cu, rates.contiguous()))
    assert torch.equal(a, npa.varlen_linear_attention(one, x["k"], x["v"], cu, x["log_decay"]))
    g = x["log_decay"].clone().requires_grad_()
    by_row = torch.autograd.grad(npa.varlen_linear_attention(x["q"], x["k"], x["v"], cu, g.expand(T, 2)), [g], x["do"])[0]
    by_head = torch.autograd.grad(npa.varlen_linear_attention(x["q"], x["k"], x["v"], cu, g), [g], x["do"])[0]
    want = R.run(*(x[n].cpu() for n in ("q", "k", "v")), cu.cpu(), g.detach().cpu(), 0.25, do=x["do"].cpu())["dlog_decay"]
    for got in (by_row, by_head):                      # (autograd's sum over the rows adds T roundings of what the rows' gradients are)
        R.assert_within(got, (want[0], want[1] + 2 * T * 2.0 ** -24 * want[0].abs()), "dlog_decay", False)
    column = torch.randn(T, 2, 7, device="cuda")[:, :, 3:4]
    assert torch.equal(npa.varlen_linear_attention(column, column, x["v"], cu, g), npa.varlen_linear_attention(column.contiguous(), column.contiguous(), x["v"], cu, g))
    with torch.inference_mode():
        q = torch.randn(3, 5000, 8, device="cuda")
        many = npa.varlen_linear_attention(q, q, q, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.zeros(5000, device="cuda"))
        few = npa.varlen_linear_attention(q[:, 4990:], q[:, 4990:], q[:, 4990:], torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.zeros(10, device="cuda"))
        assert torch.equal(many[:, 4990:], few)


@pytest.mark.parametrize("act,gdt", [(BF16, F32), (F32, F32), (BF16, BF16)])
def test_the_function_is_the_node(act, gdt):
    x = {n: t.cuda() for n, t in _inputs([90, 300], 2, 40, 64, act, gdt, "token", True).items()}
    results = []
    for call in (lambda *a: npa.varlen_linear_attention(*a[:5], initial_state=a[5], return_state=True),
                 lambda *a: npa.VarlenLinearAttentionFunction.apply(*a, None, False, True)):
        leaves = [x[n].clone().requires_grad_() for n in NAMES]
        out = call(leaves[0], leaves[1], leaves[2], x["cu"], leaves[3], leaves[4])
        results.append(list(out) + list(torch.autograd.grad(out, leaves, [x["do"], x["dstate"]])))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_custom_ops_pass_opcheck_and_compile_without_graph_breaks():
    x = {n: t.cuda() for n, t in _inputs([60, 400], 2, 16, 12, F32, F32, "token", True).items()}
    leaves = [x[n].requires_grad_() for n in NAMES]
    q, k, v, g, h0 = leaves
    for want_state in (True, False):
        torch.library.opcheck(npa.varlen_linear_attention_fwd_op, (q, k, v, x["cu"], g, h0, None, False, want_state),
                              test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))

    def f(q, k, v, g, h0):
        o, s = npa.varlen_linear_attention(q * 1.0, k, v, x["cu"], g, initial_state=h0, return_state=True)
        return o * 2.0, s
    eager = f(*leaves)
    g1 = torch.autograd.grad(eager, leaves, [x["do"], x["dstate"]])
    got = torch.compile(f, dynamic=False, fullgraph=True, backend="aot_eager")(*leaves)
    g2 = torch.autograd.grad(got, leaves, [x["do"], x["dstate"]])
    assert all(torch.equal(a, b) for a, b in zip(list(eager) + list(g1), list(got) + list(g2)))


def test_side_stream_and_graph_replay():
    x = {n: t.cuda() for n, t in _inputs([300, 0, 400], 2, 64, 40, BF16, F32, "head", True).items()}
    leaves = [x[n].clone().requires_grad_() for n in NAMES]

    def step():
        o, s = npa.varlen_linear_attention(*leaves[:3], x["cu"], leaves[3], initial_state=leaves[4], return_state=True)
        grads = torch.autograd.grad([o, s], leaves, [x["do"], x["dstate"]])
        return [o.detach(), s.detach()] + list(grads)          # (no eager graph of the leaves may live while the step is captured)
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
            leaves[0].copy_(x["q"] * (n + 1))
            leaves[4].copy_(x["initial"] * (1 - n))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, got)), n


def test_a_captured_step_goes_on():
    x = {n: None if t is None else t.cuda() for n, t in _inputs([4], 2, 32, 48, BF16, BF16, "token", False).items()}
    first = torch.randn(9, 2, 32, 48, device="cuda")
    slots = torch.tensor([8, 0, -1, 0], dtype=torch.int32).cuda()
    args = [x[n] for n in ("q", "k", "v", "log_decay")]
    table, mine = first.clone(), first.clone()
    npa.linear_attention_step(*args, table.clone(), slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = npa.linear_attention_step(*args, table, slots)
    table.copy_(first)
    for n in range(3):
        args[2].normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = npa.linear_attention_step(*args, mine, slots)
        assert torch.equal(o, want) and torch.equal(table, mine), n
