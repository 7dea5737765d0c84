"""Infinite values: what is infinite by the definition is infinite in the kernels' results, with its sign, and no NaN."""
import pytest
import torch

import nanoplm_amd as npa
from tests import recurrence_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _same_where_endless(got, want, what):
    """got has want's infinities and NaNs, and is finite where want is."""
    got = got.detach().cpu().double()
    for name, f in (("nan", torch.isnan), ("+inf", lambda t: t == float("inf")), ("-inf", lambda t: t == float("-inf"))):
        off = f(got) != f(want)
        assert not bool(off.any()), f"{what}: {name} differs in {int(off.sum())} places, first {off.nonzero()[0].tolist()}"


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("C", [6, 70])
@pytest.mark.parametrize("lens", [[30], [120], [700, 1300], [9000], [64] * 20 + [5000, 3]])
def test_an_infinite_state_stays_infinite(lens, C, act, reverse):
    """Decays from e^-0.01 to e^-12 a row: after some rows next to nothing is left of a state, and the product of the decays is 0 in fp32. (All of them are
    above 0 in 64 bits, so that an infinite state is infinite to the end of its sequence.)"""
    T, S = sum(lens), len(lens)
    g = torch.Generator().manual_seed(T + C)
    n = lambda *s: torch.randn(*s, generator=g)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    x, gates, dy = n(T, C).to(act), n(T, 2 * C).clamp(-2, 2).to(act), n(T, C).to(act)
    decay = torch.linspace(-6, 1.5, C)                         # (8 softplus(1.5) = 13.6, times a sigmoid of at most 0.89)
    h0, ds = n(S, C), n(S, C)
    inf = float("inf")
    x[T // 3, 0::3], x[T // 2, 1::6] = inf, -inf               # a third of the channels stays finite
    h0[0, 2::6], dy[T // 2, 0::2], ds[S - 1, 1::4] = -inf, inf, -inf
    h, last, k = R.forward(x, gates, cu, decay, 8.0, h0, reverse)
    assert int(h.isinf().sum()) > T // 8 and not bool(h.isnan().any()) and int(h.isfinite().sum()) > T
    c = lambda t: t.cuda()
    y, state, carries = npa.varlen_recurrence_fwd(c(x), c(gates), c(cu), c(decay), initial_state=c(h0), reverse=reverse, want_state=True, want_carries=True)
    _same_where_endless(y, h, "y")
    _same_where_endless(state, last, "state")
    dx, _, _, dinitial = npa.varlen_recurrence_bwd(c(x), c(gates), c(dy), c(cu), c(decay), carries, initial_state=c(h0), dstate=c(ds), reverse=reverse,
                                                   want_dinitial=True)
    want = R.backward(dy, cu, k, 8.0, ds, reverse)
    _same_where_endless(dx, want["dx"][0], "dx")
    _same_where_endless(dinitial, want["dinitial"][0], "dinitial")


def _norm_inputs(T, C, act, st, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, d=F32: torch.randn(*s, generator=g).to(d)
    return n(T, C, d=act), n(T, C, d=st), n(T, C, d=act), n(C), n(C), n(C), n(C), n(T, C, d=st), n(T, C, d=act)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act,st", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("T,C", [(1, 7), (1, 64), (1, 200), (1, 600), (1, 1024), (3, 130), (33, 64), (5, 1001), (1, 4100)])
def test_an_infinite_gradient_of_the_last_row_is_the_parameters(T, C, act, st, norm):
    """The last row comes alone to a block that has room for more rows: what the room holds adds nothing, whatever the row's gradients are."""
    u, x, gate, pw, pb, sc, qw, ds, dy = _norm_inputs(T, C, act, st)
    inf = float("inf")
    c = lambda t: t.cuda()
    fwd = lambda: npa.residual_norm_fwd(c(u), c(x), c(gate), c(pw), c(pb), c(sc), c(qw), norm=norm, want_stats=True)
    # dstream infinite in one channel: so are that channel's sums of dstream * v (scale) and, with its sign, no other channel's
    at = C // 2
    ds[T - 1, at] = inf
    out = npa.residual_norm_bwd(c(u), c(x), c(gate), c(pw), c(pb), c(sc), c(qw), fwd()[2], c(ds), c(dy), norm=norm, pre_bias=True)
    dscale, dpre_weight, dpre_bias = out[5], out[6], out[7]
    assert bool(torch.isinf(dscale[at])) and bool(torch.isfinite(dscale[torch.arange(C) != at]).all())
    assert bool(torch.isfinite(dpre_weight).all() and torch.isfinite(dpre_bias).all())
    # dnormed infinite in one channel: that channel's pre_bias and pre_weight
    ds[T - 1, at], dy[T - 1, at] = 0.0, -inf
    out = npa.residual_norm_bwd(c(u), c(x), c(gate), c(pw), c(pb), c(sc), c(qw), fwd()[2], c(ds), c(dy), norm=norm, pre_bias=True)
    assert float(out[7][at]) == -inf and bool(torch.isinf(out[6][at])) and bool(torch.isfinite(out[7][torch.arange(C) != at]).all())
    # without norms or gate, of a row that is itself infinite: dscale = dstream * u
    dy[T - 1, at], ds[T - 1, at] = 0.0, 0.5
    u[T - 1, at] = inf
    stats = npa.residual_norm_fwd(c(u), c(x), None, None, None, c(sc), None, want_stats=True)[2]
    out = npa.residual_norm_bwd(c(u), c(x), None, None, None, c(sc), None, stats, c(ds), None)
    assert float(out[5][at]) == inf and bool(torch.isfinite(out[5][torch.arange(C) != at]).all())
