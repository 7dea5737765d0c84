"""The residual norm in 64 bits with first-order bounds of what an fp32 evaluation may be off, each result beside its bound."""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}     # half a step, relative
SUM = 32 * U          # of a sum over a row: 16 channels a lane one after the other, at most 10 exchanges (4 + 16 waves' sums), the division


def _norm(a, ea, kind, eps):
    """(n, bound of n, rstd, its relative bound) of rows a that are off by ea."""
    mean = a.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(a[:, :1])
    em = (ea + SUM * a.abs()).mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(mean)
    d = a - mean
    ed = ea + em + U * d.abs()
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    rel = ((d.abs() * ed).mean(1, keepdim=True) + 0.5 * SUM * var) * rstd ** 2 + 4 * U
    n = d * rstd
    return n, n.abs() * (rel + 2 * U) + rstd * ed, rstd, rel


def _norm_back(d, ed, n, en, rstd, rel, kind):
    """rstd (d - mean(d) - n mean(d n)) and its bound."""
    m0 = d.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(d[:, :1])
    e0 = (ed + SUM * d.abs()).mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(m0)
    m1 = (d * n).mean(1, keepdim=True)
    e1 = (ed * n.abs() + d.abs() * en + SUM * (d * n).abs()).mean(1, keepdim=True)
    out = rstd * (d - m0 - n * m1)
    size = rstd * (d.abs() + m0.abs() + (n * m1).abs())
    return out, rstd * (ed + e0 + n.abs() * e1 + en * m1.abs()) + size * (rel + 4 * U)


def run(u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, eps, dstream=None, dnormed=None):
    """{name: (value, bound)} of the outputs and, with the outputs' gradients, of every gradient."""
    f = lambda t: None if t is None else t.detach().cpu().double()
    u, x, g, pw, pb, sc, qw, qb, ds, dy = map(f, (u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, dstream, dnormed))
    one, zero = torch.ones(u.shape[1], dtype=torch.float64), torch.zeros(u.shape[1], dtype=torch.float64)
    z = torch.zeros_like(u)
    n, en, pr, prel = (u, z, None, None) if pw is None else _norm(u, z, norm, eps)
    w, b, s = (one if pw is None else pw), (zero if pb is None else pb), (one if sc is None else sc)
    a = n * w + b
    ea = z if pw is None else en * w.abs() + 2 * U * ((n * w).abs() + b.abs())
    if g is None:
        v, ev = a, ea
    else:
        sg = torch.sigmoid(g)
        silu, es = g * sg, (2 * g.abs() + 6) * U                      # es: relative, of a sigmoid (exponent rounded twice, exp2, 1 + e, reciprocal)
        v = a * silu
        ev = ea * silu.abs() + v.abs() * (es + 2 * U)
    X = x + s * v
    eX = s.abs() * ev + 2 * U * ((s * v).abs() + x.abs())
    out = {"stream": (X, eX)}
    if qw is not None:
        q = zero if qb is None else qb
        N, eN, qr, qrel = _norm(X, eX, norm, eps)
        out["normed"] = (N * qw + q, eN * qw.abs() + 2 * U * ((N * qw).abs() + q.abs()))
    if ds is None and dy is None:
        return out
    D, eD = (z, z) if ds is None else (ds, z)
    total = lambda t, e: (t.sum(0), (e + 24 * U * t.abs()).sum(0))   # a few rows a lane, the rows of a block, then fp64
    if qw is not None and dy is not None:
        out["dpre_weight"], out["dpre_bias"] = total(dy * N, dy.abs() * eN), total(dy, z)
        back, eb = _norm_back(dy * qw, U * (dy * qw).abs(), N, eN, qr, qrel, norm)
        D, eD = D + back, eD + eb + U * (D.abs() + back.abs())
    elif qw is not None:
        out["dpre_weight"] = out["dpre_bias"] = (zero, zero)
    out["dresidual"] = (D, eD)
    out["dscale"] = total(D * v, eD * v.abs() + D.abs() * ev)
    d, ed = D * s, eD * s.abs() + U * (D * s).abs()
    if g is not None:
        slope = sg * (1 + g * (1 - sg))
        eslope = slope.abs() * (es + 3 * U) + sg * (g.abs() * (sg * es + U) + 2 * U * (1 + (g * (1 - sg)).abs()))
        out["dgate"] = (d * a * slope, (ed * a.abs() + d.abs() * (ea + 2 * U * a.abs())) * slope.abs() + (d * a).abs() * (eslope + 2 * U * slope.abs()))
        d, ed = d * silu, ed * silu.abs() + (d * silu).abs() * (es + 2 * U)
    if pw is not None:
        out["dpost_weight"], out["dpost_bias"] = total(d * n, ed * n.abs() + d.abs() * en), total(d, ed)
        d, ed = _norm_back(d * w, ed * w.abs() + U * (d * w).abs(), n, en, pr, prel, norm)
    out["du"] = (d, ed)
    return out


def assert_within(got, want, what):
    value, bound = want
    got_d = got.detach().cpu().double()
    assert got_d.shape == value.shape, (what, got_d.shape, value.shape)
    assert torch.isfinite(got_d).all(), f"{what}: non-finite values"
    room = HALF[got.dtype] * (value.abs() + bound) + 1.1 * bound + 1e-30          # (second-order terms)
    worst = (got_d - value).abs() / room
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{what}: {float(worst.max()):.2f} of the bound at {int(worst.argmax())}"
