"""Linear attention in 64 bits, one row after the other, with the rounding errors that the kernels' arithmetic may leave on each result."""
import torch

U = 2.0 ** -24                                                    # half a step of fp32, relative: one operation
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}     # of a result's type
# Errors of fp32 arithmetic, in U of the sum of absolute terms:
#   a row adds to the state a product with its weight (the weight's exp2 2, times scale 1, product 1) and a sum (1); what was there is multiplied by the chunk's
#   decay at most once a row (product 1, exp2 2): 8 a row on the state's absolute sum; an exponent b log 2 is rounded once more where it is
#   made fp32, |b| U of the weight, and a hi + lo difference likewise: 2 |log a| a row
#   a result is a sum over at most 64 rows of its chunk and the state's rows or columns, the sums of products over as many channels inside: one rounding a
#   term and another for the order in which the matrix instruction aligns them: 2 (64 + 128 + 128) and 8 for weights and scale
STATE, RESULT = 8 * U, (2 * 320 + 8) * U
FLOOR = 1e-30


def sequences(cu, T):
    """(first row, end, number or None) of every run of rows: those of cu and, around them, the rows outside [cu[0], cu[S])."""
    cu = [int(v) for v in cu]
    out = [(0, cu[0], None)] + [(a, b, i) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:]))] + [(cu[-1], T, None)]
    return [s for s in out if s[1] > s[0]]


def outer(a, b):
    return a[:, :, None] * b[:, None, :]


def run(q, k, v, cu, log_decay, scale, initial=None, reverse=False, do=None, dstate=None, fine=None):
    """{name: (value, bound)} of o and state and, with do, of every gradient. ``fine``: whether the log decays' gradient is fp32 (log_decay's dtype).

    Operands in bf16: each of the products in a chunk has one that was rounded (a score), each product with the state two (what was added to it, the state): 2 steps of
    2^-8 of the absolute terms. Where results are fp32, 24 bits of these operands are kept (a step of U each, within STATE and RESULT); for log decays in bf16 16 bits:
    2 steps of 2^-16."""
    dev, half = q.device, 0.0 if q.dtype == torch.float32 else 2 * 2.0 ** -8
    fine = log_decay.dtype == torch.float32 if fine is None else fine
    keep = 0.0 if fine or q.dtype == torch.float32 else 2 * 2.0 ** -16
    d = lambda t: None if t is None else t.detach().double()
    q, k, v, g, initial, do, dstate = map(d, (q, k, v, log_decay, initial, do, dstate))
    T, H, K = q.shape
    V, S, one = v.shape[2], len(cu) - 1, g.dim() == 1
    g = g.expand(T, H)
    a = torch.exp(g)
    grow = STATE + 2 * U * g.abs().clamp(max=200.0)
    z = lambda *n: torch.zeros(*n, dtype=torch.float64, device=dev)
    aq, ak, av = q.abs() * abs(scale), k.abs(), v.abs()
    o, eo, dq, edq = z(T, H, V), z(T, H, V), z(T, H, K), z(T, H, K)
    state = z(S, H, K, V) if initial is None else initial.clone()
    estate, mstate = z(S, H, K, V), state.abs()
    reads, ereads = z(T, H), z(T, H)                              # q . dq and its error, for the log decays
    at = lambda row, m: (row[:, None, :] @ m)[:, 0, :]            # row vectors times matrices, and matrices times columns
    by = lambda m, col: (m @ col[:, :, None])[:, :, 0]
    if do is not None:
        ado = do.abs()
        cross = z(T, H)                                           # errors of <S, dS> at a row
        kept = [None] * T
    for lo, hi, s in sequences(cu, T):
        h, m, e = (state[s], mstate[s], estate[s]) if s is not None else (z(H, K, V), z(H, K, V), z(H, K, V))
        for t in range(hi - 1, lo - 1, -1) if reverse else range(lo, hi):
            x = a[t][:, None, None]
            h = x * h + outer(k[t], v[t])
            m = x * m + outer(ak[t], av[t])
            e = x * e + grow[t][:, None, None] * m
            o[t], eo[t] = scale * at(q[t], h), at(aq[t], e) + (RESULT + half) * at(aq[t], m)
            if do is not None:
                dq[t], edq[t] = scale * by(h, do[t]), abs(scale) * (by(e, ado[t]) + (RESULT + half) * by(m, ado[t]))
                reads[t] = (q[t] * dq[t]).sum(1)
                ereads[t] = (q[t].abs() * abs(scale) * (by(e, ado[t]) + (RESULT + keep) * by(m, ado[t]))).sum(1)
                if T * H * K * V <= 1 << 25:
                    kept[t] = (m, e)
        if s is not None:
            state[s], mstate[s], estate[s] = h, m, e
    out = {"o": (o, eo), "state": (state, estate + U * state.abs())}
    if do is None:
        return out
    dk, edk, dv, edv = z(T, H, K), z(T, H, K), z(T, H, V), z(T, H, V)
    dlog, elog = z(T, H), z(T, H)
    first = z(S, H, K, V) if dstate is None else dstate.clone()
    efirst = z(S, H, K, V)
    for lo, hi, s in sequences(cu, T):
        G, m, e = (first[s], first[s].abs(), efirst[s]) if s is not None else (z(H, K, V), z(H, K, V), z(H, K, V))
        behind = (state[s] * G).sum((1, 2)) if s is not None else z(H)
        ebehind = (estate[s] * m + (2 * 128 * U) * mstate[s] * m).sum((1, 2)) if s is not None else z(H)
        worst = ebehind.clone()
        for t in range(lo, hi) if reverse else range(hi - 1, lo - 1, -1):
            G = G + scale * outer(q[t], do[t])
            m = m + outer(aq[t], ado[t])
            e = e + grow[t][:, None, None] * m
            dk[t], edk[t] = by(G, v[t]), by(e, av[t]) + (RESULT + half) * by(m, av[t])
            dv[t], edv[t] = at(k[t], G), at(ak[t], e) + (RESULT + half) * at(ak[t], m)
            given = (k[t] * dk[t]).sum(1)
            behind = behind + reads[t] - given
            # what a sum over later rows is off by, and the largest that a sum begun again at a boundary between here and the end may start with
            ebehind = ebehind + ereads[t] + (ak[t] * (by(e, av[t]) + (RESULT + keep) * by(m, av[t]))).sum(1)
            if kept[t] is not None:
                sm, se = kept[t]
                worst = torch.maximum(worst, (se * m + sm * e + (2 * 128 * U + keep) * sm * m).sum((1, 2)))
            dlog[t], elog[t] = behind, ebehind + worst
            x = a[t][:, None, None]
            G, m, e = x * G, x * m, x * e + grow[t][:, None, None] * (x * m)
        if s is not None:
            first[s], efirst[s] = G, e
    out.update(dq=(dq, edq), dk=(dk, edk), dv=(dv, edv), dinitial=(first, efirst + U * first.abs()),
               dlog_decay=(dlog.sum(0), elog.sum(0)) if one else (dlog, elog))
    return out


def assert_within(got, want, what, near=False):
    """|got - want| within the bound and half a step of got's type. ``near``: of bf16 results of independent operands of mean zero also the 2-norm: the errors of
    the operands and of the result, two or three of at most 2^-8 of every term and independent as the terms are, add up as the terms do: at most sqrt(3) 2^-8, below 2^-7."""
    value, bound = want
    got_d = got.detach().double().to(value.device)
    assert got_d.shape == value.shape, (what, got_d.shape, value.shape)
    assert torch.isfinite(got_d).all(), f"{what}: non-finite values"
    room = HALF[got.dtype] * (value.abs() + bound) + 1.1 * bound + FLOOR          # (second-order terms)
    worst = (got_d - value).abs() / room
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{what}: {float(worst.max()):.2f} of the bound at {int(worst.argmax())}"
    if near and got.dtype == torch.bfloat16 and got.numel() >= 4096:
        off = float((got_d - value).norm() / value.norm())
        assert off <= 2.0 ** -7, f"{what}: {off:.2e} in the 2-norm"
