"""The gated linear recurrence in 64 bits, one row after the other, with the rounding errors that an fp32 evaluation may leave on each result."""
import torch

# Rounding of fp32, relative: U for an addition or product; hardware exp2, reciprocal and roots are off by an ulp, 2 U.
#   sigmoid(v)         (2 |v| + 5) U: the exponent v * log2(e) is rounded twice (constant, product), then exp2, 1 + e, 1 / (1 + e)
#   z                  + 6 U for softplus (exp, log1p), scale and the two products
#   u = 1 - e^-z       + 12 U: its series, or exp2 and the difference, which is at least 0.22
#   a = 1 - u          u's error, absolute, and a rounding of a number below 1
#   b = beta si x      u's (halved by the root, its root 2 U), si's and two products
# Where z is below 1e-37, beta is 0 instead of at most 5e-19: FLOOR covers it for operands of a few units.
U = 2.0 ** -24
FLOOR = 1e-17
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}     # half a step, relative


def sequences(cu, T):
    """(first row, end, number or None) of every run of rows: those of cu and, around them, the rows outside [cu[0], cu[S])."""
    cu = [int(v) for v in cu]
    out = [(0, cu[0], None)] + [(a, b, i) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:]))] + [(cu[-1], T, None)]
    return [s for s in out if s[1] > s[0]]


def coefficients(x, gates, decay, scale):
    C = x.shape[1]
    x, r, i, lam = x.double(), gates[:, :C].double(), gates[:, C:].double(), decay.double()
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    sp = torch.where(lam > 30, lam, torch.log1p(torch.exp(lam.clamp(max=30))))
    z = scale * sp * sr
    u = -torch.expm1(-z)
    beta = torch.sqrt(u * (2 - u))
    eu = (2 * r.abs() + 24) * U                  # relative errors of u (and z), and of beta si
    eb = eu + (2 * i.abs() + 11) * U
    return dict(x=x, sr=sr, si=si, sp=sp, lam=lam, z=z, a=1 - u, beta=beta, b=beta * si * x, eu=eu, eb=eb, da=eu * u + 2 * U)


def forward(x, gates, cu, decay, scale=8.0, initial=None, reverse=False):
    """y, state, and bounds of what fp32 arithmetic leaves on h (before y is rounded)."""
    k = coefficients(x, gates, decay, scale)
    T, C = x.shape
    S = len(cu) - 1
    h = torch.zeros(T, C, dtype=torch.float64)
    before, big, err = torch.zeros_like(h), torch.zeros_like(h), torch.zeros_like(h)     # h_{t-1}, scan of |b|, error
    state = torch.zeros(S, C, dtype=torch.float64) if initial is None else initial.double().clone()
    for lo, hi, s in sequences(cu, T):
        now = state[s].clone() if s is not None else torch.zeros(C, dtype=torch.float64)
        m, e = now.abs(), torch.zeros_like(now)
        for t in range(hi - 1, lo - 1, -1) if reverse else range(lo, hi):
            before[t] = now
            now = k["a"][t] * now + k["b"][t]
            e = k["a"][t] * e + k["da"][t] * m + k["eb"][t] * k["b"][t].abs()
            m = k["a"][t] * m + k["b"][t].abs()
            e = e + 3 * U * m                    # a h + b, by way of h + P carry
            h[t], big[t], err[t] = now, m, e
        if s is not None:
            state[s] = now
    k.update(h=h, before=before, big=big, err=err)
    return h, state, k


def backward(dy, cu, k, scale=8.0, dstate=None, reverse=False):
    """dx, dgates, ddecay, dinitial with a bound of fp32's error on each."""
    T, C = dy.shape
    S = len(cu) - 1
    dy = dy.double()
    g, big, err = torch.zeros_like(dy), torch.zeros_like(dy), torch.zeros_like(dy)
    eh = torch.zeros_like(dy)                                                             # error and size of h_{t-1}
    mh = torch.zeros_like(dy)
    dinitial = torch.zeros(S, C, dtype=torch.float64) if dstate is None else dstate.double().clone()
    einitial = torch.zeros_like(dinitial)
    for lo, hi, s in sequences(cu, T):
        back = dinitial[s].clone() if s is not None else torch.zeros(C, dtype=torch.float64)
        m, e = back.abs(), torch.zeros_like(back)
        rows = list(range(lo, hi)) if reverse else list(range(hi - 1, lo - 1, -1))
        for n, t in enumerate(rows):
            g[t] = dy[t] + back
            big[t] = m + dy[t].abs()
            err[t] = e + 3 * U * big[t]
            back, m, e = k["a"][t] * g[t], k["a"][t] * big[t], k["a"][t] * err[t] + (k["da"][t] + U) * big[t]
            if n + 1 < len(rows):
                eh[t], mh[t] = k["err"][rows[n + 1]], k["big"][rows[n + 1]]
            else:
                mh[t] = k["before"][t].abs()
        if s is not None:
            dinitial[s], einitial[s] = back, e
    a, b, z, beta2 = k["a"], k["b"], k["z"], k["beta"] ** 2
    # d log a = g (a h_{t-1} - b a^2 / beta^2); where 1 - a^2 is nothing, neither is z / beta^2 * b
    over = torch.where(beta2 > 0, z * b.abs() / beta2.clamp(min=1e-300), torch.zeros_like(b))
    inner = over * torch.sign(b) * a * a - z * a * k["before"]
    m = g * inner
    inner_big = over * a * a + z * a * mh
    einner = z * a * eh + (2 * k["eu"] + k["eb"] + 12 * U) * inner_big + k["da"] * (2 * over * a + z * mh)
    em = err * inner_big + big * einner + U * big * inner_big
    ratio = torch.sigmoid(k["lam"]) / k["sp"]
    p1, p2 = k["beta"] * k["si"], b * (1 - k["si"])
    return {"dx": (g * p1, (err + (k["eb"] + 2 * U) * big) * p1),
            # 1 - sigmoid cancels where the gate is open: off by an ulp of 1
            "dr": (m * (1 - k["sr"]), em * (1 - k["sr"]) + 8 * U * m.abs()),
            "di": (g * p2, (err + (k["eb"] + 2 * U) * big) * p2.abs() + 8 * U * (g * b).abs()),
            # a wave adds up 16 rows in fp32 (15 roundings) and a chunk its 4 waves (3), the chunks are added up in fp64; sigmoid(decay) / softplus(decay) is
            # an exponential and a logarithm of 2 U each, 1 + e twice, a product and a quotient of 2 U, and a product with the sum: 10; 15 + 3 + 10 = 28
            "ddecay": (m.sum(0) * ratio, (em.sum(0) + 28 * U * (big * inner_big).sum(0)) * ratio),
            "dinitial": (dinitial, einitial + U * dinitial.abs())}


def assert_within(got, want, bound, what):
    """|got - want| within the fp32 bound and half a step of got's type."""
    got_d, want = got.detach().cpu().double(), want.double()
    assert got_d.shape == want.shape, (what, got_d.shape, want.shape)
    assert torch.isfinite(got_d).all(), f"{what}: non-finite values"
    room = HALF[got.dtype] * (want.abs() + bound) + bound + FLOOR
    worst = ((got_d - want).abs() / room)
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{what}: {float(worst.max()):.2f} of the bound at {int(worst.argmax())}"
