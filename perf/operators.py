"""The recurrent block's operators over packed rows, as cases that can be timed: the gated linear recurrence, its single-token step, and the
residual norm that closes a block.

A case is one call of a public door of the library (``varlen_recurrence``, ``recurrence_step``, ``residual_norm``), alone (``train``
false: inference) or with the gradients of everything a training step needs (``train`` true). Sizes are those of the repository's
benchmark configurations, of the default widths of the model the operators sit in (hidden 768 and 1024, intermediate 2048) and generic
ragged ones.

Fields: ``op`` recurrence | step | norm; ``C`` channels; ``act`` / ``par`` dtypes of activations and parameters (bf16 | fp32).
Recurrence: ``T`` rows; ``mix`` the lengths of the packed sequences; ``decays`` slow (a channel forgets 0.1 % to 10 % a token where its gate
is open) or wide (anything from nothing to everything); ``states`` whether it starts from given states and returns the last ones; ``reverse``.
Step: ``B`` rows, one token each; ``N`` states in the table; ``padding`` whether some of the rows are padding.
Norm: ``T`` rows; ``stream`` dtype of the residual stream; ``norm`` layer | rms; ``gated``, ``post``, ``scaled``, ``pre``, ``biased`` which
parts it has; ``sliced`` whether u and the gate are halves of one wider tensor.

``own`` false computes the same with elementary operations in fp32 (fp64 for the long sums of parameters' gradients).
"""
import math
import types

import numpy as np
import torch

own = False

DEV = "cuda"
SCALE = 8.0
EPS = 1e-5
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}


def _recurrence(name, T, C, act, par, mix, train, decays="slow", states=False, reverse=False):
    return dict(name=name, op="recurrence", T=T, C=C, act=act, par=par, mix=mix, train=train, decays=decays, states=states, reverse=reverse)


def _step(name, B, C, N, act, par, padding):
    return dict(name=name, op="step", B=B, C=C, N=N, act=act, par=par, padding=padding)


def _norm(name, T, C, act, stream, par, norm, train, gated=True, post=True, scaled=True, pre=True, biased=False, sliced=False):
    return dict(name=name, op="norm", T=T, C=C, act=act, stream=stream, par=par, norm=norm, train=train, gated=gated, post=post, scaled=scaled,
                pre=pre, biased=biased, sliced=sliced)


def listed():
    return [
        # a training step of one small batch through a narrow layer, from the right, with states carried in and out: latency
        _recurrence("recurrence_train_small", 776, 64, "fp32", "fp32", "short", True, states=True, reverse=True),
        # the headline packed batch (131072 rows, hidden 1024), forward and backward
        _recurrence("recurrence_train_packed", 131072, 1024, "bf16", "bf16", "usual", True),
        # autocast's fp32 stream at hidden 768, many sequences of a few rows
        _recurrence("recurrence_train_fp32_stress", 32768, 768, "fp32", "fp32", "stress", True, decays="wide"),
        # one long sequence trained whole, an odd width (rows of partial cache lines), from the right
        _recurrence("recurrence_train_long", 20011, 1001, "bf16", "fp32", "one", True, states=True, reverse=True),
        # prefill of one very long sequence at the intermediate width, state handed on
        _recurrence("recurrence_prefill_long", 65536, 2048, "bf16", "bf16", "one", False, states=True),
        # one token of one sequence
        _step("step_single", 1, 1024, 8, "bf16", "bf16", False),
        # a serving batch at the intermediate width, some rows padding
        _step("step_batch", 250, 2048, 1024, "bf16", "fp32", True),
        # the end of a block for a few tokens: latency
        _norm("norm_tokens", 8, 2048, "bf16", "bf16", "bf16", "rms", False),
        # the end of a block in a training step of the headline batch
        _norm("norm_train_packed", 131072, 1024, "bf16", "bf16", "bf16", "layer", True),
        # the same under autocast: bf16 branch, fp32 stream and parameters with biases, hidden 768; u and gate halves of one projection
        _norm("norm_train_autocast", 50021, 768, "bf16", "fp32", "fp32", "layer", True, biased=True, sliced=True),
        # an odd width in fp32, no gate
        _norm("norm_train_odd", 5003, 1001, "fp32", "fp32", "fp32", "rms", True, gated=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    return rng.choice([64, 512, 768, 1000, 1024, 2048, rng.randrange(65, 2050), 8 * rng.randrange(8, 257)])


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "recurrence", "step", "norm", "norm"])
    act, par = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
    C = _width(rng)
    if op == "step":
        B = _log(rng, 1, 512)
        case = _step("", B, C, B + rng.randrange(1, 600), act, par, rng.random() < 0.5)
    else:
        most = 131072 * 1024 * 2 // (C * _BYTES[act])           # as many bytes as the headline batch
        train = rng.random() < 0.7
        if op == "recurrence":
            mix = rng.choice(["usual", "usual", "skewed", "stress", "short", "ragged", "one"])
            T = _log(rng, 1, min(most, 65536 if mix == "one" else 131072))
            case = _recurrence("", T, C, act, par, mix, train, rng.choice(["slow", "wide"]), rng.random() < 0.4, rng.random() < 0.4)
        else:
            stream = "fp32" if act == "fp32" or (par == "fp32" and rng.random() < 0.7) else "bf16"
            T = _log(rng, 1, min(most, 131072))
            case = _norm("", T, C, act, stream, par, rng.choice(["layer", "rms"]), train, rng.random() < 0.7, rng.random() < 0.7,
                         rng.random() < 0.6, rng.random() < 0.8, rng.random() < 0.3, rng.random() < 0.3)
    del case["name"]
    return case


def _lengths(mix, T, rs):
    if mix == "one":
        return [T]
    got, left = [], T
    while left > 0:
        if mix == "short":
            n = rs.randint(20, 129)
        elif mix == "usual":
            n = rs.randint(20, 513)
        elif mix == "skewed":
            n = int(min(max(round(math.exp(rs.randn() * 0.8 + 5.5)), 20), 1024))
        elif mix == "stress":
            n = rs.randint(1, 9) if rs.rand() < 0.6 else rs.randint(400, 513)
        elif mix == "ragged":                                    # anything from empty to a quarter of the rows
            n = int(math.exp(rs.rand() * math.log(T / 4 + 2))) - 1
        else:
            raise ValueError(mix)
        got.append(min(n, left))
        left -= got[-1]
    return got


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed * 7919 + 11)
    s = types.SimpleNamespace(case=case)
    C, act, par = case["C"], _DT[case["act"]], _DT[case["par"]]

    def normal(*shape, dtype=act, std=1.0, mean=0.0, grad=False):
        t = torch.randn(*shape, device=DEV, generator=g).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(grad)

    if case["op"] == "norm":
        T, train, st = case["T"], case["train"], _DT[case["stream"]]
        # a branch's output and its gate; the stream has grown over the layers below
        if case["sliced"]:
            s.wide = normal(T, 2 * C)
            s.u, s.gate = s.wide[:, :C], s.wide[:, C:]
            s.u.requires_grad_(train), s.gate.requires_grad_(train)
        else:
            s.u, s.gate = normal(T, C, grad=train), normal(T, C, grad=train)
        s.gate = s.gate if case["gated"] else None
        s.residual = normal(T, C, dtype=st, std=3.0, grad=train)
        has = lambda part, *a, **k: normal(C, *a, dtype=par, std=0.1, grad=train, **k) if part else None  # noqa: E731
        s.post_weight, s.post_bias = has(case["post"], mean=1.0), has(case["post"] and case["biased"])
        s.scale = has(case["scaled"], mean=0.3)
        s.pre_weight, s.pre_bias = has(case["pre"], mean=1.0), has(case["pre"] and case["biased"])
        s.dstream, s.dnormed = normal(T, C, dtype=st), (normal(T, C) if case["pre"] else None)
        return s
    train = case.get("train", False)
    if case.get("decays") == "wide":
        s.decay = normal(C, dtype=torch.float32, std=3.0)
    else:
        a = torch.rand(C, device=DEV, generator=g).mul_(0.099).add_(0.9)                   # what an open gate keeps
        s.decay = torch.log(torch.expm1(-torch.log(a) / SCALE))
    s.decay = s.decay.to(par).requires_grad_(train)
    rs = np.random.RandomState(seed % (1 << 32))
    if case["op"] == "step":
        B, N = case["B"], case["N"]
        s.x, s.gates = normal(B, C), normal(B, 2 * C)
        slots = rs.permutation(N)[:B]
        if case["padding"]:
            slots[rs.rand(B) < 0.1] = -1
        s.slots = torch.from_numpy(slots.astype(np.int32)).to(DEV)
        s.state = normal(N, C, dtype=torch.float32, std=0.5)
        s.out_state = s.state.clone()                            # (the old states stay until the token is accepted)
        return s
    T = case["T"]
    lengths = _lengths(case["mix"], T, rs)
    S = len(lengths)
    s.longest = max(lengths)
    s.cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).to(DEV)
    s.x, s.gates = normal(T, C, grad=train), normal(T, 2 * C, grad=train)
    s.initial = normal(S, C, dtype=torch.float32, std=0.5, grad=train) if case["states"] else None
    s.dy = normal(T, C) if train else None
    s.dstate = normal(S, C, dtype=torch.float32) if train and case["states"] else None
    return s


def run(s):
    return {"recurrence": _run_recurrence, "step": _run_step, "norm": _run_norm}[s.case["op"]](s)


def _named(names, values):
    return {n: v for n, v in zip(names, values) if v is not None}


# ---- the framework's calls ------------------------------------------------------------------------------------------------------------
def _grads(outs, douts, names, leaves):
    """Gradients of the outputs that there are, by name."""
    kept = [(n, t) for n, t in zip(names, leaves) if t is not None]
    pairs = [(o, d) for o, d in zip(outs, douts) if o is not None]
    return dict(zip([n for n, _ in kept], torch.autograd.grad([o for o, _ in pairs], [t for _, t in kept], [d for _, d in pairs])))


def _own_recurrence(s):
    import nanoplm_amd as npa
    out = npa.varlen_recurrence(s.x, s.gates, s.cu, s.decay, scale=SCALE, initial_state=s.initial, reverse=s.case["reverse"],
                                return_state=s.case["states"])
    y, state = out if s.case["states"] else (out, None)
    res = _named(("y", "state"), (y, state))
    if s.case["train"]:
        res.update(_grads((y, state), (s.dy, s.dstate), ("dx", "dgates", "ddecay", "dinitial"), (s.x, s.gates, s.decay, s.initial)))
    return res


def _own_step(s):
    import nanoplm_amd as npa
    y = npa.recurrence_step(s.x, s.gates, s.decay, s.state, s.slots, scale=SCALE, out_state=s.out_state)
    return {"y": y, "state": s.out_state}


def _own_norm(s):
    import nanoplm_amd as npa
    stream, normed = npa.residual_norm(s.u, s.residual, gate=s.gate, post_weight=s.post_weight, post_bias=s.post_bias, scale=s.scale,
                                       pre_weight=s.pre_weight, pre_bias=s.pre_bias, norm=s.case["norm"], eps=EPS)
    res = _named(("stream", "normed"), (stream, normed))
    if s.case["train"]:
        res.update(_grads((stream, normed), (s.dstream, s.dnormed),
                          ("du", "dgate", "dresidual", "dpost_weight", "dpost_bias", "dscale", "dpre_weight", "dpre_bias"),
                          (s.u, s.gate, s.residual, s.post_weight, s.post_bias, s.scale, s.pre_weight, s.pre_bias)))
    return res


# ---- the plain form of the recurrence ---------------------------------------------------------------------------------------------------
def _coefficients(x, gates, decay):
    """(a, b, beta^2, sigmoid(i), sigmoid(r), z) in fp32; 1 - a and 1 - a^2 without cancellation."""
    C = x.shape[1]
    sr, si = torch.sigmoid(gates[:, :C].float()), torch.sigmoid(gates[:, C:].float())
    z = SCALE * torch.nn.functional.softplus(decay.float()) * sr
    a, beta2 = torch.exp(-z), -torch.expm1(-2 * z)
    return a, torch.sqrt(beta2) * si * x.float(), beta2, si, sr, z


def _scan(a, b, longest):
    """h_t = a_t h_{t-1} + b_t down the rows, by doubling; a is zero where a sequence begins. Overwrites both."""
    k = 1
    while k < longest:
        nb = torch.addcmul(b[k:], a[k:], b[:-k])
        na = a[k:] * a[:-k]
        b[k:], a[k:] = nb, na
        k *= 2
    return b


def _first_rows(cu, S, T, reverse):
    """(first row, last row, whether it has any) of each sequence in the scan's order; empty ones point at a row that exists."""
    lo, hi = cu[:-1].long(), cu[1:].long() - 1
    some = hi >= lo
    lo, hi = lo.clamp(0, T - 1), hi.clamp(0, T - 1)
    return (hi, lo, some) if reverse else (lo, hi, some)


def _run_recurrence(s):
    if own:
        return _own_recurrence(s)
    case, reverse = s.case, s.case["reverse"]
    with torch.no_grad():
        T, S = case["T"], s.cu.numel() - 1
        first, last, some = _first_rows(s.cu, S, T, reverse)
        marks = lambda rows: torch.zeros(T, device=DEV, dtype=torch.int32).index_add_(0, rows, some.int())[:, None] > 0  # noqa: E731
        starts = marks(first)
        a, b, beta2, si, sr, z = _coefficients(s.x, s.gates, s.decay)
        flip = (lambda t: t.flip(0)) if reverse else (lambda t: t)  # noqa: E731
        h0 = torch.zeros(T, 1, device=DEV) if s.initial is None else torch.zeros_like(a).index_add_(0, first, s.initial * some[:, None])
        h = flip(_scan(flip(torch.where(starts, 0.0, a)).contiguous(), flip(torch.addcmul(b, a, h0)).contiguous(), s.longest))
        state = None if s.initial is None else torch.where(some[:, None], h[last], s.initial)
        res = _named(("y", "state"), (h.to(s.x.dtype), state))
        if not case["train"]:
            return res
        step = -1 if reverse else 1
        before = torch.where(starts, h0, h.roll(step, 0))                       # h_{t-1}
        g = s.dy.float()
        if s.dstate is not None:
            g = g.index_add(0, last, s.dstate * some[:, None])
        after = torch.where(marks(last), 0.0, a.roll(-step, 0))                        # a_{t+1}
        back = (lambda t: t) if reverse else (lambda t: t.flip(0))  # noqa: E731
        g = back(_scan(back(after).contiguous(), back(g).contiguous(), s.longest))
        beta = torch.sqrt(beta2)
        dlog = g * (a * before - b * a * a / beta2)
        m = -z * dlog
        decay = s.decay.float()
        ddecay = m.sum(0, dtype=torch.float64).float() * (torch.sigmoid(decay) / torch.nn.functional.softplus(decay))
        res["dx"] = (g * beta * si).to(s.x.dtype)
        res["dgates"] = torch.cat([m * (1 - sr), g * b * (1 - si)], 1).to(s.gates.dtype)
        res["ddecay"] = ddecay.to(s.decay.dtype)
        if s.initial is not None:
            res["dinitial"] = torch.where(some[:, None], a[first] * g[first], s.dstate)
        return res


def _run_step(s):
    if own:
        return _own_step(s)
    with torch.no_grad():
        a, b = _coefficients(s.x, s.gates, s.decay)[:2]
        real = (s.slots >= 0)[:, None]
        at = s.slots.long().clamp(min=0)
        h = torch.addcmul(b, a, s.state[at])
        # a padding row writes to a row behind the table
        table = torch.cat([s.state, s.state[:1]])
        table[torch.where(s.slots >= 0, at, s.state.shape[0])] = h
        s.out_state.copy_(table[:-1])
        return {"y": torch.where(real, h, 0.0).to(s.x.dtype), "state": s.out_state}


# ---- the plain form of the residual norm ------------------------------------------------------------------------------------------------
def _normalise(v, kind):
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    rstd = torch.rsqrt((v - mean).square().mean(1, keepdim=True) + EPS)
    return (v - mean) * rstd, rstd


def _normalise_back(d, n, rstd, kind):
    d = d - n * (d * n).mean(1, keepdim=True)
    return rstd * (d - d.mean(1, keepdim=True) if kind == "layer" else d)


def _run_norm(s):
    if own:
        return _own_norm(s)
    case, kind = s.case, s.case["norm"]
    f = lambda t: None if t is None else t.float()  # noqa: E731
    with torch.no_grad():
        u, gate, post, post_b, scale, pre, pre_b = map(f, (s.u, s.gate, s.post_weight, s.post_bias, s.scale, s.pre_weight, s.pre_bias))
        n, rstd = _normalise(u, kind) if post is not None else (u, None)
        v = n if post is None else n * post if post_b is None else n * post + post_b
        sig = None if gate is None else torch.sigmoid(gate)
        w = v if gate is None else v * (gate * sig)
        stream = s.residual.float() + (w if scale is None else scale * w)
        n2, rstd2 = _normalise(stream, kind) if pre is not None else (None, None)
        normed = None if pre is None else n2 * pre if pre_b is None else n2 * pre + pre_b
        res = _named(("stream", "normed"), (stream.to(s.residual.dtype), None if normed is None else normed.to(s.u.dtype)))
        if not case["train"]:
            return res
        par = _DT[case["par"]]
        total = lambda t: t.sum(0, dtype=torch.float64).to(par)  # noqa: E731
        d = s.dstream.float()
        if pre is not None:
            dnormed = s.dnormed.float()
            res["dpre_weight"] = total(dnormed * n2)
            if pre_b is not None:
                res["dpre_bias"] = total(dnormed)
            d = d + _normalise_back(dnormed * pre, n2, rstd2, kind)
        res["dresidual"] = d.to(s.residual.dtype)
        if scale is not None:
            res["dscale"] = total(d * w)
            d = d * scale
        if gate is not None:
            res["dgate"] = (d * v * (sig * (1 + gate * (1 - sig)))).to(s.gate.dtype)
            d = d * (gate * sig)
        if post is not None:
            res["dpost_weight"] = total(d * n)
            if post_b is not None:
                res["dpost_bias"] = total(d)
            d = _normalise_back(d * post, n, rstd, kind)
        res["du"] = d.to(s.u.dtype)
        return res


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def work(case):
    e, C = _BYTES[case["act"]], case["C"]
    if case["op"] == "step":
        n = case["B"] * C
        return {"bytes": n * (4 * e + 8), "flops": 14 * n}
    n = case["T"] * C
    if case["op"] == "recurrence":
        # x, both gates and y; training: dy in, dx and both gates' gradients out as well
        return {"bytes": n * e * (8 if case["train"] else 4), "flops": n * (36 if case["train"] else 14)}
    st, ga, pre = _BYTES[case["stream"]], int(case["gated"]), int(case["pre"])
    forward = e * (1 + ga + pre) + 2 * st                        # u, gate, normed; residual, stream
    back = e * (1 + ga + pre) + 2 * st                           # du, dgate, dnormed; dstream, dresidual
    return {"bytes": n * (forward + (back if case["train"] else 0)), "flops": n * (45 if case["train"] else 16)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """What ``run`` returns, from the definition in fp64: the recurrence one position after the other, gradients by differentiating the definition."""
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "step": _exact_step, "norm": _exact_norm}[case["op"]](s)


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_()


def _definition(x, r, i, decay):
    z = SCALE * torch.nn.functional.softplus(decay, threshold=700) * torch.sigmoid(r)
    return torch.exp(-z), torch.sqrt(-torch.expm1(-2 * z)) * torch.sigmoid(i) * x


def _walk(cu, longest, flipped):
    """The rows at each position of all sequences that reach it, longest sequences first."""
    lo, n = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    n, order = torch.sort(n, descending=True, stable=True)
    lo = lo[order]
    alive = torch.bincount(n.cpu(), minlength=longest + 1).flip(0).cumsum(0).flip(0).tolist()       # alive[p]: sequences of at least p rows
    for p in range(longest):
        k = alive[p + 1]
        yield order[:k], (lo[:k] + (n[:k] - 1 - p if flipped else p))


def _exact_recurrence(s):
    case, reverse, C = s.case, s.case["reverse"], s.case["C"]
    x, r, i = _leaf(s.x), _leaf(s.gates[:, :C]), _leaf(s.gates[:, C:])
    decay = _leaf(s.decay)
    a, b = _definition(x, r, i, decay)
    S = s.cu.numel() - 1
    with torch.no_grad():
        h = torch.zeros(S, C, device=DEV, dtype=torch.float64) if s.initial is None else s.initial.detach().double()
        y, before = torch.empty_like(b), torch.empty_like(b)
        one = S == 1
        for which, rows in _walk(s.cu, s.longest, reverse) if not one else ():
            old = h[which]
            before[rows] = old
            new = a[rows] * old + b[rows]
            y[rows] = new
            h[which] = new
        if one:
            T = case["T"]
            now = h[0]
            for t in range(T - 1, -1, -1) if reverse else range(T):
                before[t] = now
                now = torch.addcmul(b[t], a[t], now, out=y[t])
            h = now[None].clone()
        res = _named(("y", "state"), (y, h if case["states"] else None))
        if not case["train"]:
            return res
        g = torch.zeros_like(h) if s.dstate is None else s.dstate.double()      # the gradient that comes down to the row
        dy, dh = s.dy.double(), torch.empty_like(b)
        for which, rows in _walk(s.cu, s.longest, not reverse) if not one else ():
            here = dy[rows] + g[which]
            dh[rows] = here
            g[which] = a[rows] * here
        if one:
            for t in range(T) if reverse else range(T - 1, -1, -1):
                torch.add(dy[t], g[0], out=dh[t])
                torch.mul(a[t], dh[t], out=g[0])
    dx, dr, di, ddecay = torch.autograd.grad((a, b), (x, r, i, decay), (dh * before, dh))
    res.update(dx=dx, dgates=torch.cat([dr, di], 1), ddecay=ddecay)
    if s.initial is not None:
        res["dinitial"] = g
    return res


def _exact_step(s):
    C = s.case["C"]
    g = s.gates.double()
    a, b = _definition(s.x.double(), g[:, :C], g[:, C:], s.decay.double())
    state, y = s.state.double(), torch.zeros_like(b)
    for k, slot in enumerate(s.slots.tolist()):
        if slot >= 0:
            y[k] = state[slot] = a[k] * state[slot] + b[k]
    return {"y": y, "state": state}


def _exact_norm(s):
    case = s.case
    names = ("u", "gate", "residual", "post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
    L = {n: _leaf(getattr(s, n)) for n in names}

    def norm(v, w, b):
        c = v - v.mean(1, keepdim=True) if case["norm"] == "layer" else v
        out = c / torch.sqrt((c * c).mean(1, keepdim=True) + EPS) * w
        return out if b is None else out + b

    v = L["u"] if L["post_weight"] is None else norm(L["u"], L["post_weight"], L["post_bias"])
    if L["gate"] is not None:
        v = v * L["gate"] * torch.sigmoid(L["gate"])
    stream = L["residual"] + (v if L["scale"] is None else v * L["scale"])
    normed = None if L["pre_weight"] is None else norm(stream, L["pre_weight"], L["pre_bias"])
    res = {n: t.detach() for n, t in _named(("stream", "normed"), (stream, normed)).items()}
    if case["train"]:
        kept = [n for n in names if L[n] is not None]
        outs, douts = [stream], [s.dstream.double()]
        if normed is not None:
            outs, douts = outs + [normed], douts + [s.dnormed.double()]
        res.update({"d" + n: d for n, d in zip(kept, torch.autograd.grad(outs, [L[n] for n in kept], douts))})
    return res
