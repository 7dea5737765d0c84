"""Operators around the recurrent block, as cases that can be timed: linear attention with a decay for each head over packed rows, its single-token
step, and layer norm over whole rows or each head's channels.

A case is one call of a public door of the library (``varlen_linear_attention``, ``linear_attention_step``, ``layer_norm``), alone (``train`` false:
inference) or with the gradients of everything a training step needs (``train`` true). Sizes are those of the repository's benchmark configurations, of
the default widths of the model the operators sit in (hidden 768 and 1024, intermediate 2048) in heads of 64 and 128 channels, and generic ragged ones.

Fields: ``op`` attn | step | norm; ``act`` / ``par`` dtypes of activations and parameters (bf16 | fp32).
Attention: ``T`` rows of ``H`` heads, keys of ``K`` channels and values of ``V``; ``mix`` the lengths of the packed sequences; ``rate`` whether a decay
is one number a head or one a token and head; ``decays`` slow (a head forgets 0.2 % to 3 % a token) or wide (anything from nothing to nearly
everything); ``states`` whether it starts from given states and returns the last ones; ``reverse``.
Step: ``B`` rows, one token each; ``N`` states in the table; ``padding`` whether some of the rows are padding.
Norm: ``T`` rows of ``C`` channels in ``heads`` groups; ``norm`` layer | rms; ``gated``, ``biased`` which parts it has; ``shared`` whether the heads
share one weight; ``sliced`` whether x and the gate are halves of one wider tensor.

``own`` false computes the same with elementary operations in fp32 (fp64 for sums of log decays and the long sums of parameters' gradients).
"""
import math
import types

import numpy as np
import torch

own = False

DEV = "cuda"
CHUNK = 64
EPS = 1e-5
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}
_MEAN = {"one": None, "short": 74, "usual": 266, "skewed": 330, "stress": 185, "ragged": 300}


def _attn(name, T, H, K, V, act, par, mix, train, rate="token", decays="slow", states=False, reverse=False):
    return dict(name=name, op="attn", T=T, H=H, K=K, V=V, act=act, par=par, mix=mix, train=train, rate=rate, decays=decays, states=states, reverse=reverse)


def _step(name, B, H, K, V, N, act, par, rate, padding):
    return dict(name=name, op="step", B=B, H=H, K=K, V=V, N=N, act=act, par=par, rate=rate, padding=padding)


def _norm(name, T, C, heads, act, par, norm, train, gated=False, biased=False, shared=False, sliced=False):
    return dict(name=name, op="norm", T=T, C=C, heads=heads, act=act, par=par, norm=norm, train=train, gated=gated, biased=biased, shared=shared,
                sliced=sliced)


def listed():
    return [
        # a training step of one small batch through a narrow layer, from the right, with states carried in and out: latency
        _attn("attn_train_small", 776, 2, 32, 32, "fp32", "fp32", "short", True, states=True, reverse=True),
        # the headline packed batch (131072 rows, hidden 1024 in heads of 64), forward and backward
        _attn("attn_train_packed", 131072, 16, 64, 64, "bf16", "bf16", "usual", True),
        # an fp32 stream at hidden 768, many sequences of a few rows, one learned decay a head
        _attn("attn_train_fp32_stress", 32768, 12, 64, 64, "fp32", "fp32", "stress", True, rate="head"),
        # one long sequence trained whole, from the right, values wider than keys, decays in fp32 beside bf16 activations
        _attn("attn_train_long", 20011, 8, 64, 128, "bf16", "fp32", "one", True, decays="wide", states=True, reverse=True),
        # heads of odd width: rows that no vector fits
        _attn("attn_train_odd", 5003, 11, 48, 91, "bf16", "bf16", "usual", True, rate="head"),
        # prefill of one very long sequence at the intermediate width in heads of 128, state handed on
        _attn("attn_prefill_long", 65536, 16, 128, 128, "bf16", "bf16", "one", False, rate="head", states=True),
        # one token of one sequence
        _step("attn_step_single", 1, 16, 64, 64, 8, "bf16", "bf16", "head", False),
        # a serving batch at the intermediate width, some rows padding
        _step("attn_step_batch", 250, 16, 128, 128, 300, "bf16", "fp32", "token", True),
        # the norm in front of a block for a few tokens: latency
        _norm("norm_tokens", 8, 2048, 1, "bf16", "bf16", "layer", False),
        # the first norm of the model in a training step of the headline batch
        _norm("norm_train_packed", 131072, 1024, 1, "bf16", "bf16", "layer", True, biased=True),
        # behind the attention: rms of each head, gated, one weight for all heads
        _norm("norm_train_heads", 131072, 1024, 16, "bf16", "bf16", "rms", True, gated=True, shared=True, sliced=True),
        # an odd width in fp32
        _norm("norm_train_odd", 5003, 1001, 1, "fp32", "fp32", "layer", True, biased=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _head(rng):
    return rng.choice([32, 64, 64, 128, 128, rng.randrange(3, 129), 8 * rng.randrange(2, 17)])


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "step", "norm", "norm"])
    act, par = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
    e = _BYTES[act]
    if op == "norm":
        C = rng.choice([64, 512, 768, 1000, 1024, 2048, rng.randrange(65, 2050), 8 * rng.randrange(8, 257)])
        heads = rng.choice([1, 1] + [h for h in (2, 4, 7, 8, 12, 16, 32) if C % h == 0 and C // h >= 16])
        T = _log(rng, 1, min(131072, 131072 * 1024 * 2 // (C * e)))
        case = _norm("", T, C, heads, act, par, rng.choice(["layer", "rms"]), rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.4,
                     heads > 1 and rng.random() < 0.6, rng.random() < 0.3)
        del case["name"]
        return case
    H, K, V = rng.choice([1, 2, 4, 8, 12, 16, rng.randrange(1, 17)]), _head(rng), _head(rng)
    if rng.random() < 0.5:
        V = K
    rate = rng.choice(["token", "head"])
    if op == "step":
        B = _log(rng, 1, 256)
        case = _step("", B, H, K, V, B + rng.randrange(1, 64), act, par, rate, rng.random() < 0.5)
    else:
        train = rng.random() < 0.7
        mix = rng.choice(["usual", "usual", "skewed", "stress", "short", "ragged", "one"])
        most = min(131072, 131072 * 16 * 128 * 2 // (H * (K + V) * e), 131072 * 16 * 4096 // (H * K * V))
        if mix == "one":
            most = min(most, 32768 if train else 65536)
        T = _log(rng, 1, most)
        case = _attn("", T, H, K, V, act, par, mix, train, rate, rng.choice(["slow", "wide"]), rng.random() < 0.4, rng.random() < 0.4)
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
    g = torch.Generator(DEV).manual_seed(seed * 7919 + 13)
    s = types.SimpleNamespace(case=case)
    act, par, train = _DT[case["act"]], _DT[case["par"]], case.get("train", False)

    def normal(*shape, dtype=act, std=1.0, mean=0.0, grad=False):
        t = torch.randn(*shape, device=DEV, generator=g).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(grad)

    if case["op"] == "norm":
        T, C = case["T"], case["C"]
        if case["sliced"]:
            s.wide = normal(T, 2 * C, mean=0.2)
            s.x, s.gate = s.wide[:, :C], s.wide[:, C:]
            s.x.requires_grad_(train), s.gate.requires_grad_(train)
        else:
            s.x, s.gate = normal(T, C, std=2.0, mean=0.3, grad=train), normal(T, C, grad=train)
        s.gate = s.gate if case["gated"] else None
        n = C // case["heads"] if case["shared"] else C
        s.weight = normal(n, dtype=par, std=0.1, mean=1.0, grad=train)
        s.bias = normal(n, dtype=par, std=0.1, grad=train) if case["biased"] else None
        s.dy = normal(T, C) if train else None
        return s
    H, K, V = case["H"], case["K"], case["V"]
    n = case["B"] if case["op"] == "step" else case["T"]
    s.scale = K ** -0.5
    # queries, keys and values are column slices of one projection's rows
    s.wide = normal(n, H * (2 * K + V))
    s.q, s.k, s.v = (t.view(n, H, -1) for t in s.wide.split([H * K, H * K, H * V], 1))
    shape = (H,) if case["rate"] == "head" else (n, H)
    if case.get("decays") == "wide":
        kept = torch.sigmoid(normal(*shape, dtype=torch.float32, std=3.0))
    else:
        kept = torch.rand(*shape, device=DEV, generator=g).mul_(0.028).add_(0.97)
    s.log_decay = torch.log(kept).to(par).requires_grad_(train)
    rs = np.random.RandomState(seed % (1 << 32))
    if case["op"] == "step":
        slots = rs.permutation(case["N"])[:n]
        if case["padding"]:
            slots[rs.rand(n) < 0.1] = -1
        s.slots = torch.from_numpy(slots.astype(np.int32)).to(DEV)
        s.state = normal(case["N"], H, K, V, dtype=torch.float32, std=2.0)
        s.out_state = s.state.clone()                            # (the old states stay until the token is accepted)
        return s
    for t in (s.q, s.k, s.v):
        t.requires_grad_(train)
    lengths = rs.permutation(_lengths(case["mix"], n, np.random.RandomState(n))).tolist()    # (as many sequences whatever the seed)
    s.longest = max(lengths)
    s.cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).to(DEV)
    s.initial = normal(len(lengths), H, K, V, dtype=torch.float32, grad=train) if case["states"] else None
    s.do = normal(n, H, V) if train else None
    s.dstate = normal(len(lengths), H, K, V, dtype=torch.float32, std=0.1) if train and case["states"] else None
    return s


def run(s):
    return {"attn": _run_attn, "step": _run_step, "norm": _run_norm}[s.case["op"]](s)


def _named(names, values):
    return {n: v for n, v in zip(names, values) if v is not None}


# ---- the framework's calls ------------------------------------------------------------------------------------------------------------
def _grads(outs, douts, names, leaves):
    """Gradients of the outputs that there are, by name."""
    kept = [(n, t) for n, t in zip(names, leaves) if t is not None]
    pairs = [(o, d) for o, d in zip(outs, douts) if o is not None]
    return dict(zip([n for n, _ in kept], torch.autograd.grad([o for o, _ in pairs], [t for _, t in kept], [d for _, d in pairs])))


def _own_attn(s):
    import nanoplm_amd as npa
    out = npa.varlen_linear_attention(s.q, s.k, s.v, s.cu, s.log_decay, scale=s.scale, initial_state=s.initial, reverse=s.case["reverse"],
                                      return_state=s.case["states"])
    o, state = out if s.case["states"] else (out, None)
    res = _named(("o", "state"), (o, state))
    if s.case["train"]:
        res.update(_grads((o, state), (s.do, s.dstate), ("dq", "dk", "dv", "dlog_decay", "dinitial"), (s.q, s.k, s.v, s.log_decay, s.initial)))
    return res


def _own_step(s):
    import nanoplm_amd as npa
    o = npa.linear_attention_step(s.q, s.k, s.v, s.log_decay, s.state, s.slots, scale=s.scale, out_state=s.out_state)
    return {"o": o, "state": s.out_state}


def _own_norm(s):
    import nanoplm_amd as npa
    y = npa.layer_norm(s.x, s.weight, s.bias, gate=s.gate, heads=s.case["heads"], norm=s.case["norm"], eps=EPS)
    res = {"y": y}
    if s.case["train"]:
        res.update(_grads((y,), (s.dy,), ("dx", "dgate", "dweight", "dbias"), (s.x, s.gate, s.weight, s.bias)))
    return res


# ---- the plain form of the attention ----------------------------------------------------------------------------------------------------
def _table(s):
    """Pieces of CHUNK rows of the sequences: rows [n, CHUNK] (T where there is none), the sequence of each piece, whether it is its first, the
    last piece of each sequence (pieces without rows stand between the sequences)."""
    T, S = s.case["T"], s.cu.numel() - 1
    lo, hi = s.cu[:-1].long(), s.cu[1:].long()
    base = lo // CHUNK + torch.arange(S, device=DEV)
    n = T // CHUNK + S + 1
    c = torch.arange(n, device=DEV)
    which = torch.searchsorted(base, c, right=True).sub_(1).clamp_(min=0)
    at = (c - base[which])[:, None] * CHUNK + torch.arange(CHUNK, device=DEV)
    real = at < (hi - lo)[which][:, None]
    rows = hi[which][:, None] - 1 - at if s.case["reverse"] else lo[which][:, None] + at
    last = torch.cat([base[1:], base.new_tensor([n])]) - 1
    return torch.where(real, rows, T), which, at[:, 0] == 0, last


def _scan(a, x, longest):
    """x_c = a_c x_{c-1} + x_c down the pieces, by doubling; a is zero where a sequence begins. Overwrites both."""
    k = 1
    while k < longest:
        nx = torch.addcmul(x[k:], a[k:], x[:-k])
        na = a[k:] * a[:-k]
        x[k:], a[k:] = nx, na
        k *= 2
    return x


def _run_attn(s):
    if own:
        return _own_attn(s)
    case = s.case
    with torch.no_grad():
        T, H, K, V = case["T"], case["H"], case["K"], case["V"]
        rows, which, first, last = _table(s)
        longest = rows.shape[0]

        def pieces(t):                                           # [T, H, n] -> [pieces, H, CHUNK, n]
            return torch.cat([t.float(), torch.zeros(1, *t.shape[1:], device=DEV)])[rows].transpose(1, 2).contiguous()

        def whole(t, n):                                         # and back
            out = torch.zeros(T + 1, H, n, device=DEV)
            out[rows] = t.transpose(1, 2)
            return out[:T]

        q, k, v = pieces(s.q) * s.scale, pieces(s.k), pieces(s.v)
        log_decay = s.log_decay.double().expand(T, H)
        b = torch.cumsum(torch.cat([log_decay, torch.zeros(1, H, device=DEV, dtype=torch.float64)])[rows].transpose(1, 2), 2)
        i = torch.arange(CHUNK, device=DEV)
        D = torch.exp(torch.where(i[:, None] >= i, b[..., :, None] - b[..., None, :], -math.inf)).float()
        left = torch.exp(b[..., -1:] - b).float()[..., None]     # what is left of a row's product at the piece's end
        since = torch.exp(b).float()[..., None]                  # and of the state in front of the piece, at a row
        whole_decay = since[:, :, -1:]
        start = first[:, None, None, None]
        carried = torch.zeros(1, device=DEV) if s.initial is None else s.initial[which]
        out_state = (k * left).transpose(2, 3) @ v
        out_state = out_state + whole_decay * torch.where(start, carried, 0.0)
        out_state = _scan(torch.where(start, 0.0, whole_decay), out_state, longest)
        into = torch.where(start, carried, out_state.roll(1, 0))
        A = q @ k.transpose(2, 3)
        o = whole((A * D) @ v + since * (q @ into), V)
        res = {"o": o.to(s.q.dtype)}
        if case["states"]:
            res["state"] = out_state[last]
        if not case["train"]:
            return res
        do = pieces(s.do)
        end = torch.zeros_like(first)
        end[last] = True
        end = end[:, None, None, None]
        coming = torch.zeros(1, device=DEV) if s.dstate is None else s.dstate[which]
        d_in = (q * since).transpose(2, 3) @ do
        d_in = d_in + whole_decay * torch.where(end, coming, 0.0)
        d_in = _scan(torch.where(end, 0.0, whole_decay).flip(0), d_in.flip(0), longest).flip(0)
        d_out = torch.where(end, coming, d_in.roll(-1, 0))
        dA = (do @ v.transpose(2, 3)) * D
        dq = dA @ k + since * (do @ into.transpose(2, 3))                                       # of scale * q
        dk = dA.transpose(2, 3) @ q + left * (v @ d_out.transpose(2, 3))
        dv = (A * D).transpose(2, 3) @ do + left * (k @ d_out)
        # a decay scales every product that crosses it: of rows in front of it and behind it in its piece (a row's product with itself crosses none), of
        # the state in front of the piece and a row behind it, of a row in front of it and what reads the state behind the piece, of both states
        crossing = (A * dA * (i[:, None] > i)).double()
        e = crossing.sum(3) - crossing.sum(2) + (q * since * (do @ into.transpose(2, 3))).double().sum(3) - (k * left * (v @ d_out.transpose(2, 3))).double().sum(3)
        behind = torch.flip(torch.cumsum(torch.flip(e, (2,)), 2), (2,))
        across = (out_state * d_out).sum((2, 3), dtype=torch.float64)
        dlog = whole((behind + across[..., None]).float()[..., None], 1)[..., 0]
        res["dq"], res["dk"], res["dv"] = (whole(t, n).to(s.q.dtype) for t, n in ((dq * s.scale, K), (dk, K), (dv, V)))
        res["dlog_decay"] = (dlog.sum(0, dtype=torch.float64) if case["rate"] == "head" else dlog).to(s.log_decay.dtype)
        if s.initial is not None:
            begin = torch.nonzero(first, as_tuple=True)[0]
            res["dinitial"] = torch.zeros_like(s.initial).index_copy_(0, which[begin], d_in[begin])
        return res


def _run_step(s):
    if own:
        return _own_step(s)
    with torch.no_grad():
        q, k, v = s.q.float() * s.scale, s.k.float(), s.v.float()
        a = torch.exp(s.log_decay.float()).expand(q.shape[:2])[..., None, None]
        real = s.slots >= 0
        at = s.slots.long().clamp(min=0)
        h = a * s.state[at] + k[..., :, None] * v[..., None, :]
        # a padding row writes to a row behind the table
        table = torch.cat([s.state, s.state[:1]])
        table[torch.where(real, at, s.state.shape[0])] = h
        s.out_state.copy_(table[:-1])
        o = (q[..., :, None] * h).sum(2)
        return {"o": torch.where(real[:, None, None], o, 0.0).to(s.q.dtype), "state": s.out_state}


# ---- the plain form of the norm ---------------------------------------------------------------------------------------------------------
def _run_norm(s):
    if own:
        return _own_norm(s)
    case = s.case
    with torch.no_grad():
        T, C, G = case["T"], case["C"], case["heads"]
        n = C // G
        f = lambda t: None if t is None else t.float().view(-1, G if t.shape[-1] == C else 1, n)  # noqa: E731
        x, gate, w, b = f(s.x.contiguous()), None if s.gate is None else f(s.gate.contiguous()), f(s.weight), f(s.bias)
        c = x - x.mean(2, keepdim=True) if case["norm"] == "layer" else x
        rstd = torch.rsqrt(c.square().mean(2, keepdim=True) + EPS)
        normed = c * rstd
        y = normed * w if b is None else normed * w + b
        sig = None if gate is None else torch.sigmoid(gate)
        res = {"y": (y if gate is None else y * (gate * sig)).to(s.x.dtype).view(T, C)}
        if not case["train"]:
            return res
        par = _DT[case["par"]]
        d = f(s.dy)
        if gate is not None:
            res["dgate"] = (d * y * (sig * (1 + gate * (1 - sig)))).to(s.gate.dtype).view(T, C)
            d = d * (gate * sig)
        total = lambda t: t.sum((0, 1) if case["shared"] else 0, dtype=torch.float64).to(par).flatten()  # noqa: E731
        res["dweight"] = total(d * normed)
        if b is not None:
            res["dbias"] = total(d)
        d = d * w
        d = d - normed * (d * normed).mean(2, keepdim=True)
        d = rstd * (d - d.mean(2, keepdim=True) if case["norm"] == "layer" else d)
        res["dx"] = d.to(s.x.dtype).view(T, C)
        return {k: res[k] for k in ("y", "dx", "dgate", "dweight", "dbias") if k in res}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def work(case):
    e = _BYTES[case["act"]]
    if case["op"] == "norm":
        n = case["T"] * case["C"]
        g = int(case["gated"])
        # x, gate, y; training: dy in, dx and the gate's gradient out as well
        return {"bytes": n * e * ((2 + g) + (2 + g if case["train"] else 0)), "flops": n * ((20 if case["train"] else 8) + 10 * g)}
    H, K, V = case["H"], case["K"], case["V"]
    if case["op"] == "step":
        return {"bytes": case["B"] * H * (8 * K * V + e * (2 * K + 2 * V)), "flops": case["B"] * H * 5 * K * V}
    n = case["T"] * H
    # q, k, v and o; training: the gradient of o in, those of q, k and v out as well. A row's outer product joins the state and the state is read,
    # two operations an element each; training: four such products more
    rows = n * e * (2 * K + 2 * V) + (n * e * (2 * K + 2 * V) if case["train"] else 0)
    rate = 0 if case["rate"] == "head" else n * _BYTES[case["par"]] * (2 if case["train"] else 1)
    S = 1 if _MEAN[case["mix"]] is None else case["T"] // _MEAN[case["mix"]] + 1
    states = S * H * K * V * 4 * (4 if case["train"] else 2) if case["states"] else 0
    return {"bytes": rows + rate + states, "flops": n * K * V * (12 if case["train"] else 4)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """What ``run`` returns, from the definition in fp64: the attention one position after the other, the norm's gradients by differentiating it."""
    s = prepare(case, seed)
    return {"attn": _exact_attn, "step": _exact_step, "norm": _exact_norm}[case["op"]](s)


def _walk(cu, longest, flipped):
    """The rows at each position of all sequences that reach it, longest sequences first."""
    lo, n = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    n, order = torch.sort(n, descending=True, stable=True)
    lo = lo[order]
    alive = torch.bincount(n.cpu(), minlength=longest + 1).flip(0).cumsum(0).flip(0).tolist()       # alive[p]: sequences of at least p rows
    for p in range(longest):
        m = alive[p + 1]
        yield order[:m], (lo[:m] + (n[:m] - 1 - p if flipped else p))


def _exact_attn(s):
    case, reverse = s.case, s.case["reverse"]
    T, H, K, V = case["T"], case["H"], case["K"], case["V"]
    d = lambda t: t.detach().double()  # noqa: E731
    with torch.no_grad():
        q, k, v = d(s.q) * s.scale, d(s.k), d(s.v)
        a = torch.exp(d(s.log_decay)).expand(T, H)
        S = s.cu.numel() - 1
        new = lambda *n: torch.zeros(*n, device=DEV, dtype=torch.float64)  # noqa: E731
        h = new(S, H, K, V) if s.initial is None else d(s.initial).clone()
        o, do = new(T, H, V), None if s.do is None else d(s.do)
        dq = new(T, H, K)
        for which, rows in _walk(s.cu, s.longest, reverse):
            now = a[rows][..., None, None] * h[which] + k[rows][..., :, None] * v[rows][..., None, :]
            h[which] = now
            o[rows] = (q[rows][..., None, :] @ now)[..., 0, :]
            if do is not None:
                dq[rows] = (now @ do[rows][..., None])[..., 0]
        res = _named(("o", "state"), (o, h if case["states"] else None))
        if not case["train"]:
            return res
        g = new(S, H, K, V) if s.dstate is None else d(s.dstate).clone()
        dk, dv = new(T, H, K), new(T, H, V)
        for which, rows in _walk(s.cu, s.longest, not reverse):
            now = g[which] + q[rows][..., :, None] * do[rows][..., None, :]
            dk[rows] = (now @ v[rows][..., None])[..., 0]
            dv[rows] = (k[rows][..., None, :] @ now)[..., 0, :]
            g[which] = a[rows][..., None, None] * now
        # log a_t is in every exp(b_i - b_j) with j < t <= i: d/db_t is q_t dq_t - k_t dk_t, and d/dlog a_t its sum from t to the sequence's end
        e = (q * dq - k * dk).sum(2)
        lengths = (s.cu[1:] - s.cu[:-1]).long()
        some = lengths > 0
        ends = (s.cu[:-1] if reverse else s.cu[1:] - 1).long()[some]
        if s.dstate is not None:
            e[ends] += (h * d(s.dstate)).sum((2, 3))[some]
        up = (lambda t: t) if reverse else (lambda t: t.flip(0))  # noqa: E731
        sums = up(torch.cumsum(up(e), 0))
        # what lies behind a sequence's last row (in the walk's order)
        behind = (sums[ends] - e[ends]).repeat_interleave(lengths[some], 0)
        dlog = sums - behind
        res.update(dq=dq * s.scale, dk=dk, dv=dv, dlog_decay=dlog.sum(0) if case["rate"] == "head" else dlog)
        if s.initial is not None:
            res["dinitial"] = g
        return res


def _exact_step(s):
    q, k, v = s.q.double() * s.scale, s.k.double(), s.v.double()
    a = torch.exp(s.log_decay.double()).expand(q.shape[:2])
    state, o = s.state.double(), torch.zeros_like(v)
    for row, slot in enumerate(s.slots.tolist()):
        if slot >= 0:
            state[slot] = a[row][:, None, None] * state[slot] + k[row][:, :, None] * v[row][:, None, :]
            o[row] = (q[row][:, None, :] @ state[slot])[:, 0]
    return {"o": o, "state": state}


def _exact_norm(s):
    case = s.case
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_()  # noqa: E731
    x, gate, weight, bias = leaves = [leaf(t) for t in (s.x, s.gate, s.weight, s.bias)]
    T, C, G = case["T"], case["C"], case["heads"]
    u = x.reshape(T, G, C // G)
    if case["norm"] == "layer":
        u = u - u.sum(2, keepdim=True) / (C // G)
    u = u / torch.sqrt((u * u).sum(2, keepdim=True) / (C // G) + EPS)
    spread = lambda t: t.repeat(G) if t.numel() != C else t  # noqa: E731
    y = u.reshape(T, C) * spread(weight)
    if bias is not None:
        y = y + spread(bias)
    if gate is not None:
        y = y * gate / (1 + torch.exp(-gate))
    res = {"y": y.detach()}
    if case["train"]:
        kept = [(n, t) for n, t in zip(("dx", "dgate", "dweight", "dbias"), leaves) if t is not None]
        res.update(zip([n for n, _ in kept], torch.autograd.grad(y, [t for _, t in kept], s.dy.double())))
    return res
