"""The packed recurrent block: pre-norm conv, gated linear recurrence and residual norm as a layer uses them together; refusals on device tensors."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

import nanoplm_amd as npa
from tests import recurrence_ref as R

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


class Block(nn.Module):
    """normed rows -> projection -> short conv -> gates -> recurrence (both directions) -> gated norm, residual and the next block's norm."""

    def __init__(self, C):
        super().__init__()
        self.proj, self.to_gates = nn.Linear(C, 2 * C, bias=False), nn.Linear(C, 2 * C)
        self.conv = npa.VarlenDWConv1d(C, 5, residual=True)
        self.left, self.right = npa.VarlenRecurrence(C), npa.VarlenRecurrence(C, reverse=True)
        self.join = npa.ResidualNorm(C, norm="rms", scale_init=0.5)

    def forward(self, stream, normed, cu):
        x, gate = self.proj(normed).chunk(2, dim=-1)
        x = self.conv(x, cu)
        gates = self.to_gates(x)
        return self.join(self.left(x, gates, cu) + self.right(x, gates, cu), stream, gate)


def _reference(block, stream, normed, cu, lens):
    """The same in fp64 on the CPU, differentiable."""
    C = normed.shape[1]
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in block.named_parameters()}
    s, x0 = stream.detach().cpu().double().requires_grad_(), normed.detach().cpu().double().requires_grad_()
    x, gate = (x0 @ p["proj.weight"].t()).chunk(2, dim=-1)
    rows = []
    for part in x.split(lens):
        y = F.conv1d(part.t()[None], p["conv.weight"][:, None], p["conv.bias"], padding=2, groups=C)[0].t() if part.shape[0] else part
        rows.append(part + y)
    x = torch.cat(rows)
    gates = x @ p["to_gates.weight"].t() + p["to_gates.bias"]
    u = torch.zeros_like(x)
    for name, reverse in (("left", False), ("right", True)):
        k = R.coefficients(x, gates, p[f"{name}.decay"], 8.0)
        out = [None] * x.shape[0]
        for lo, hi, _ in R.sequences(cu.cpu(), x.shape[0]):
            h = torch.zeros(C, dtype=torch.float64)
            for t in range(hi - 1, lo - 1, -1) if reverse else range(lo, hi):
                h = k["a"][t] * h + k["b"][t]
                out[t] = h
        u = u + torch.stack(out)
    rms = lambda a: a / torch.sqrt((a * a).mean(1, keepdim=True) + 1e-5)
    new = s + p["join.scale"] * rms(u) * p["join.post_weight"] * F.silu(gate)
    return (new, rms(new) * p["join.pre_weight"]), [s, x0] + list(p.values())


def test_a_block_and_its_gradients():
    """fp32 against fp64. Each of the eight steps in either direction leaves at most about 32 roundings of 2^-24 (2e-6) on its terms, and none gains
    more than a few times: 1e-4 of a tensor's norm."""
    torch.manual_seed(0)
    C, lens = 48, [70, 0, 1, 130, 64, 5]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    T = sum(lens)
    block = Block(C).cuda()
    stream, normed = torch.randn(T, C, device="cuda", requires_grad=True), torch.randn(T, C, device="cuda", requires_grad=True)
    d = [torch.randn(T, C, device="cuda") for _ in range(2)]
    want, leaves = _reference(block, stream, normed, cu, lens)
    wgrads = torch.autograd.grad(want, leaves, [t.cpu().double() for t in d])
    out = block(stream, normed, cu)
    grads = torch.autograd.grad(out, [stream, normed] + list(block.parameters()), d)
    for name, a, b in zip(["stream", "normed", "d stream", "d normed"] + [n for n, _ in block.named_parameters()], list(out) + list(grads), list(want) + list(wgrads)):
        off = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 1e-4, (name, off)


def test_two_blocks_under_autocast_compiled_and_replayed():
    """bf16 branches on an fp32 stream, two blocks chained through (stream, normed): eager, compiled, and captured with its backward into a graph."""
    torch.manual_seed(1)
    C, lens = 128, [300, 17, 0, 500, 207]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    T = sum(lens)
    blocks = nn.ModuleList([Block(C), Block(C)]).cuda()
    stream, normed = torch.randn(T, C, device="cuda"), torch.randn(T, C, device="cuda")
    params = list(blocks.parameters())

    def step(stream, normed):
        with torch.autocast("cuda", BF16, cache_enabled=False):
            for b in blocks:
                stream, normed = b(stream, normed, cu)
        assert stream.dtype == F32
        loss = stream.square().mean() + normed.float().square().mean()
        return [loss.detach(), stream.detach()] + list(torch.autograd.grad(loss, params))
    want = [t.clone() for t in step(stream, normed)]
    assert all(bool(torch.isfinite(t).all()) for t in want)
    got = torch.compile(step, dynamic=False, backend="aot_eager")(stream, normed)
    assert all(torch.equal(a, b) for a, b in zip(want[:2], got[:2]))
    del got
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(stream, normed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(stream, normed)
    for k in range(3):
        stream.normal_()
        graph.replay()
        torch.cuda.synchronize()
        # the stream, which no library sum over blocks had a part in
        assert torch.equal(step(stream, normed)[1], outs[1]), k


def test_two_calls_at_once_on_two_streams():
    g = torch.Generator("cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    T, C = 5000, 256
    cu = torch.tensor([0, 100, 4700, T], dtype=torch.int32).cuda()
    ins = [[n(T, C), n(T, 2 * C), n(C), n(T, C)] for _ in range(2)]

    def call(x, gates, decay, dy):
        y, _, carries = npa.varlen_recurrence_fwd(x, gates, cu, decay, want_carries=True)
        out = npa.varlen_recurrence_bwd(x, gates, dy, cu, decay, carries)
        stream, normed, stats = npa.residual_norm_fwd(y, x, dy, decay, pre_weight=decay, want_stats=True)
        return [y, *out[:3], stream, normed, *[t for t in npa.residual_norm_bwd(y, x, dy, decay, None, None, decay, stats, dy, x) if t is not None]]
    want = [call(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, i in zip(streams, ins):
            with torch.cuda.stream(s):
                got.append(call(*i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_recurrence_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    cu = torch.tensor([0, 5], dtype=torch.int32).cuda()
    good = dict(x=z(5, 4), gates=z(5, 8), cu_seqlens=cu, decay=z(4))
    npa.varlen_recurrence(**good)
    for bad, err in [(dict(gates=z(5, 7)), ValueError), (dict(gates=z(4, 8)), ValueError), (dict(gates=z(5, 8, d=BF16)), TypeError), (dict(decay=z(5)), ValueError),
                     (dict(decay=z(4, d=torch.float16)), TypeError), (dict(cu_seqlens=cu.long()), TypeError), (dict(cu_seqlens=cu[:0]), TypeError),
                     (dict(cu_seqlens=cu.cpu()), RuntimeError), (dict(gates=z(5, 8).cpu()), RuntimeError), (dict(decay=z(4).cpu()), RuntimeError),
                     (dict(x=z(5, 0), gates=z(5, 0), decay=z(0)), ValueError), (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError),
                     (dict(initial_state=z(2, 4)), ValueError), (dict(initial_state=z(1, 4, d=BF16)), ValueError),
                     (dict(initial_state=z(1, 4).cpu()), RuntimeError)]:
        with pytest.raises(err):
            npa.varlen_recurrence(**{**good, **bad})
    _, _, carries = npa.varlen_recurrence_fwd(**good, want_carries=True)
    args = (good["x"], good["gates"], z(5, 4), cu, good["decay"])
    npa.varlen_recurrence_bwd(*args, carries)
    for a, c, k in ((args, None, {}), (args, carries[:, :3], {}), (args, carries, dict(dstate=z(3, 4))), (args[:2] + (z(5, 4, d=BF16),) + args[3:], carries, {})):
        with pytest.raises(ValueError):
            npa.varlen_recurrence_bwd(*a, c, **k)


def test_step_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(x=z(5, 4), gates=z(5, 8), decay=z(4), state=z(6, 4), slots=z(5, d=torch.int32))
    npa.recurrence_step(**good)
    for bad, err in [(dict(state=z(6, 5)), ValueError), (dict(state=z(6, 4, d=BF16)), ValueError), (dict(state=z(4, 6).t()), ValueError),
                     (dict(out_state=z(5, 4)), ValueError), (dict(slots=z(5, d=torch.int64)), TypeError), (dict(slots=z(4, d=torch.int32)), TypeError),
                     (dict(slots=None, state=z(4, 4)), ValueError), (dict(slots=z(5, d=torch.int32).cpu()), RuntimeError), (dict(state=z(6, 4).cpu()), RuntimeError),
                     (dict(x=z(5, 4).requires_grad_()), RuntimeError)]:
        with pytest.raises(err):
            npa.recurrence_step(**{**good, **bad})
    with torch.no_grad():
        npa.recurrence_step(**{**good, "x": z(5, 4).requires_grad_()})
    assert npa.recurrence_step(z(0, 4), z(0, 8), z(4), z(6, 4)).shape == (0, 4)


def test_residual_norm_refusals():
    z = lambda *s, d=F32: torch.zeros(*s, dtype=d, device="cuda")
    good = dict(u=z(5, 4), residual=z(5, 4), gate=z(5, 4), post_weight=z(4), pre_weight=z(4))
    npa.residual_norm(**good)
    for bad, err in [(dict(residual=z(5, 5)), ValueError), (dict(residual=z(5, 4, d=BF16)), TypeError), (dict(gate=z(4, 4)), ValueError),
                     (dict(gate=z(5, 4, d=BF16)), ValueError), (dict(post_weight=z(5)), ValueError), (dict(scale=z(4, d=torch.float16)), TypeError),
                     (dict(post_weight=None, post_bias=z(4)), ValueError), (dict(pre_weight=None, pre_bias=z(4)), ValueError), (dict(norm="none"), ValueError),
                     (dict(eps=-1.0), ValueError), (dict(scale=z(4).cpu()), RuntimeError), (dict(residual=z(5, 4).cpu()), RuntimeError),
                     (dict(u=z(2, 16385), residual=z(2, 16385), gate=None, post_weight=None, pre_weight=None), ValueError)]:
        with pytest.raises(err):
            npa.residual_norm(**{**good, **bad})
