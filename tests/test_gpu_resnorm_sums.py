"""The parameters' gradients of the residual norm where a lane adds up many rows: against sums in 64 bits on the device."""
import pytest
import torch

import nanoplm_amd as npa

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _whole(T, C, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-2, 3, (T, C), dtype=torch.int8, device="cuda", generator=g).to(dtype)


def _column_sums(*factors):
    """The sum over the rows of the product of some [T, C] tensors, in fp64, piece by piece."""
    total = torch.zeros(factors[0].shape[1], dtype=torch.float64, device="cuda")
    for parts in zip(*(f.split(1 << 15) for f in factors)):
        t = parts[0].double()
        for p in parts[1:]:
            t = t * p.double()
        total += t.sum(0)
    return total


# 128 and 256 rows a lane; more rows than the usual number of blocks may add up (4096 a lane)
@pytest.mark.parametrize("T,C,act,st", [(131072, 1024, BF16, BF16), (131071, 1024, BF16, F32), (131072, 768, F32, F32), (131073, 2050, BF16, BF16),
                                        (2200000, 1032, BF16, BF16)])
def test_sums_of_whole_numbers_are_exact(T, C, act, st):
    """Whole numbers from -2 to 2: every product and every partial sum is below 2^24, so no row may be left out, or come twice, or be rounded."""
    assert 4 * T < 2 ** 24
    u, x, ds = _whole(T, C, act, 0), _whole(T, C, st, 1), _whole(T, C, st, 2)
    one = torch.ones(C, device="cuda")
    stats = npa.residual_norm_fwd(u, x, None, None, None, one, None, want_stats=True)[2]
    out = npa.residual_norm_bwd(u, x, None, None, None, one, None, stats, ds, None)
    assert torch.equal(out[5].double(), _column_sums(ds, u)), "dscale"
    del out
    stats = npa.residual_norm_fwd(u, x, None, one, one, None, None, want_stats=True)[2]
    out = npa.residual_norm_bwd(u, x, None, one, one, None, None, stats, ds, None)
    assert torch.equal(out[4].double(), _column_sums(ds)), "dpost_bias"
    del out, ds
    dy = _whole(T, C, act, 3)
    stats = npa.residual_norm_fwd(u, x, None, None, None, None, one, one, want_stats=True)[2]
    out = npa.residual_norm_bwd(u, x, None, None, None, None, one, stats, None, dy, pre_bias=True)
    assert torch.equal(out[7].double(), _column_sums(dy)), "dpre_bias"


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("act,st", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_weights_of_both_norms(act, st, norm):
    """T=131072, C=1024: a lane adds up 128 rows, two lanes' sums are added, then 512 blocks' in fp64. What fp32 may leave on a term g * n: n's mean and
    variance are sums of 32 roundings at most (16 channels a lane, exchanges, division), its input x + s u two, and the rows here have unit spread: 55 roundings
    of |n| and 60 of 1, so 64 of |n| + 1; then 128 + 8 roundings of the sum's terms, and half a step of the result."""
    T, C = 131072, 1024
    g = torch.Generator("cuda").manual_seed(5)
    n = lambda *s, d=F32: torch.randn(*s, device="cuda", generator=g).to(d)
    u, x, ds, dy = n(T, C, d=act), n(T, C, d=st), n(T, C, d=st), n(T, C, d=act)
    w, b, s = 1 + 0.1 * n(C), n(C), (0.1 * n(C)).clamp(-0.5, 0.5)

    def check(got, grad, rows, what):
        total, room = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
        for gp, rp in zip(grad.split(1 << 14), rows.split(1 << 14)):
            gp, rp = gp.double(), rp.double()
            mean = rp.mean(1, keepdim=True) if norm == "layer" else 0.0
            hat = (rp - mean) / torch.sqrt(((rp - mean) ** 2).mean(1, keepdim=True) + 1e-5)
            total += (gp * hat).sum(0)
            room += (64 * U * gp.abs() * (hat.abs() + 1) + (128 + 8) * U * (gp * hat).abs()).sum(0)
        worst = float(((got.double() - total).abs() / (room + U * total.abs())).max())
        assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"
    stats = npa.residual_norm_fwd(u, x, None, w, b, None, None, norm=norm, want_stats=True)[2]
    check(npa.residual_norm_bwd(u, x, None, w, b, None, None, stats, ds, None, norm=norm)[3], ds, u, "dpost_weight")
    stats = npa.residual_norm_fwd(u, x, None, None, None, s, w, b, norm=norm, want_stats=True)[2]
    got = npa.residual_norm_bwd(u, x, None, None, None, s, w, stats, None, dy, norm=norm, pre_bias=True)[6]
    check(got, dy, x.double() + s.double() * u.double(), "dpre_weight")
