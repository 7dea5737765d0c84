"""Forms of call of the recurrence, its step and the residual norm that the block's own tests do not make: forward mode."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import nanoplm_amd as npa

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _inputs(T=300, C=70, act=F32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s, d=act: torch.randn(*s, device="cuda", generator=g).to(d)
    return dict(x=n(T, C), gates=n(T, 2 * C), cu=torch.tensor([0, 100, 100, T], dtype=torch.int32, device="cuda"), decay=n(C, d=F32) - 4, h0=n(3, C, d=F32),
                gate=n(T, C), weight=n(C, d=F32), table=n(T + 5, C, d=F32))


def _calls(i, table=None):
    table = i["table"].clone() if table is None else table
    return {"recurrence": lambda: npa.varlen_recurrence(i["x"], i["gates"], i["cu"], i["decay"], initial_state=i["h0"], return_state=True),
            "norm": lambda: npa.residual_norm(i["x"], i["x"], i["gate"], pre_weight=i["weight"]),
            "step": lambda: (npa.recurrence_step(i["x"], i["gates"], i["decay"], table),)}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["recurrence", "norm", "step"])
def test_forward_mode_is_refused(name, grad):
    i = _inputs()
    for which in ("x", "gates", "decay", "h0", "gate", "weight"):
        used = {"recurrence": ("x", "gates", "decay", "h0"), "norm": ("x", "gate", "weight"), "step": ("x", "gates", "decay")}[name]
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            call = _calls({**i, which: forward_ad.make_dual(i[which], torch.ones_like(i[which]))})[name]
            if which in used:
                with pytest.raises(NotImplementedError):
                    call()
            else:
                call()
    want, (got,) = _calls(i)[name](), [None]
    with forward_ad.dual_level():
        got = _calls(i)[name]()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
