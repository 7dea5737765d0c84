"""Layer norm over whole rows or over each head's channels, with an optional gate: the norm that stands alone.

:func:`~nanoplm_amd.residual_norm` closes a block and begins the next one; what stands in front of the first block, behind the last one, or between an attention's
heads and its output projection has no residual::

    y = (norm(x) * weight + bias) * silu(gate)            # (weight 1, bias 0, no gate where they are None)

``x`` and ``gate`` ``[T, C]`` may be column slices of wider tensors; with ``heads`` the norm is over each of that many groups of ``C / heads`` adjacent channels,
and ``weight`` and ``bias`` are ``[C]``, or ``[C / heads]`` for all heads. ``norm`` is "layer" or "rms". The backward forms the statistics again from x and gives
every gradient in one kernel, parameters' gradients in a second small one; nothing is stored for it.

The reference's norms are torch's (src/nanoplm/pretraining/models/modern_bert/modeling.py:404-438). All arithmetic runs in hand-written HIP kernels
behind include/nplm_layernorm.h; there is no CPU implementation.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import _lib
from .dwconv import _DTYPES, _launch_on, _ptr
from .padded import _operations_are_recorded
from .recurrence import _refuse_tangents, _row_stride, _rows
from .resnorm import _as, _one_dtype

MAX_GROUP = 16384    # NPLM_LAYERNORM_MAX_GROUP
MAX_HEADS = 65535    # NPLM_LAYERNORM_MAX_HEADS
_NORMS = {"layer": 0, "rms": _lib.LAYERNORM_RMS}


def _check(x, weight, bias, gate, heads, norm, eps):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D tensor [T, C]")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError(f"layer_norm runs only on a ROCm device (x is on {x.device}); there is no CPU implementation")
    T, C = x.shape
    if C < 1 or not 1 <= heads <= MAX_HEADS or C % heads or C // heads > MAX_GROUP:
        raise ValueError(f"1 to {MAX_HEADS} heads must divide rows into groups of 1 to {MAX_GROUP} channels, got {heads} heads of {C} channels")
    if norm not in _NORMS:
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if gate is not None and (gate.shape != x.shape or gate.dtype != x.dtype):
        raise ValueError("gate must match x in shape and dtype")
    if bias is not None and weight is None:
        raise ValueError("a norm's bias needs its weight (pass ones)")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) not in ((C,), (C // heads,)):
            raise ValueError(f"{name} must be [C={C}]" + (f" or [C / heads={C // heads}]" if heads > 1 else "") + f", got {tuple(t.shape)}")
        if t is not None and t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if bias is not None and bias.shape != weight.shape:
        raise ValueError(f"bias must have weight's shape {tuple(weight.shape)}, got {tuple(bias.shape)}")
    for name, t in (("gate", gate), ("weight", weight), ("bias", bias)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} is on {t.device}, x is on {x.device}")
    return T, C


def _flags(weight, C, norm):
    return _NORMS[norm] | (_lib.LAYERNORM_SHARED if weight is not None and weight.shape[0] != C else 0)


def layer_norm_fwd(x, weight=None, bias=None, gate=None, *, heads: int = 1, norm: str = "layer", eps: float = 1e-5) -> torch.Tensor:
    """Raw forward (no autograd)."""
    T, C = _check(x, weight, bias, gate, heads, norm, eps)
    lib = _lib.load()
    (weight, bias), wdt = _one_dtype((weight, bias))
    x, gate = _rows(x), None if gate is None else _rows(gate)
    y = torch.empty((T, C), dtype=x.dtype, device=x.device)
    with _launch_on(x) as dev:
        rc = lib.nplm_layernorm_fwd(_ptr(x), _row_stride(x), _ptr(gate), 0 if gate is None else _row_stride(gate), _ptr(weight), _ptr(bias), float(eps), _ptr(y),
                                    T, C, heads, _DTYPES[x.dtype], _DTYPES[wdt], _flags(weight, C, norm), dev.stream)
    _lib.check(rc, "nplm_layernorm_fwd")
    return y


def layer_norm_bwd(x, weight, bias, gate, dy, *, heads: int = 1, norm: str = "layer", eps: float = 1e-5, want_params: bool = True, grads_bf16: bool = False):
    """Raw backward of :func:`layer_norm_fwd`: ``(dx, dgate, dweight, dbias)`` with None for what the call does not have. Parameters' gradients come in fp32,
    in bf16 with ``grads_bf16``, or not at all without ``want_params``."""
    T, C = _check(x, weight, bias, gate, heads, norm, eps)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must match x in shape, dtype and device")
    lib = _lib.load()
    (weight, bias), wdt = _one_dtype((weight, bias))
    x, dy, gate = _rows(x), _rows(dy), None if gate is None else _rows(gate)
    dx = torch.empty((T, C), dtype=x.dtype, device=x.device)
    dgate = None if gate is None else torch.empty_like(dx)
    gdt = torch.bfloat16 if grads_bf16 else torch.float32
    dweight, dbias = (torch.empty(t.shape, dtype=gdt, device=x.device) if want_params and t is not None else None for t in (weight, bias))
    with _launch_on(x) as dev:
        nbytes = int(lib.nplm_layernorm_bwd_workspace_bytes(T, C, heads)) if dweight is not None else 0
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes else None
        rc = lib.nplm_layernorm_bwd(_ptr(x), _row_stride(x), _ptr(gate), 0 if gate is None else _row_stride(gate), _ptr(dy), _row_stride(dy), _ptr(weight), _ptr(bias),
                                    float(eps), _ptr(dx), _ptr(dgate), _ptr(dweight), _ptr(dbias), _ptr(workspace), nbytes, T, C, heads, _DTYPES[x.dtype],
                                    _DTYPES[wdt], _flags(weight, C, norm) | (_lib.LAYERNORM_GRADS_BF16 if grads_bf16 else 0), dev.stream)
    _lib.check(rc, "nplm_layernorm_bwd")
    return dx, dgate, dweight, dbias


def _grads_bf16(weight, bias):
    return weight is not None and all(t is None or t.dtype == torch.bfloat16 for t in (weight, bias))


class LayerNormFunction(torch.autograd.Function):
    """``apply(x, weight, bias, gate, heads, norm, eps) -> y``."""

    @staticmethod
    def forward(ctx, x, weight, bias, gate, heads, norm, eps):
        ctx.save_for_backward(x, weight, bias, gate)
        ctx.heads, ctx.norm, ctx.eps = heads, norm, eps
        return layer_norm_fwd(x, weight, bias, gate, heads=heads, norm=norm, eps=eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, gate = ctx.saved_tensors
        dx, dgate, dweight, dbias = layer_norm_bwd(x, weight, bias, gate, _as(dy, x), heads=ctx.heads, norm=ctx.norm, eps=ctx.eps,
                                                   want_params=any(ctx.needs_input_grad[1:3]), grads_bf16=_grads_bf16(weight, bias))
        return (dx, None if dweight is None else _as(dweight, weight), None if dbias is None else _as(dbias, bias), dgate, None, None, None)


def layer_norm(x, weight=None, bias=None, *, gate=None, heads: int = 1, norm: str = "layer", eps: float = 1e-5) -> torch.Tensor:
    """Differentiable norm of the module docstring. Where operations are recorded (``torch.compile``, ``torch.jit.trace``, a dispatch mode) the call goes through
    the registered custom ops (same kernels; a recorded launch would be an ``empty`` that nothing fills); otherwise the native node takes it or, for a call that is
    not of its form, leaves it to the Function."""
    if not torch.compiler.is_compiling():
        if norm in _NORMS:
            y = _lib.load_node().layer_norm(x, weight, bias, gate, heads, norm == "rms", eps)
            if y is not None:
                return y
        _refuse_tangents("layer_norm", x, weight, bias, gate)
    if _operations_are_recorded():
        return layer_norm_fwd_op(x, weight, bias, gate, heads, norm, eps)
    return LayerNormFunction.apply(x, weight, bias, gate, heads, norm, eps)


# ---------------------------------------------------------------------------------------------
# torch.library registration, so that a compiled model (src/nanoplm/pretraining/pure_pipeline.py:519-524) keeps one graph. An op returns tensors
# only: what a call does not have is an empty tensor.
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("nanoplm_amd::layer_norm_fwd", mutates_args=(), device_types="cuda")
def layer_norm_fwd_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], gate: Optional[torch.Tensor], heads: int = 1,
                      norm: str = "layer", eps: float = 1e-5) -> torch.Tensor:
    return layer_norm_fwd(x, weight, bias, gate, heads=heads, norm=norm, eps=eps)


@layer_norm_fwd_op.register_fake
def _(x, weight, bias, gate, heads=1, norm="layer", eps=1e-5):
    return x.new_empty(x.shape)


@torch.library.custom_op("nanoplm_amd::layer_norm_bwd", mutates_args=(), device_types="cuda")
def layer_norm_bwd_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], gate: Optional[torch.Tensor], dy: torch.Tensor, heads: int,
                      norm: str, eps: float, want_params: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgate, dweight, dbias), the last two in their parameters' dtypes."""
    dx, dgate, dweight, dbias = layer_norm_bwd(x, weight, bias, gate, dy, heads=heads, norm=norm, eps=eps, want_params=want_params,
                                               grads_bf16=_grads_bf16(weight, bias))
    none = x.new_empty((0,))
    return dx, none if dgate is None else dgate, *(x.new_empty((0,)) if d is None else _as(d, t) for d, t in ((dweight, weight), (dbias, bias)))


@layer_norm_bwd_op.register_fake
def _(x, weight, bias, gate, dy, heads, norm, eps, want_params):
    par = lambda t: torch.empty_like(t) if want_params and t is not None else x.new_empty((0,))
    return x.new_empty(x.shape), x.new_empty((0,) if gate is None else x.shape), par(weight), par(bias)


def _op_setup_context(ctx, inputs, output):
    x, weight, bias, gate, heads, norm, eps = inputs
    ctx.save_for_backward(x, weight, bias, gate)
    ctx.heads, ctx.norm, ctx.eps = heads, norm, eps


def _op_backward(ctx, dy):
    x, weight, bias, gate = ctx.saved_tensors
    want = any(ctx.needs_input_grad[1:3])
    dx, dgate, dweight, dbias = layer_norm_bwd_op(x, weight, bias, gate, _as(dy, x), ctx.heads, ctx.norm, ctx.eps, want)
    return (dx, dweight if want and weight is not None else None, dbias if want and bias is not None else None, None if gate is None else dgate, None, None, None)


layer_norm_fwd_op.register_autograd(_op_backward, setup_context=_op_setup_context)


class LayerNorm(nn.Module):
    """``forward(x, gate=None)`` with the parameters of :func:`layer_norm`: ``weight`` (and ``bias``) ``[channels]``, or ``[channels / heads]`` for all heads with
    ``shared``. All parameters are 1-D, which the reference's grouping rules send to AdamW without weight decay (src/nanoplm/pretraining/optim.py:43-51,
    src/nanoplm/pretraining/pure_pipeline.py:68-76)."""

    def __init__(self, channels: int, heads: int = 1, norm: str = "layer", bias: bool = False, shared: bool = False, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        if channels < 1 or not 1 <= heads <= MAX_HEADS or channels % heads or channels // heads > MAX_GROUP:
            raise ValueError(f"1 to {MAX_HEADS} heads must divide channels into groups of 1 to {MAX_GROUP}, got {heads} and {channels}")
        if norm not in _NORMS:
            raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
        self.channels, self.heads, self.norm, self.eps = channels, heads, norm, eps
        n = channels // heads if shared else channels
        self.weight = nn.Parameter(torch.empty((n,), device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty((n,), device=device, dtype=dtype)) if bias else None
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        self.weight.fill_(1.0)
        if self.bias is not None:
            self.bias.fill_(0.0)

    def forward(self, x, gate=None):
        return layer_norm(x, self.weight, self.bias, gate=gate, heads=self.heads, norm=self.norm, eps=self.eps)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, heads={self.heads}, norm={self.norm}, bias={self.bias is not None}, shared={self.weight.shape[0] != self.channels}, eps={self.eps}"
