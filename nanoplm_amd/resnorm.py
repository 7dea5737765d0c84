"""The end of a block fused with the norm in front of the next one.

In a pre-norm layer (src/nanoplm/pretraining/models/modern_bert/modeling.py:404-438) a sub-module's output is added to the residual stream and the
next sub-module begins with a norm of it. ``residual_norm`` is everything between the two, in one pass over the rows::

    v      = norm(u) * post_weight + post_bias        # (u itself without post_weight)
    v      = v * silu(gate)                           # (with gate)
    stream = residual + scale * v                     # (scale [C]; 1 without it)
    normed = norm(stream) * pre_weight + pre_bias     # (None without pre_weight)

``u`` and ``gate`` ``[T, C]`` may be column slices of wider tensors. ``residual`` has their dtype, or fp32 beside bf16 branches (what
``torch.autocast`` leaves); ``stream`` has residual's dtype, ``normed`` has u's. ``norm`` is "layer" or "rms". The backward reads the forward's inputs
once and writes every gradient in one kernel, parameters' gradients in a second small one; nothing normalised or gated is stored.

All arithmetic runs in hand-written HIP kernels behind include/nplm_resnorm.h; there is no CPU implementation.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib
from .dwconv import _DTYPES, _launch_on, _ptr
from .padded import _operations_are_recorded
from .recurrence import _dense, _refuse_tangents, _row_stride, _rows

MAX_CHANNELS = 16384    # NPLM_RESNORM_MAX_C
_NORMS = {"layer": 0, "rms": _lib.RESNORM_RMS}


def _check(u, residual, gate, params, norm, eps):
    """Shape, dtype and device checks shared by forward and backward. ``params``: the five parameters, in order."""
    if not isinstance(u, torch.Tensor) or u.dim() != 2:
        raise ValueError("u must be a 2-D tensor [T, C]")
    if u.dtype not in _DTYPES:
        raise TypeError(f"u must be float32 or bfloat16, got {u.dtype}")
    if not u.is_cuda:
        raise RuntimeError(f"residual_norm runs only on a ROCm device (u is on {u.device}); there is no CPU implementation")
    T, C = u.shape
    if not 1 <= C <= MAX_CHANNELS:
        raise ValueError(f"rows of 1 to {MAX_CHANNELS} channels, got {C}")
    if norm not in _NORMS:
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if not isinstance(residual, torch.Tensor) or residual.shape != u.shape:
        raise ValueError(f"residual must be [T={T}, C={C}]")
    if residual.dtype != u.dtype and not (residual.dtype == torch.float32 and u.dtype == torch.bfloat16):
        raise TypeError(f"residual must have u's dtype {u.dtype}, or float32 beside bfloat16, got {residual.dtype}")
    if gate is not None and (gate.shape != u.shape or gate.dtype != u.dtype):
        raise ValueError("gate must match u in shape and dtype")
    names = ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")
    for name, t in zip(names, params):
        if t is not None and tuple(t.shape) != (C,):
            raise ValueError(f"{name} must be [C={C}], got {tuple(t.shape)}")
        if t is not None and t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    post_weight, post_bias, _, pre_weight, pre_bias = params
    if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
        raise ValueError("a norm's bias needs its weight (pass ones)")
    for name, t in (("residual", residual), ("gate", gate)) + tuple(zip(names, params)):
        if t is not None and t.device != u.device:
            raise RuntimeError(f"{name} is on {t.device}, u is on {u.device}")
    return T, C


def _one_dtype(params):
    """The parameters in the one dtype that the kernels take them in: theirs where they share it, else fp32 (no parameter is rounded)."""
    dtypes = {t.dtype for t in params if t is not None}
    dt = dtypes.pop() if len(dtypes) == 1 else torch.float32
    return [None if t is None else _dense(t.to(dt)) for t in params], dt


def residual_norm_fwd(u, residual, gate=None, post_weight=None, post_bias=None, scale=None, pre_weight=None, pre_bias=None, *, norm: str = "layer",
                      eps: float = 1e-5, want_stats: bool = False):
    """Raw forward (no autograd): ``(stream, normed, stats)``; normed None without ``pre_weight``, stats ``[T, 4]`` fp32 for
    :func:`residual_norm_bwd` (None unless wanted)."""
    params = (post_weight, post_bias, scale, pre_weight, pre_bias)
    T, C = _check(u, residual, gate, params, norm, eps)
    lib = _lib.load()
    params, wdt = _one_dtype(params)
    u, residual, gate = _rows(u), _rows(residual), None if gate is None else _rows(gate)
    stream = torch.empty((T, C), dtype=residual.dtype, device=u.device)
    normed = None if pre_weight is None else torch.empty((T, C), dtype=u.dtype, device=u.device)
    stats = torch.empty((T, 4), dtype=torch.float32, device=u.device) if want_stats else None
    with _launch_on(u) as dev:
        rc = lib.nplm_resnorm_fwd(_ptr(u), _row_stride(u), _ptr(gate), 0 if gate is None else _row_stride(gate), _ptr(residual), _row_stride(residual),
                                  *map(_ptr, params), float(eps), _ptr(stream), _ptr(normed), _ptr(stats), T, C, _DTYPES[u.dtype],
                                  _DTYPES[residual.dtype], _DTYPES[wdt], _NORMS[norm], dev.stream)
    _lib.check(rc, "nplm_resnorm_fwd")
    return stream, normed, stats


def residual_norm_bwd(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats, dstream, dnormed, *, norm: str = "layer",
                      pre_bias: bool = False, want_params: bool = True, grads_bf16: bool = False):
    """Raw backward of :func:`residual_norm_fwd`: ``(du, dresidual, dgate, dpost_weight, dpost_bias, dscale, dpre_weight, dpre_bias)`` with None for what
    the call does not have (``pre_bias``: whether it had that one). Either of ``dstream`` and ``dnormed`` may be None. Parameters' gradients come in fp32, in
    bf16 with ``grads_bf16``, or not at all without ``want_params``."""
    T, C = _check(u, residual, gate, (post_weight, post_bias, scale, pre_weight, None), norm, 0.0)
    for name, t, like in (("dstream", dstream, residual), ("dnormed", dnormed, u)):
        if t is not None and (t.shape != u.shape or t.dtype != like.dtype or t.device != u.device):
            raise ValueError(f"{name} must be [T={T}, C={C}] {like.dtype} on {u.device}")
    if dnormed is not None and pre_weight is None:
        raise ValueError("dnormed needs pre_weight")
    if stats is None or tuple(stats.shape) != (T, 4) or stats.dtype != torch.float32 or stats.device != u.device:
        raise ValueError(f"stats must be the forward's [T={T}, 4] fp32")
    lib = _lib.load()
    (post_weight, post_bias, scale, pre_weight), wdt = _one_dtype((post_weight, post_bias, scale, pre_weight))
    u, residual, stats = _rows(u), _rows(residual), _dense(stats)
    gate, dstream, dnormed = (None if t is None else _rows(t) for t in (gate, dstream, dnormed))
    du, dresidual = torch.empty((T, C), dtype=u.dtype, device=u.device), torch.empty((T, C), dtype=residual.dtype, device=u.device)
    dgate = None if gate is None else torch.empty_like(du)
    gdt = torch.bfloat16 if grads_bf16 else torch.float32
    has = (post_weight is not None, post_bias is not None, scale is not None, pre_weight is not None, pre_bias)
    grads = [torch.empty((C,), dtype=gdt, device=u.device) if want_params and h else None for h in has]
    stride = lambda t: 0 if t is None else _row_stride(t)
    with _launch_on(u) as dev:
        nbytes = int(lib.nplm_resnorm_bwd_workspace_bytes(T, C)) if any(t is not None for t in grads) else 0
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=u.device) if nbytes else None
        rc = lib.nplm_resnorm_bwd(_ptr(u), _row_stride(u), _ptr(gate), stride(gate), _ptr(residual), _row_stride(residual), _ptr(dstream), stride(dstream),
                                  _ptr(dnormed), stride(dnormed), _ptr(stats), _ptr(post_weight), _ptr(post_bias), _ptr(scale), _ptr(pre_weight),
                                  _ptr(du), _ptr(dgate), _ptr(dresidual), *map(_ptr, grads), _ptr(workspace), nbytes, T, C, _DTYPES[u.dtype],
                                  _DTYPES[residual.dtype], _DTYPES[wdt], _NORMS[norm] | (_lib.RESNORM_GRADS_BF16 if grads_bf16 else 0), dev.stream)
    _lib.check(rc, "nplm_resnorm_bwd")
    return (du, dresidual, dgate, *grads)


def _as(t: Optional[torch.Tensor], like: torch.Tensor) -> Optional[torch.Tensor]:
    return t if t is None or t.dtype == like.dtype else t.to(like.dtype)


class ResidualNormFunction(torch.autograd.Function):
    """``apply(u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, eps) -> (stream, normed)``; normed is None without
    pre_weight."""

    @staticmethod
    def forward(ctx, u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, eps):
        stream, normed, stats = residual_norm_fwd(u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm=norm, eps=eps,
                                                  want_stats=any(ctx.needs_input_grad))
        ctx.save_for_backward(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats)
        ctx.norm, ctx.pre_bias_dtype = norm, None if pre_bias is None else pre_bias.dtype
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dstream, dnormed):
        u, residual, gate, post_weight, post_bias, scale, pre_weight, stats = ctx.saved_tensors
        dtypes = [None if t is None else t.dtype for t in (post_weight, post_bias, scale, pre_weight)] + [ctx.pre_bias_dtype]
        grads = residual_norm_bwd(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats, _as(dstream, residual), _as(dnormed, u),
                                  norm=ctx.norm, pre_bias=ctx.pre_bias_dtype is not None, want_params=any(ctx.needs_input_grad[3:8]),
                                  grads_bf16=all(d in (None, torch.bfloat16) for d in dtypes))
        params = [None if g is None else g.to(d) for g, d in zip(grads[3:], dtypes)]
        return (*grads[:3], *params, None, None)


def residual_norm(u, residual, gate=None, post_weight=None, post_bias=None, scale=None, pre_weight=None, pre_bias=None, *, norm: str = "layer",
                  eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Differentiable ``(stream, normed)`` of the module docstring. Where operations are recorded (``torch.compile``, ``torch.jit.trace``, a dispatch
    mode) the call goes through the registered custom ops (same kernels; a recorded launch would be an ``empty`` that nothing fills); otherwise the native
    node takes it or, for a call that is not of its form, leaves it to the Function."""
    args = (u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias)
    if not torch.compiler.is_compiling():
        if norm in _NORMS:
            out = _lib.load_node().residual_norm(*args, norm == "rms", eps)
            if out is not None:
                return out
        _refuse_tangents("residual_norm", *args)
    if _operations_are_recorded():
        stream, normed, _ = residual_norm_fwd_op(*args, norm, eps)
        return stream, None if pre_weight is None else normed
    return ResidualNormFunction.apply(*args, norm, eps)


# ---------------------------------------------------------------------------------------------
# torch.library registration, so that a compiled model (src/nanoplm/pretraining/pure_pipeline.py:519-524) keeps one graph. An op returns tensors
# only: what a call does not have is an empty tensor.
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("nanoplm_amd::residual_norm_fwd", mutates_args=(), device_types="cuda")
def residual_norm_fwd_op(u: torch.Tensor, residual: torch.Tensor, gate: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                         post_bias: Optional[torch.Tensor], scale: Optional[torch.Tensor], pre_weight: Optional[torch.Tensor],
                         pre_bias: Optional[torch.Tensor], norm: str = "layer",
                         eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(stream, normed, stats)."""
    stream, normed, stats = residual_norm_fwd(u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm=norm, eps=eps, want_stats=True)
    return stream, u.new_empty((0,)) if normed is None else normed, stats


@residual_norm_fwd_op.register_fake
def _(u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm="layer", eps=1e-5):
    T, C = u.shape
    return residual.new_empty((T, C)), u.new_empty((0,) if pre_weight is None else (T, C)), u.new_empty((T, 4), dtype=torch.float32)


@torch.library.custom_op("nanoplm_amd::residual_norm_bwd", mutates_args=(), device_types="cuda")
def residual_norm_bwd_op(u: torch.Tensor, residual: torch.Tensor, gate: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                         post_bias: Optional[torch.Tensor], scale: Optional[torch.Tensor], pre_weight: Optional[torch.Tensor], stats: torch.Tensor,
                         dstream: Optional[torch.Tensor], dnormed: Optional[torch.Tensor], norm: str, pre_bias: bool,
                         grads_bf16: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                                    torch.Tensor]:
    """(du, dresidual, dgate, dpost_weight, dpost_bias, dscale, dpre_weight, dpre_bias)."""
    grads = residual_norm_bwd(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats, dstream, dnormed, norm=norm, pre_bias=pre_bias,
                              grads_bf16=grads_bf16)
    return tuple(u.new_empty((0,)) if g is None else g for g in grads)


@residual_norm_bwd_op.register_fake
def _(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats, dstream, dnormed, norm, pre_bias, grads_bf16):
    T, C = u.shape
    par = lambda there: u.new_empty((C,), dtype=torch.bfloat16 if grads_bf16 else torch.float32) if there else u.new_empty((0,))
    return (u.new_empty((T, C)), residual.new_empty((T, C)), u.new_empty((0,) if gate is None else (T, C)), par(post_weight is not None),
            par(post_bias is not None), par(scale is not None), par(pre_weight is not None), par(pre_bias))


def _op_setup_context(ctx, inputs, output):
    u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, norm, _ = inputs
    ctx.save_for_backward(u, residual, gate, post_weight, post_bias, scale, pre_weight, output[2])
    ctx.norm, ctx.pre_bias_dtype = norm, None if pre_bias is None else pre_bias.dtype
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dstream, dnormed, _dstats):
    u, residual, gate, post_weight, post_bias, scale, pre_weight, stats = ctx.saved_tensors
    dtypes = [None if t is None else t.dtype for t in (post_weight, post_bias, scale, pre_weight)] + [ctx.pre_bias_dtype]
    dnormed = None if pre_weight is None else _as(dnormed, u)
    grads = residual_norm_bwd_op(u, residual, gate, post_weight, post_bias, scale, pre_weight, stats, _as(dstream, residual), dnormed, ctx.norm,
                                 ctx.pre_bias_dtype is not None, all(d in (None, torch.bfloat16) for d in dtypes))
    params = [None if d is None else g.to(d) for g, d in zip(grads[3:], dtypes)]
    return (grads[0], grads[1], None if gate is None else grads[2], *params, None, None)


residual_norm_fwd_op.register_autograd(_op_backward, setup_context=_op_setup_context)


class ResidualNorm(nn.Module):
    """``forward(u, residual, gate=None) -> (stream, normed)`` with the parameters of :func:`residual_norm`.

    ``post`` and ``pre`` choose the norms (a module without ``pre`` returns None for normed: the end of the last block), ``bias`` their biases,
    ``scale_init`` the residual scale's first value (None: no scale; 0 makes the block begin as the identity). All parameters are 1-D, which the reference's
    grouping rules send to AdamW without weight decay (src/nanoplm/pretraining/optim.py:43-51, src/nanoplm/pretraining/pure_pipeline.py:68-76)."""

    def __init__(self, channels: int, norm: str = "layer", post: bool = True, pre: bool = True, bias: bool = False, scale_init: Optional[float] = None,
                 eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        if not 1 <= channels <= MAX_CHANNELS:
            raise ValueError(f"channels must lie in 1 .. {MAX_CHANNELS}, got {channels}")
        if norm not in _NORMS:
            raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
        self.channels, self.norm, self.eps, self.scale_init = channels, norm, eps, scale_init
        make = lambda there: nn.Parameter(torch.empty((channels,), device=device, dtype=dtype)) if there else None
        self.post_weight, self.post_bias = make(post), make(post and bias)
        self.scale = make(scale_init is not None)
        self.pre_weight, self.pre_bias = make(pre), make(pre and bias)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        for t, value in ((self.post_weight, 1.0), (self.post_bias, 0.0), (self.scale, self.scale_init), (self.pre_weight, 1.0), (self.pre_bias, 0.0)):
            if t is not None:
                t.fill_(value)

    def forward(self, u, residual, gate=None):
        return residual_norm(u, residual, gate, self.post_weight, self.post_bias, self.scale, self.pre_weight, self.pre_bias, norm=self.norm, eps=self.eps)

    def extra_repr(self) -> str:
        return (f"channels={self.channels}, norm={self.norm}, post={self.post_weight is not None}, pre={self.pre_weight is not None}, "
                f"bias={self.post_bias is not None or self.pre_bias is not None}, scale_init={self.scale_init}, eps={self.eps}")
