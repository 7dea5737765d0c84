"""Gated linear recurrence over packed sequences: the long-range partner of the depthwise conv, on the same ``[T, C]`` rows.

Per channel, from each sequence's first row to its last one (from the last to the first with ``reverse``)::

    a_t = exp(-scale * softplus(decay) * sigmoid(r_t))
    h_t = a_t * h_{t-1} + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t          y = h

``gates`` ``[T, 2C]`` holds r in columns ``[0, C)`` and i in ``[C, 2C)``: one projection gives both. ``x`` and ``gates`` may be column
slices of wider tensors (any row stride, adjacent elements). Sequences begin with zeros or with ``initial_state`` ``[S, C]`` and end with a state that
``return_state`` hands out, so that a long sequence can be run in pieces and a prompt be continued token by token with :func:`recurrence_step`.
States are fp32 whatever the activations' dtype is.

The reference's packed path (src/nanoplm/pretraining/models/modern_bert/modeling.py:421-439) hands its sub-modules ``x:[total_tokens, hidden]`` and
int32 ``cu_seqlens``; it has no recurrence to replace. All arithmetic runs in hand-written HIP kernels behind include/nplm_recurrence.h; there is
no CPU implementation.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as forward_ad
from torch import nn

from . import _lib
from .dwconv import _DTYPES, _launch_on, _ptr
from .padded import _operations_are_recorded

CHUNK = 32              # NPLM_RECURRENCE_CHUNK
MAX_SLOTS = 1 << 18     # NPLM_RECURRENCE_MAX_SLOTS


def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t's values one behind the other: a contiguous copy of strided tensors and of views that negate their values when they are read."""
    return None if t is None else t.resolve_neg().contiguous()


def _plain(t: torch.Tensor) -> bool:
    return t.is_contiguous() and not t.is_neg()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where its rows are runs of adjacent elements, one behind the other without overlap; else a contiguous copy."""
    t = t.resolve_neg()
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])         # (of a single row, any)


def _refuse_tangents(name: str, *tensors) -> None:
    """The kernels carry no tangents. (An autograd Function without a rule for them says so itself; a registered op would drop them.)"""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _check_rows(x, gates, decay, name):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D tensor [T, C] of packed tokens")
    if x.dtype not in _DTYPES:
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError(f"{name} runs only on a ROCm device (x is on {x.device}); there is no CPU implementation")
    T, C = x.shape
    if C < 1:
        raise ValueError("x must have at least one channel")
    if not isinstance(gates, torch.Tensor) or tuple(gates.shape) != (T, 2 * C):
        raise ValueError(f"gates must be [T={T}, 2C={2 * C}]: recurrence-gate columns followed by input-gate columns")
    if gates.dtype != x.dtype:
        raise TypeError(f"gates must have x's dtype {x.dtype}, got {gates.dtype}")
    if tuple(decay.shape) != (C,):
        raise ValueError(f"decay must be [C={C}], got {tuple(decay.shape)}")
    if decay.dtype not in _DTYPES:
        raise TypeError(f"decay must be float32 or bfloat16, got {decay.dtype}")
    for what, t in (("gates", gates), ("decay", decay)):
        if t.device != x.device:
            raise RuntimeError(f"{what} is on {t.device}, x is on {x.device}")
    return T, C


def _check_scale(scale):
    if not 0.0 < float(scale) < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")


def _check_state(t, rows, C, device, name):
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != (rows, C) or t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 [{rows}, C={C}]")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, x is on {device}")


def _check(x, gates, cu_seqlens, decay, scale, initial_state):
    T, C = _check_rows(x, gates, decay, "varlen_recurrence")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise TypeError("cu_seqlens must be a 1-D int32 tensor with at least one entry")
    if cu_seqlens.device != x.device:
        raise RuntimeError(f"cu_seqlens is on {cu_seqlens.device}, x is on {x.device}")
    S = cu_seqlens.numel() - 1
    _check_scale(scale)
    _check_state(initial_state, S, C, x.device, "initial_state")
    return T, C, S


def varlen_recurrence_fwd(x, gates, cu_seqlens, decay, *, scale: float = 8.0, initial_state: Optional[torch.Tensor] = None,
                          reverse: bool = False, want_state: bool = False, want_carries: bool = False):
    """Raw forward (no autograd): ``(y, state, carries)``: y in x's dtype, state ``[S, C]`` and carries ``[ceil(T / 32), C]`` in fp32 (None
    unless wanted). The carries are what :func:`varlen_recurrence_bwd` restarts the recurrence from."""
    T, C, S = _check(x, gates, cu_seqlens, decay, scale, initial_state)
    lib = _lib.load()
    x, gates, cu_seqlens, decay = _rows(x), _rows(gates), _dense(cu_seqlens), _dense(decay)
    initial_state = _dense(initial_state)
    act = _DTYPES[x.dtype]
    y = torch.empty((T, C), dtype=x.dtype, device=x.device)
    state = torch.empty((S, C), dtype=torch.float32, device=x.device) if want_state else None
    carries = torch.empty((-(-T // CHUNK), C), dtype=torch.float32, device=x.device) if want_carries else None
    with _launch_on(x) as dev:
        nbytes = int(lib.nplm_recurrence_fwd_workspace_bytes(T, C, S, act))
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes else None
        rc = lib.nplm_recurrence_fwd(_ptr(x), _row_stride(x), _ptr(gates), _row_stride(gates), _ptr(cu_seqlens), _ptr(decay), float(scale),
                                     _ptr(initial_state), _ptr(y), _ptr(state), _ptr(carries), _ptr(workspace), nbytes, T, C, S, act,
                                     _DTYPES[decay.dtype], _lib.RECURRENCE_REVERSE if reverse else 0, dev.stream)
    _lib.check(rc, "nplm_recurrence_fwd")
    return y, state, carries


def varlen_recurrence_bwd(x, gates, dy, cu_seqlens, decay, carries, *, scale: float = 8.0, initial_state: Optional[torch.Tensor] = None,
                          dstate: Optional[torch.Tensor] = None, reverse: bool = False, want_dinitial: bool = False, grads_bf16: bool = False):
    """Raw backward of :func:`varlen_recurrence_fwd`: ``(dx, dgates, ddecay, dinitial)``; dx and dgates in x's dtype, ddecay in fp32 (in bf16, rounded once, with
    ``grads_bf16``), dinitial ``[S, C]`` in fp32 (None unless wanted). ``carries`` are the forward's, ``dstate`` the gradient of its state."""
    T, C, S = _check(x, gates, cu_seqlens, decay, scale, initial_state)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != x.device:
        raise ValueError("dy must match x in shape, dtype and device")
    _check_state(carries, -(-T // CHUNK), C, x.device, "carries")
    _check_state(dstate, S, C, x.device, "dstate")
    if carries is None:
        raise ValueError("carries must be the forward's (want_carries)")
    lib = _lib.load()
    x, gates, dy, cu_seqlens, decay, carries = _rows(x), _rows(gates), _rows(dy), _dense(cu_seqlens), _dense(decay), _dense(carries)
    initial_state, dstate = _dense(initial_state), _dense(dstate)
    act = _DTYPES[x.dtype]
    dx = torch.empty((T, C), dtype=x.dtype, device=x.device)
    dgates = torch.empty((T, 2 * C), dtype=x.dtype, device=x.device)
    ddecay = torch.empty((C,), dtype=torch.bfloat16 if grads_bf16 else torch.float32, device=x.device)
    dinitial = torch.empty((S, C), dtype=torch.float32, device=x.device) if want_dinitial else None
    with _launch_on(x) as dev:
        nbytes = int(lib.nplm_recurrence_bwd_workspace_bytes(T, C, S, act))
        workspace = torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes else None
        rc = lib.nplm_recurrence_bwd(_ptr(x), _row_stride(x), _ptr(gates), _row_stride(gates), _ptr(dy), _row_stride(dy), _ptr(cu_seqlens),
                                     _ptr(decay), float(scale), _ptr(initial_state), _ptr(dstate), _ptr(carries), _ptr(dx), _ptr(dgates),
                                     _ptr(ddecay), _ptr(dinitial), _ptr(workspace), nbytes, T, C, S, act, _DTYPES[decay.dtype],
                                     (_lib.RECURRENCE_REVERSE if reverse else 0) | (_lib.RECURRENCE_GRADS_BF16 if grads_bf16 else 0), dev.stream)
    _lib.check(rc, "nplm_recurrence_bwd")
    return dx, dgates, ddecay, dinitial


def recurrence_step(x, gates, decay, state, slots: Optional[torch.Tensor] = None, *, scale: float = 8.0,
                    out_state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B sequences: y ``[B, C]`` in x's dtype. No gradients.

    ``state`` is a table ``[N, C]`` of fp32 states; row b of ``x`` ``[B, C]`` and ``gates`` ``[B, 2C]`` belongs to the state in row ``slots[b]`` (int32;
    row b without ``slots``), which is replaced by the new one, or, with ``out_state``, another table of the same size, left as it is and the new one
    written there (tokens that may be taken back; no memory shared with ``state``). Rows of ``out_state`` that no slot names are left alone. Rows that name the same slot are consecutive
    tokens of one sequence, in their order. A slot outside ``[0, N)`` marks a padding row: y is 0 and no state is touched. Time grows with the square of the rows
    that name slots (2^18 at most): from some thousands on they are better given in pieces."""
    if not torch.compiler.is_compiling():
        y = _lib.load_node().recurrence_step(x, gates, decay, state, slots, scale, out_state)
        if y is not None:
            return y
        _refuse_step_gradients(x, gates, decay, state, out_state)
    if _operations_are_recorded():
        if out_state is None or out_state is state:
            return recurrence_step_op(x, gates, decay, state, slots, scale)
        return recurrence_step_to_op(x, gates, decay, state, slots, scale, out_state)
    return _step(x, gates, decay, state, slots, scale, out_state)


def _refuse_step_gradients(*tensors):
    _refuse_tangents("recurrence_step", *tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError("recurrence_step has no gradient: call it under torch.no_grad(), or use varlen_recurrence")


def _step(x, gates, decay, state, slots, scale, out_state):
    """:func:`recurrence_step` at once, through ctypes."""
    B, C = _check_rows(x, gates, decay, "recurrence_step")
    _check_scale(scale)
    if not isinstance(state, torch.Tensor) or state.dim() != 2 or state.shape[1] != C or state.dtype != torch.float32 or not _plain(state):
        raise ValueError(f"state must be a contiguous float32 table [N, C={C}]")
    out_state = state if out_state is None else out_state
    if out_state.shape != state.shape or out_state.dtype != torch.float32 or not _plain(out_state):
        raise ValueError("out_state must be a contiguous float32 table of state's shape")
    if 0 < abs(out_state.data_ptr() - state.data_ptr()) < 4 * state.numel():
        raise ValueError("out_state must be state itself or a table apart from it: it shares some of its memory")
    for what, t in (("state", state), ("out_state", out_state), ("slots", slots)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{what} is on {t.device}, x is on {x.device}")
    N = state.shape[0]
    if slots is not None and (slots.dtype != torch.int32 or tuple(slots.shape) != (B,)):
        raise TypeError(f"slots must be int32 [B={B}]")
    if slots is not None and B > MAX_SLOTS:
        raise ValueError(f"at most {MAX_SLOTS} rows a step with slots, got {B}: every row looks through all of them")
    if slots is None and B > N:
        raise ValueError(f"{B} rows need as many states, the table has {N} (or pass slots)")
    lib = _lib.load()
    x, gates, decay, slots = _rows(x), _rows(gates), _dense(decay), _dense(slots)
    y = torch.empty((B, C), dtype=x.dtype, device=x.device)
    if not out_state.is_inference():
        torch.autograd.graph.increment_version(out_state)
    with _launch_on(x) as dev:
        rc = lib.nplm_recurrence_step(_ptr(x), _row_stride(x), _ptr(gates), _row_stride(gates), _ptr(decay), float(scale), _ptr(state),
                                      _ptr(out_state), _ptr(slots), _ptr(y), B, C, N, _DTYPES[x.dtype], _DTYPES[decay.dtype], dev.stream)
    _lib.check(rc, "nplm_recurrence_step")
    return y


class VarlenRecurrenceFunction(torch.autograd.Function):
    """``apply(x, gates, cu_seqlens, decay, initial_state, scale, reverse, return_state) -> (y, state)``; gradients for x, gates, decay and
    initial_state. state is None without ``return_state``."""

    @staticmethod
    def forward(ctx, x, gates, cu_seqlens, decay, initial_state=None, scale=8.0, reverse=False, return_state=False):
        y, state, carries = varlen_recurrence_fwd(x, gates, cu_seqlens, decay, scale=scale, initial_state=initial_state, reverse=reverse,
                                                  want_state=return_state, want_carries=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, gates, cu_seqlens, decay, initial_state, carries)
        ctx.scale, ctx.reverse = scale, reverse
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        x, gates, cu_seqlens, decay, initial_state, carries = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy if dy.dtype == x.dtype else dy.to(x.dtype)
        dx, dgates, ddecay, dinitial = varlen_recurrence_bwd(x, gates, dy, cu_seqlens, decay, carries, scale=ctx.scale, initial_state=initial_state,
                                                             dstate=dstate, reverse=ctx.reverse, want_dinitial=initial_state is not None and ctx.needs_input_grad[4],
                                                             grads_bf16=decay.dtype == torch.bfloat16)
        return dx, dgates, None, ddecay, dinitial, None, None, None


def varlen_recurrence(x, gates, cu_seqlens, decay, *, scale: float = 8.0, initial_state: Optional[torch.Tensor] = None, reverse: bool = False,
                      return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Differentiable gated linear recurrence over packed sequences: y, or ``(y, state)`` with ``return_state`` (see the module docstring). Where
    operations are recorded (``torch.compile``, ``torch.jit.trace``, a dispatch mode) the call goes through the registered custom ops (same kernels; a
    recorded launch would be an ``empty`` that nothing fills); otherwise the native node takes it or, for a call that is not of its form, leaves it to the
    Function."""
    if not torch.compiler.is_compiling():
        out = _lib.load_node().recurrence(x, gates, cu_seqlens, decay, initial_state, scale, reverse, return_state)
        if out is not None:
            return out if return_state else out[0]
        _refuse_tangents("varlen_recurrence", x, gates, decay, initial_state)
    if _operations_are_recorded():
        y, state, _ = varlen_recurrence_fwd_op(x, gates, cu_seqlens, decay, initial_state, scale, reverse)
        return (y, state) if return_state else y
    y, state = VarlenRecurrenceFunction.apply(x, gates, cu_seqlens, decay, initial_state, scale, reverse, return_state)
    return (y, state) if return_state else y


# ---------------------------------------------------------------------------------------------
# torch.library registration, so that a compiled model (src/nanoplm/pretraining/pure_pipeline.py:519-524) keeps one graph.
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("nanoplm_amd::varlen_recurrence_fwd", mutates_args=(), device_types="cuda")
def varlen_recurrence_fwd_op(x: torch.Tensor, gates: torch.Tensor, cu_seqlens: torch.Tensor, decay: torch.Tensor,
                             initial_state: Optional[torch.Tensor], scale: float = 8.0,
                             reverse: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, state, carries)."""
    return varlen_recurrence_fwd(x, gates, cu_seqlens, decay, scale=scale, initial_state=initial_state, reverse=reverse, want_state=True,
                                 want_carries=True)


@varlen_recurrence_fwd_op.register_fake
def _(x, gates, cu_seqlens, decay, initial_state, scale=8.0, reverse=False):
    T, C = x.shape
    f = lambda n: x.new_empty((n, C), dtype=torch.float32)
    return x.new_empty((T, C)), f(cu_seqlens.shape[0] - 1), f((T + CHUNK - 1) // CHUNK)


@torch.library.custom_op("nanoplm_amd::varlen_recurrence_bwd", mutates_args=(), device_types="cuda")
def varlen_recurrence_bwd_op(x: torch.Tensor, gates: torch.Tensor, dy: torch.Tensor, cu_seqlens: torch.Tensor, decay: torch.Tensor,
                             carries: torch.Tensor, initial_state: Optional[torch.Tensor], dstate: Optional[torch.Tensor], scale: float = 8.0,
                             reverse: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgates, ddecay in decay's dtype, dinitial)."""
    return varlen_recurrence_bwd(x, gates, dy, cu_seqlens, decay, carries, scale=scale, initial_state=initial_state, dstate=dstate, reverse=reverse,
                                 want_dinitial=True, grads_bf16=decay.dtype == torch.bfloat16)


@varlen_recurrence_bwd_op.register_fake
def _(x, gates, dy, cu_seqlens, decay, carries, initial_state, dstate, scale=8.0, reverse=False):
    T, C = x.shape
    return x.new_empty((T, C)), x.new_empty((T, 2 * C)), torch.empty_like(decay), x.new_empty((cu_seqlens.shape[0] - 1, C), dtype=torch.float32)


def _op_setup_context(ctx, inputs, output):
    x, gates, cu_seqlens, decay, initial_state, scale, reverse = inputs
    ctx.save_for_backward(x, gates, cu_seqlens, decay, initial_state, output[2])
    ctx.scale, ctx.reverse = scale, bool(reverse)
    ctx.set_materialize_grads(False)


def _op_backward(ctx, dy, dstate, _dcarries):
    x, gates, cu_seqlens, decay, initial_state, carries = ctx.saved_tensors
    dy = torch.zeros_like(x) if dy is None else dy if dy.dtype == x.dtype else dy.to(x.dtype)
    dx, dgates, ddecay, dinitial = varlen_recurrence_bwd_op(x, gates, dy, cu_seqlens, decay, carries, initial_state, dstate, ctx.scale, ctx.reverse)
    return dx, dgates, None, ddecay, None if initial_state is None else dinitial, None, None


varlen_recurrence_fwd_op.register_autograd(_op_backward, setup_context=_op_setup_context)


def _step_now(x, gates, decay, state, slots, scale, out_state):
    """A step inside of an op: whatever records operations has the op."""
    y = _lib.load_node().recurrence_step(x, gates, decay, state, slots, scale, out_state)
    return _step(x, gates, decay, state, slots, scale, out_state) if y is None else y


@torch.library.custom_op("nanoplm_amd::recurrence_step", mutates_args=("state",), device_types="cuda")
def recurrence_step_op(x: torch.Tensor, gates: torch.Tensor, decay: torch.Tensor, state: torch.Tensor, slots: Optional[torch.Tensor],
                       scale: float = 8.0) -> torch.Tensor:
    """A step whose table holds the new states afterwards."""
    return _step_now(x, gates, decay, state, slots, scale, None)


@torch.library.custom_op("nanoplm_amd::recurrence_step_to", mutates_args=("out_state",), device_types="cuda")
def recurrence_step_to_op(x: torch.Tensor, gates: torch.Tensor, decay: torch.Tensor, state: torch.Tensor, slots: Optional[torch.Tensor], scale: float,
                          out_state: torch.Tensor) -> torch.Tensor:
    """A step that leaves the old states and writes the new ones into another table."""
    return _step_now(x, gates, decay, state, slots, scale, out_state)


@recurrence_step_op.register_fake
def _(x, gates, decay, state, slots, scale=8.0):
    return x.new_empty(x.shape)


@recurrence_step_to_op.register_fake
def _(x, gates, decay, state, slots, scale, out_state):
    return x.new_empty(x.shape)


class VarlenRecurrence(nn.Module):
    """Gated linear recurrence over packed sequences: ``forward(x:[T, C], gates:[T, 2C], cu_seqlens:int32[S+1])``.

    ``decay`` ``[C]`` is initialised so that a channel whose recurrence gate is open keeps between 0.9 and 0.999 of its state a token. It is a 1-D
    parameter, which the reference's grouping rules send to AdamW without weight decay (src/nanoplm/pretraining/optim.py:43-51,
    src/nanoplm/pretraining/pure_pipeline.py:68-76)."""

    def __init__(self, channels: int, scale: float = 8.0, reverse: bool = False, device=None, dtype=None):
        super().__init__()
        if channels < 1 or not scale > 0:
            raise ValueError(f"channels and scale must be positive, got {channels} and {scale}")
        self.channels, self.scale, self.reverse = channels, float(scale), bool(reverse)
        self.decay = nn.Parameter(torch.empty((channels,), device=device, dtype=dtype))
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        kept = torch.empty(self.channels, dtype=torch.float64).uniform_(0.9, 0.999)
        self.decay.copy_(torch.log(torch.expm1(-torch.log(kept) / self.scale)))

    def forward(self, x, gates, cu_seqlens, initial_state=None, return_state: bool = False):
        return varlen_recurrence(x, gates, cu_seqlens, self.decay, scale=self.scale, initial_state=initial_state, reverse=self.reverse,
                                 return_state=return_state)

    def forward_padded(self, x: torch.Tensor, gates: torch.Tensor, attention_mask: torch.Tensor) -> torch.Tensor:
        """Padded-batch door: ``x:[B, L, C]``, ``gates:[B, L, 2C]`` and a right-padded ``attention_mask:[B, L]``, in place (no gather). Padding positions
        hold the recurrence over the pad run they belong to, as with the conv's door (see nanoplm_amd.padded)."""
        from .padded import _flat_cu_seqlens
        if x.dim() != 3 or gates.dim() != 3 or gates.shape[:2] != x.shape[:2] or attention_mask.shape != x.shape[:2]:
            raise ValueError("x must be [B, L, C], gates [B, L, 2C] and attention_mask [B, L]")
        B, L, C = x.shape
        cu = _flat_cu_seqlens(attention_mask, x)
        return self.forward(x.reshape(B * L, C), gates.reshape(B * L, gates.shape[2]), cu).view(B, L, C)

    def step(self, x, gates, state, slots=None, out_state=None) -> torch.Tensor:
        """One token of each sequence in a table of states (see :func:`recurrence_step`), under ``torch.no_grad()``: ``decay`` is a parameter."""
        if self.reverse:
            raise RuntimeError("a recurrence from the last token to the first one has no next token to step to")
        return recurrence_step(x, gates, self.decay, state, slots, scale=self.scale, out_state=out_state)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, scale={self.scale}, reverse={self.reverse}"
