"""Linear attention with a decay for each head over packed sequences: a recurrence whose state is a matrix, on the rows that the depthwise conv and the
gated recurrence work on.

Per head, from each sequence's first row to its last one (from the last to the first with ``reverse``)::

    S_t = exp(log_decay_t) * S_{t-1} + k_t v_t^T                    S: [dk, dv]
    o_t = scale * q_t S_t                                           scale: dk ** -0.5 unless given

``q``, ``k`` ``[T, H, dk]`` and ``v`` ``[T, H, dv]`` may be views of wider tensors, or expanded over heads that share them (any strides, adjacent channels; the
gradient of what was expanded is autograd's sum). ``log_decay`` is ``[H]`` or ``[T, H]``, in fp32 or the activations' dtype, 0 or less (-inf: the state is
forgotten). Sequences begin with zeros or with ``initial_state`` ``[S, H, dk, dv]`` and end with a state that ``return_state`` hands out, so that a long sequence
can be run in pieces and a prompt be continued token by token with :func:`linear_attention_step`. States are fp32 whatever the activations' dtype is.

The reference's packed path (src/nanoplm/pretraining/models/modern_bert/modeling.py:421-439) hands its sub-modules ``x:[total_tokens, hidden]`` and int32
``cu_seqlens``; its attention is softmax attention, which this does not replace. All arithmetic runs in hand-written HIP kernels behind
include/nplm_linattn.h; there is no CPU implementation.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch import nn

from . import _lib
from .dwconv import _DTYPES, _launch_on, _ptr
from .padded import _operations_are_recorded
from .recurrence import _dense, _plain, _refuse_tangents

MAX_DIM = 128           # NPLM_LINATTN_MAX_DIM
MAX_SLOTS = 1 << 16     # NPLM_LINATTN_MAX_SLOTS
_SEGMENT_ROWS, _SEGMENTS = 2048, 512        # the longest segment; shorter ones are taken for at most so many of them, over all heads


def _heads(t: torch.Tensor) -> torch.Tensor:
    """t itself where the channels of a head are adjacent; else a contiguous copy."""
    t = t.resolve_neg()
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _strides(t: torch.Tensor):
    """Elements from row to row and from head to head (0 along a dimension of one)."""
    return tuple(0 if n == 1 else st for n, st in zip(t.shape[:2], t.stride()[:2]))


def _rates(log_decay: torch.Tensor) -> torch.Tensor:
    return log_decay.resolve_neg()


def _rate_strides(g: torch.Tensor):
    return _strides(g) if g.dim() == 2 else (0, 0 if g.shape[0] == 1 else g.stride(0))


def _rate_flag(g: torch.Tensor) -> int:
    return _lib.LINATTN_HEAD_DECAY if g.dim() == 1 else 0


def _scale_of(scale: Optional[float], dk: int) -> float:
    return dk ** -0.5 if scale is None else float(scale)


def _check_rows(q, k, v, log_decay, scale, name, rows="T"):
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError(f"q must be a 3-D tensor [{rows}, H, dk]")
    if q.dtype not in _DTYPES:
        raise TypeError(f"q must be float32 or bfloat16, got {q.dtype}")
    if not q.is_cuda:
        raise RuntimeError(f"{name} runs only on a ROCm device (q is on {q.device}); there is no CPU implementation")
    T, H, dk = q.shape
    if not isinstance(k, torch.Tensor) or k.shape != q.shape:
        raise ValueError(f"k must be [{rows}={T}, H={H}, dk={dk}], as q is")
    if not isinstance(v, torch.Tensor) or v.dim() != 3 or tuple(v.shape[:2]) != (T, H):
        raise ValueError(f"v must be [{rows}={T}, H={H}, dv]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"k and v must have q's dtype {q.dtype}, got {k.dtype} and {v.dtype}")
    dv = v.shape[2]
    if H < 1 or not 1 <= dk <= MAX_DIM or not 1 <= dv <= MAX_DIM:
        raise ValueError(f"at least one head, 1 to {MAX_DIM} channels of keys and of values, got H={H}, dk={dk}, dv={dv}")
    if not isinstance(log_decay, torch.Tensor) or tuple(log_decay.shape) not in ((H,), (T, H)):
        raise ValueError(f"log_decay must be [H={H}] or [{rows}={T}, H={H}]")
    if log_decay.dtype != torch.float32 and log_decay.dtype != q.dtype:
        raise TypeError(f"log_decay must be float32 or have q's dtype {q.dtype}, got {log_decay.dtype}")
    for what, t in (("k", k), ("v", v), ("log_decay", log_decay)):
        if t.device != q.device:
            raise RuntimeError(f"{what} is on {t.device}, q is on {q.device}")
    if not math.isfinite(_scale_of(scale, dk)):
        raise ValueError(f"scale must be finite, got {scale}")
    return T, H, dk, dv


def _check_state(t, shape, device, name):
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != shape or t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 {list(shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, q is on {device}")


def _check(q, k, v, cu_seqlens, log_decay, scale, initial_state):
    T, H, dk, dv = _check_rows(q, k, v, log_decay, scale, "varlen_linear_attention")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise TypeError("cu_seqlens must be a 1-D int32 tensor with at least one entry")
    if cu_seqlens.device != q.device:
        raise RuntimeError(f"cu_seqlens is on {cu_seqlens.device}, q is on {q.device}")
    S = cu_seqlens.numel() - 1
    _check_state(initial_state, (S, H, dk, dv), q.device, "initial_state")
    return T, H, dk, dv, S


def _bounds_bytes(T, H, S, dk, dv, act) -> int:
    return int(_lib.load().nplm_linattn_bounds_bytes(T, H, S, dk, dv, act))


def _most_bounds_bytes(T, H, dk, dv):
    """At least :func:`_bounds_bytes` whatever S is, in arithmetic that symbolic sizes can follow: segments shorter than the longest are ``T * H / _SEGMENTS`` rows or more."""
    return (_SEGMENTS // H + T // _SEGMENT_ROWS + 1) * H * (dk * dv + 1) * 4 + 512


def varlen_linear_attention_fwd(q, k, v, cu_seqlens, log_decay, *, scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                                reverse: bool = False, want_state: bool = False):
    """Raw forward (no autograd): ``(o, state, bounds)``: o in q's dtype, state ``[S, H, dk, dv]`` in fp32 (None unless wanted), and the bytes that
    :func:`varlen_linear_attention_bwd` restarts long sequences from (empty where there are none that long)."""
    return _fwd(q, k, v, cu_seqlens, log_decay, scale, initial_state, reverse, want_state, False)


def _fwd(q, k, v, cu_seqlens, log_decay, scale, initial_state, reverse, want_state, most):
    """most: bounds of :func:`_most_bounds_bytes`, for the registered op, whose outputs' sizes are known before S is."""
    T, H, dk, dv, S = _check(q, k, v, cu_seqlens, log_decay, scale, initial_state)
    lib = _lib.load()
    q, k, v, g, cu_seqlens, initial_state = _heads(q), _heads(k), _heads(v), _rates(log_decay), _dense(cu_seqlens), _dense(initial_state)
    act = _DTYPES[q.dtype]
    o = torch.empty((T, H, dv), dtype=q.dtype, device=q.device)
    state = torch.empty((S, H, dk, dv), dtype=torch.float32, device=q.device) if want_state else None
    nbytes = _bounds_bytes(T, H, S, dk, dv, act)
    bounds = torch.empty((_most_bounds_bytes(T, H, dk, dv) if most else nbytes,), dtype=torch.uint8, device=q.device)
    with _launch_on(q) as dev:
        rc = lib.nplm_linattn_fwd(_ptr(q), *_strides(q), _ptr(k), *_strides(k), _ptr(v), *_strides(v), _ptr(cu_seqlens), _ptr(g), *_rate_strides(g),
                                  _scale_of(scale, dk), _ptr(initial_state), _ptr(o), _ptr(state), _ptr(bounds) if nbytes else None, nbytes, T, H, S, dk, dv,
                                  act, _DTYPES[g.dtype], _rate_flag(g) | (_lib.LINATTN_REVERSE if reverse else 0), dev.stream)
    _lib.check(rc, "nplm_linattn_fwd")
    return o, state, bounds


def varlen_linear_attention_bwd(q, k, v, do, cu_seqlens, log_decay, bounds, *, scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                                state: Optional[torch.Tensor] = None, dstate: Optional[torch.Tensor] = None, reverse: bool = False,
                                want_dlog_decay: bool = True, want_dinitial: bool = False):
    """Raw backward of :func:`varlen_linear_attention_fwd`: ``(dq, dk, dv, dlog_decay, dinitial)``, the first four in their tensors' dtypes, dinitial in fp32 (the
    last two None unless wanted). ``bounds`` are the forward's; ``dstate`` is the gradient of its ``state``, which the log decays' gradient then needs as well."""
    T, H, dk, dv, S = _check(q, k, v, cu_seqlens, log_decay, scale, initial_state)
    if do.shape != v.shape or do.dtype != q.dtype or do.device != q.device:
        raise ValueError("do must match v in shape, dtype and device")
    for name, t in (("state", state), ("dstate", dstate)):
        _check_state(t, (S, H, dk, dv), q.device, name)
    if dstate is not None and state is None and want_dlog_decay:
        raise ValueError("dlog_decay beside dstate needs the forward's state")
    lib = _lib.load()
    act = _DTYPES[q.dtype]
    nbytes = _bounds_bytes(T, H, S, dk, dv, act)
    most = _most_bounds_bytes(T, H, dk, dv)
    if not isinstance(bounds, torch.Tensor) or bounds.dtype != torch.uint8 or bounds.numel() not in (nbytes, most) or bounds.device != q.device:
        raise ValueError(f"bounds must be the forward's ({nbytes} bytes, the registered op's {most})")
    q, k, v, do, g, cu_seqlens = _heads(q), _heads(k), _heads(v), _heads(do), _rates(log_decay), _dense(cu_seqlens)
    initial_state, state, dstate, bounds = _dense(initial_state), _dense(state), _dense(dstate), _dense(bounds)
    new = lambda d: torch.empty((T, H, d), dtype=q.dtype, device=q.device)
    dq, dk_, dv_ = new(dk), new(dk), new(dv)
    dlog = torch.empty(g.shape, dtype=g.dtype, device=q.device) if want_dlog_decay else None
    dinitial = torch.empty((S, H, dk, dv), dtype=torch.float32, device=q.device) if want_dinitial else None
    with _launch_on(q) as dev:
        wbytes = int(lib.nplm_linattn_bwd_workspace_bytes(T, H, S, dk, dv, act))
        workspace = torch.empty((max(wbytes, 256),), dtype=torch.uint8, device=q.device)
        rc = lib.nplm_linattn_bwd(_ptr(q), *_strides(q), _ptr(k), *_strides(k), _ptr(v), *_strides(v), _ptr(do), *_strides(do), _ptr(cu_seqlens), _ptr(g),
                                  *_rate_strides(g), _scale_of(scale, dk), _ptr(initial_state), _ptr(state), _ptr(dstate), _ptr(bounds) if nbytes else None, nbytes,
                                  _ptr(dq), _ptr(dk_), _ptr(dv_), _ptr(dlog), _ptr(dinitial), _ptr(workspace), wbytes, T, H, S, dk, dv, act, _DTYPES[g.dtype],
                                  _rate_flag(g) | (_lib.LINATTN_REVERSE if reverse else 0), dev.stream)
    _lib.check(rc, "nplm_linattn_bwd")
    return dq, dk_, dv_, dlog, dinitial


def linear_attention_step(q, k, v, log_decay, state, slots: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                          out_state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B sequences: o ``[B, H, dv]`` in q's dtype. No gradients.

    ``state`` is a table ``[N, H, dk, dv]`` of fp32 states; row b of ``q``, ``k`` ``[B, H, dk]`` and ``v`` ``[B, H, dv]`` (with its log decays, ``[H]`` or row b of
    ``[B, H]``) belongs to the state in row ``slots[b]`` (int32; row b without ``slots``), which is replaced by the new one, or, with ``out_state``, another table of the
    same size, left as it is and the new one written there (tokens that may be taken back; no memory shared with ``state``). Rows of ``out_state`` that no slot names
    are left alone. Rows that name the same slot are consecutive tokens of one sequence, in their order. A slot outside ``[0, N)`` marks a padding row: o is 0 and
    no state is touched. At most 2^16 rows name slots."""
    if not torch.compiler.is_compiling():
        o = _lib.load_node().linear_attention_step(q, k, v, log_decay, state, slots, scale, out_state)
        if o is not None:
            return o
        _refuse_step_gradients(q, k, v, log_decay, state, out_state)
    if _operations_are_recorded():
        if out_state is None or out_state is state:
            return linear_attention_step_op(q, k, v, log_decay, state, slots, scale)
        return linear_attention_step_to_op(q, k, v, log_decay, state, slots, scale, out_state)
    return _step(q, k, v, log_decay, state, slots, scale, out_state)


def _refuse_step_gradients(*tensors):
    _refuse_tangents("linear_attention_step", *tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError("linear_attention_step has no gradient: call it under torch.no_grad(), or use varlen_linear_attention")


def _step(q, k, v, log_decay, state, slots, scale, out_state):
    """:func:`linear_attention_step` at once, through ctypes."""
    B, H, dk, dv = _check_rows(q, k, v, log_decay, scale, "linear_attention_step", "B")
    if not isinstance(state, torch.Tensor) or state.dim() != 4 or tuple(state.shape[1:]) != (H, dk, dv) or state.dtype != torch.float32 or not _plain(state):
        raise ValueError(f"state must be a contiguous float32 table [N, H={H}, dk={dk}, dv={dv}]")
    out_state = state if out_state is None else out_state
    if out_state.shape != state.shape or out_state.dtype != torch.float32 or not _plain(out_state):
        raise ValueError("out_state must be a contiguous float32 table of state's shape")
    if 0 < abs(out_state.data_ptr() - state.data_ptr()) < 4 * state.numel():
        raise ValueError("out_state must be state itself or a table apart from it: it shares some of its memory")
    for what, t in (("state", state), ("out_state", out_state), ("slots", slots)):
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{what} is on {t.device}, q is on {q.device}")
    N = state.shape[0]
    if slots is not None and (slots.dtype != torch.int32 or tuple(slots.shape) != (B,)):
        raise TypeError(f"slots must be int32 [B={B}]")
    if slots is not None and B > MAX_SLOTS:
        raise ValueError(f"at most {MAX_SLOTS} rows a step with slots, got {B}: every row looks through all of them")
    if slots is None and B > N:
        raise ValueError(f"{B} rows need as many states, the table has {N} (or pass slots)")
    lib = _lib.load()
    q, k, v, g, slots = _heads(q), _heads(k), _heads(v), _rates(log_decay), _dense(slots)
    o = torch.empty((B, H, dv), dtype=q.dtype, device=q.device)
    if not out_state.is_inference():
        torch.autograd.graph.increment_version(out_state)
    with _launch_on(q) as dev:
        rc = lib.nplm_linattn_step(_ptr(q), *_strides(q), _ptr(k), *_strides(k), _ptr(v), *_strides(v), _ptr(g), *_rate_strides(g), _scale_of(scale, dk),
                                   _ptr(state), _ptr(out_state), _ptr(slots), _ptr(o), B, H, N, dk, dv, _DTYPES[q.dtype], _DTYPES[g.dtype], _rate_flag(g),
                                   dev.stream)
    _lib.check(rc, "nplm_linattn_step")
    return o


class VarlenLinearAttentionFunction(torch.autograd.Function):
    """``apply(q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, return_state) -> (o, state)``; gradients for q, k, v, log_decay and
    initial_state. state is None without ``return_state``."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, log_decay, initial_state=None, scale=None, reverse=False, return_state=False):
        o, state, bounds = varlen_linear_attention_fwd(q, k, v, cu_seqlens, log_decay, scale=scale, initial_state=initial_state, reverse=reverse,
                                                       want_state=return_state)
        ctx.save_for_backward(q, k, v, cu_seqlens, log_decay, initial_state, state, bounds)
        ctx.scale, ctx.reverse = scale, reverse
        ctx.set_materialize_grads(False)
        return o, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dstate):
        q, k, v, cu_seqlens, log_decay, initial_state, state, bounds = ctx.saved_tensors
        do = torch.zeros_like(v) if do is None else do if do.dtype == q.dtype else do.to(q.dtype)
        dq, dk, dv, dlog, dinitial = varlen_linear_attention_bwd(q, k, v, do, cu_seqlens, log_decay, bounds, scale=ctx.scale, initial_state=initial_state,
                                                                 state=state, dstate=dstate, reverse=ctx.reverse, want_dlog_decay=ctx.needs_input_grad[4],
                                                                 want_dinitial=initial_state is not None and ctx.needs_input_grad[5])
        return dq, dk, dv, None, dlog, dinitial, None, None, None


def varlen_linear_attention(q, k, v, cu_seqlens, log_decay, *, scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                            reverse: bool = False, return_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Differentiable linear attention over packed sequences: o, or ``(o, state)`` with ``return_state`` (see the module docstring). Where operations are
    recorded (``torch.compile``, ``torch.jit.trace``, a dispatch mode) the call goes through the registered custom ops (same kernels; a recorded launch would be an
    ``empty`` that nothing fills); otherwise the native node takes it or, for a call that is not of its form, leaves it to the Function."""
    if not torch.compiler.is_compiling():
        out = _lib.load_node().linear_attention(q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, return_state)
        if out is not None:
            return out if return_state else out[0]
        _refuse_tangents("varlen_linear_attention", q, k, v, log_decay, initial_state)
    if _operations_are_recorded():
        o, state, _ = varlen_linear_attention_fwd_op(q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, return_state)
        return (o, state) if return_state else o
    o, state = VarlenLinearAttentionFunction.apply(q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, return_state)
    return (o, state) if return_state else o


# ---------------------------------------------------------------------------------------------
# torch.library registration, so that a compiled model (src/nanoplm/pretraining/pure_pipeline.py:519-524) keeps one graph. An op returns tensors
# only: what a call does not have is an empty tensor.
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("nanoplm_amd::varlen_linear_attention_fwd", mutates_args=(), device_types="cuda")
def varlen_linear_attention_fwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, log_decay: torch.Tensor,
                                   initial_state: Optional[torch.Tensor], scale: Optional[float], reverse: bool,
                                   want_state: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(o, state, bounds), the last as large as it gets for any number of sequences."""
    o, state, bounds = _fwd(q, k, v, cu_seqlens, log_decay, scale, initial_state, reverse, want_state, True)
    return o, q.new_empty((0,), dtype=torch.float32) if state is None else state, bounds


@varlen_linear_attention_fwd_op.register_fake
def _(q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, want_state):
    (T, H, dk), dv, S = q.shape, v.shape[2], cu_seqlens.shape[0] - 1
    nbytes = _most_bounds_bytes(T, H, dk, dv)                  # (sizes may be symbols: nothing here asks for their values)
    return (q.new_empty((T, H, dv)), q.new_empty((S, H, dk, dv) if want_state else (0,), dtype=torch.float32), q.new_empty((nbytes,), dtype=torch.uint8))


@torch.library.custom_op("nanoplm_amd::varlen_linear_attention_bwd", mutates_args=(), device_types="cuda")
def varlen_linear_attention_bwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, do: torch.Tensor, cu_seqlens: torch.Tensor, log_decay: torch.Tensor,
                                   bounds: torch.Tensor, initial_state: Optional[torch.Tensor], state: Optional[torch.Tensor],
                                   dstate: Optional[torch.Tensor], scale: Optional[float], reverse: bool, want_dlog_decay: bool,
                                   want_dinitial: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv, dlog_decay, dinitial)."""
    dq, dk, dv, dlog, dinitial = varlen_linear_attention_bwd(q, k, v, do, cu_seqlens, log_decay, bounds, scale=scale, initial_state=initial_state, state=state,
                                                             dstate=dstate, reverse=reverse, want_dlog_decay=want_dlog_decay, want_dinitial=want_dinitial)
    return (dq, dk, dv, log_decay.new_empty((0,)) if dlog is None else dlog, q.new_empty((0,), dtype=torch.float32) if dinitial is None else dinitial)


@varlen_linear_attention_bwd_op.register_fake
def _(q, k, v, do, cu_seqlens, log_decay, bounds, initial_state, state, dstate, scale, reverse, want_dlog_decay, want_dinitial):
    S = cu_seqlens.shape[0] - 1
    return (q.new_empty(q.shape), q.new_empty(q.shape), q.new_empty(v.shape), log_decay.new_empty(log_decay.shape if want_dlog_decay else (0,)),
            q.new_empty((S, q.shape[1], q.shape[2], v.shape[2]) if want_dinitial else (0,), dtype=torch.float32))


def _op_setup_context(ctx, inputs, output):
    q, k, v, cu_seqlens, log_decay, initial_state, scale, reverse, want_state = inputs
    ctx.save_for_backward(q, k, v, cu_seqlens, log_decay, initial_state, output[1] if want_state else None, output[2])
    ctx.scale, ctx.reverse = scale, bool(reverse)
    ctx.set_materialize_grads(False)


def _op_backward(ctx, do, dstate, _dbounds):
    q, k, v, cu_seqlens, log_decay, initial_state, state, bounds = ctx.saved_tensors
    do = torch.zeros_like(v) if do is None else do if do.dtype == q.dtype else do.to(q.dtype)
    want = ctx.needs_input_grad[4], initial_state is not None and ctx.needs_input_grad[5]
    dq, dk, dv, dlog, dinitial = varlen_linear_attention_bwd_op(q, k, v, do, cu_seqlens, log_decay, bounds, initial_state, state,
                                                                None if state is None else dstate, ctx.scale, ctx.reverse, *want)
    return dq, dk, dv, None, dlog if want[0] else None, dinitial if want[1] else None, None, None, None


varlen_linear_attention_fwd_op.register_autograd(_op_backward, setup_context=_op_setup_context)


def _step_now(q, k, v, log_decay, state, slots, scale, out_state):
    """A step inside of an op: whatever records operations has the op."""
    o = _lib.load_node().linear_attention_step(q, k, v, log_decay, state, slots, scale, out_state)
    return _step(q, k, v, log_decay, state, slots, scale, out_state) if o is None else o


@torch.library.custom_op("nanoplm_amd::linear_attention_step", mutates_args=("state",), device_types="cuda")
def linear_attention_step_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                             slots: Optional[torch.Tensor], scale: Optional[float]) -> torch.Tensor:
    """A step whose table holds the new states afterwards."""
    return _step_now(q, k, v, log_decay, state, slots, scale, None)


@torch.library.custom_op("nanoplm_amd::linear_attention_step_to", mutates_args=("out_state",), device_types="cuda")
def linear_attention_step_to_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                                slots: Optional[torch.Tensor], scale: Optional[float], out_state: torch.Tensor) -> torch.Tensor:
    """A step that leaves the old states and writes the new ones into another table."""
    return _step_now(q, k, v, log_decay, state, slots, scale, out_state)


@linear_attention_step_op.register_fake
def _(q, k, v, log_decay, state, slots, scale):
    return q.new_empty(v.shape)


@linear_attention_step_to_op.register_fake
def _(q, k, v, log_decay, state, slots, scale, out_state):
    return q.new_empty(v.shape)


class VarlenLinearAttention(nn.Module):
    """Linear attention over packed sequences: ``forward(q:[T, H, dk], k:[T, H, dk], v:[T, H, dv], cu_seqlens:int32[S+1], gates:[T, H] = None)``.

    A head keeps ``sigmoid(decay)`` of its state a token, ``sigmoid(decay + gates_t)`` with gates from a projection. ``decay`` ``[H]`` is initialised so that the
    heads keep 1 - 2^-5 to 1 - 2^-9. It is a 1-D parameter, which the reference's grouping rules send to AdamW without weight decay
    (src/nanoplm/pretraining/optim.py:43-51, src/nanoplm/pretraining/pure_pipeline.py:68-76)."""

    def __init__(self, heads: int, scale: Optional[float] = None, reverse: bool = False, device=None, dtype=None):
        super().__init__()
        if heads < 1 or (scale is not None and not math.isfinite(scale)):
            raise ValueError(f"heads must be positive and scale finite, got {heads} and {scale}")
        self.heads, self.scale, self.reverse = heads, scale, bool(reverse)
        self.decay = nn.Parameter(torch.empty((heads,), device=device, dtype=dtype))
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        lost = 2.0 ** -torch.linspace(5, 9, self.heads, dtype=torch.float64)
        self.decay.copy_(torch.log((1 - lost) / lost))

    def log_decay(self, gates: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The log decays ``[H]``, or ``[T, H]`` with gates."""
        return F.logsigmoid(self.decay if gates is None else self.decay + gates)

    def forward(self, q, k, v, cu_seqlens, gates=None, initial_state=None, return_state: bool = False):
        return varlen_linear_attention(q, k, v, cu_seqlens, self.log_decay(gates), scale=self.scale, initial_state=initial_state, reverse=self.reverse,
                                       return_state=return_state)

    def forward_padded(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, attention_mask: torch.Tensor, gates: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Padded-batch door: ``q``, ``k`` ``[B, L, H, dk]``, ``v`` ``[B, L, H, dv]``, gates ``[B, L, H]`` and a right-padded ``attention_mask:[B, L]``, in place (no
        gather). Padding positions hold the attention over the pad run they belong to, as with the conv's door (see nanoplm_amd.padded)."""
        from .padded import _flat_cu_seqlens
        if any(t.dim() != 4 or t.shape[:2] != attention_mask.shape for t in (q, k, v)) or (gates is not None and gates.shape != q.shape[:3]):
            raise ValueError("q, k and v must be [B, L, H, channels], gates [B, L, H] and attention_mask [B, L]")
        B, L = attention_mask.shape
        flat = lambda t: None if t is None else t.reshape(B * L, *t.shape[2:])
        return self.forward(flat(q), flat(k), flat(v), _flat_cu_seqlens(attention_mask, q), flat(gates)).view(B, L, *v.shape[2:])

    def step(self, q, k, v, state, slots=None, gates=None, out_state=None) -> torch.Tensor:
        """One token of each sequence in a table of states (see :func:`linear_attention_step`), under ``torch.no_grad()``: ``decay`` is a parameter."""
        if self.reverse:
            raise RuntimeError("a recurrence from the last token to the first one has no next token to step to")
        return linear_attention_step(q, k, v, self.log_decay(gates), state, slots, scale=self.scale, out_state=out_state)

    def extra_repr(self) -> str:
        return f"heads={self.heads}, scale={self.scale}, reverse={self.reverse}"
