"""Linear attention with a decay for each head: the recurrences of this package on a matrix state,

    S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T,      o[t] = scale * q[t]^T S[t]

``lti.linear_attention`` (one decay per head) and ``lpv.linear_attention`` (one per token and head) are
thin front ends of this module, like ``linear_recurrence`` and ``state_space`` beside them: torch custom ops
(``torch.ops.philtorch_b200.linear_attention*``), an autograd Function with fused adjoint kernels, and the
argument checks.  The coefficient with time index t multiplies the PREVIOUS state, as everywhere in
this package; it is passed as its logarithm, so that decays near one keep their precision and a decay of
zero (``-inf``: the sequence starts anew at this token) is an ordinary value.
"""
from __future__ import annotations

import ctypes
from typing import Any, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib, ptr
from .norm import check_parameters, layer_norm, layer_norm_of_sums
from .ops import _LIB, _TAGS

__all__ = ["LinearAttention", "MAX_HEAD_DIM"]

MAX_HEAD_DIM = 128
_CODES = {torch.float32: _lib.PTB_F32, torch.float64: _lib.PTB_F64, torch.float16: _lib.PTB_F16,
          torch.bfloat16: _lib.PTB_BF16}


def state_dtype(dtype: torch.dtype) -> torch.dtype:
    """Type of the states and of the log decays: float64 beside float64 tensors, else float32."""
    return torch.float64 if dtype == torch.float64 else torch.float32


_stride_arrays: dict = {}


def _array(strides: tuple):
    """The strides as a ctypes array (kept by value: a program's tensors have few different ones)."""
    a = _stride_arrays.get(strides)
    if a is None:
        if len(_stride_arrays) > 4096:
            _stride_arrays.clear()
        a = _stride_arrays[strides] = (ctypes.c_int64 * len(strides))(*strides)
    return a


def _outer_strides(t: Tensor):
    return _array(t.stride()[:-1])


def _rows(t: Tensor) -> Tensor:
    """The tensor with its last axis dense; the other strides are the kernels' arguments (views of one fused
    projection, or heads shared through ``expand``, are read in place)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _code(t: Tensor) -> int:
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise RuntimeError("linear attention takes float32, float64, float16 and bfloat16 tensors, "
                           f"got {t.dtype}") from None


def _check(q: Tensor, k: Tensor, v: Tensor, g: Tensor, init: Optional[Tensor], lengths: Optional[Tensor]) -> None:
    # the common case in one expression: the explanations below cost more host time than the launch
    shape, dt = q.shape, q.dtype
    if (len(shape) == 4 and k.shape == shape and v.dim() == 4 and v.shape[:3] == shape[:3] and k.dtype == dt and v.dtype == dt
            and 1 <= shape[3] <= MAX_HEAD_DIM and 1 <= v.shape[3] <= MAX_HEAD_DIM and lengths is None
            and g.dtype == state_dtype(dt) and (g.shape == shape[2:3] or g.shape == shape[:3])
            and (init is None or (init.dtype == g.dtype and init.shape == (shape[0], shape[2], shape[3], v.shape[3])))):
        return
    torch._check(q.dim() == 4, lambda: f"q must be 4D (batch, time, heads, Dk), got {tuple(q.shape)}")
    torch._check(k.shape == q.shape, lambda: f"k must have the shape of q, got {tuple(k.shape)} and {tuple(q.shape)}")
    torch._check(v.dim() == 4 and v.shape[:3] == q.shape[:3],
                 lambda: f"v must be (batch, time, heads, Dv) beside q {tuple(q.shape)}, got {tuple(v.shape)}")
    B, T, H, Dk = q.shape
    Dv = v.shape[3]
    torch._check(1 <= Dk <= MAX_HEAD_DIM and 1 <= Dv <= MAX_HEAD_DIM,
                 lambda: f"head sizes Dk = {Dk}, Dv = {Dv}: the kernels cover 1..{MAX_HEAD_DIM}.")
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype,
                 lambda: f"q, k and v must have the same type, got {q.dtype}, {k.dtype}, {v.dtype}")
    wide = state_dtype(q.dtype)
    torch._check(g.dtype == wide, lambda: f"log_decay must be {wide} beside {q.dtype} tensors, got {g.dtype}")
    torch._check(tuple(g.shape) in ((H,), (B, T, H)),
                 lambda: f"log_decay must be (heads,) or (batch, time, heads), got {tuple(g.shape)}")
    if init is not None:
        torch._check(tuple(init.shape) == (B, H, Dk, Dv),
                     lambda: f"the initial state must be {(B, H, Dk, Dv)}, got {tuple(init.shape)}")
        torch._check(init.dtype == wide, lambda: f"the initial state must be {wide} beside {q.dtype} tensors, got {init.dtype}")
    if lengths is not None:
        torch._check(tuple(lengths.shape) == (B,), lambda: f"lengths must be ({B},), got {tuple(lengths.shape)}")
        torch._check(lengths.dtype in (torch.int32, torch.int64), lambda: f"lengths must be int32 or int64, got {lengths.dtype}")


def _decay_strides(g: Tensor):
    return _array((0, 0, g.stride(0)) if g.dim() == 1 else g.stride())


_ws_bytes: dict = {}


def _workspace_bytes(*key) -> int:
    n = _ws_bytes.get(key)
    if n is None:
        if len(_ws_bytes) > 4096:   # a server sees many lengths
            _ws_bytes.clear()
        n = _ws_bytes[key] = lib.ptb_linear_attention_workspace_bytes(*key)
    return n


_ANY_ROWS = lib.ptb_linear_attention_any_rows_tokens(_lib.PTB_BF16)   # longer bfloat16 sequences run on the tensor cores


def _copies(T: int, *tensors: Tensor) -> int:
    """The operands whose rows the tensor-core kernels' TMA loads cannot address, a bit for each: they are copied."""
    if T <= _ANY_ROWS or tensors[0].dtype != torch.bfloat16:
        return 0
    mask = 0
    for i, t in enumerate(tensors):
        b, s, h, _ = t.stride()
        if t.data_ptr() % 16 or s % 8 or s == 0 or (h % 8 and t.shape[2] > 1) or (b % 8 and t.shape[0] > 1):
            mask |= 1 << i
    return mask


def _lengths_args(lengths: Optional[Tensor]):
    return (None, 0) if lengths is None else (lengths.data_ptr(), int(lengths.dtype == torch.int64))


# ------------------------------------------------------------------------------------------------ ops
_LIB.define("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? init, Tensor? lengths, "
            "float scale, bool want_state, bool wide=False) -> (Tensor, Tensor)", tags=_TAGS)
_LIB.define("linear_attention_bwd(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? init, Tensor? lengths, "
            "float scale, Tensor? grad_o, Tensor? grad_state, bool need_q, bool need_k, bool need_v, "
            "bool need_decay, bool need_init) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", tags=_TAGS)
_LIB.define("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float scale, "
            "bool wide=False) -> Tensor", tags=_TAGS)


def _linear_attention(q, k, v, log_decay, init, lengths, scale, want_state, wide=False):
    _check(q, k, v, log_decay, init, lengths)
    dev = _lib.require_cuda(q, k, v, log_decay, init, lengths)
    code = _code(q)
    B, T, H, Dk = q.shape
    Dv = v.shape[3]
    q, k, v = _rows(q), _rows(k), _rows(v)
    init = None if init is None else init.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    o = (log_decay if wide else v).new_empty((B, T, H, Dv))   # wide: in the sums' type, for a normalisation that follows
    state = log_decay.new_empty((B, H, Dk, Dv) if want_state else (0,))
    if B and H and (T or want_state):
        copies = _copies(T, q, k, v)
        _lib.call(lib.ptb_linear_attention_fwd, dev, B, T, code, B, T, H, Dk, Dv, ptr(q), _outer_strides(q), ptr(k), _outer_strides(k),
                  ptr(v), _outer_strides(v), ptr(log_decay), _decay_strides(log_decay), *_lengths_args(lengths), ptr(init), scale, copies,
                  ptr(o),
                  int(o.dtype != v.dtype), ptr(state) if want_state else None, ws_bytes=_workspace_bytes(code, B, T, H, Dk, Dv, 0, 0, copies))
    return o, state


def _linear_attention_bwd(q, k, v, log_decay, init, lengths, scale, grad_o, grad_state, need_q, need_k, need_v,
                          need_decay, need_init):
    dev = _lib.require_cuda(q, k, v, log_decay, init, lengths, grad_o, grad_state)
    code = _code(q)
    B, T, H, Dk = q.shape
    Dv = v.shape[3]
    if grad_o is None:   # only the final state was used
        grad_o = v.new_zeros(Dv).expand(B, T, H, Dv)
    q, k, v, grad_o = _rows(q), _rows(k), _rows(v), _rows(grad_o)
    init = None if init is None else init.contiguous()
    grad_state = None if grad_state is None else grad_state.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    gq, gk, gv = (t.new_empty(t.shape if need else (0,)) for t, need in ((q, need_q), (k, need_k), (v, need_v)))
    gg = log_decay.new_empty(log_decay.shape if need_decay else (0,))
    ginit = log_decay.new_empty((B, H, Dk, Dv) if need_init else (0,))
    if B and H:
        copies = _copies(T, q, k, v, grad_o)
        opt = lambda t, need: ptr(t) if need else None   # noqa: E731
        _lib.call(lib.ptb_linear_attention_bwd, dev, B, T, code, B, T, H, Dk, Dv, ptr(q), _outer_strides(q), ptr(k), _outer_strides(k),
                  ptr(v), _outer_strides(v), ptr(log_decay), _decay_strides(log_decay), *_lengths_args(lengths), ptr(init), scale, copies,
                  ptr(grad_o),
                  _outer_strides(grad_o), ptr(grad_state), opt(gq, need_q), opt(gk, need_k), opt(gv, need_v),
                  opt(gg, need_decay), int(log_decay.dim() == 3), opt(ginit, need_init),
                  ws_bytes=_workspace_bytes(code, B, T, H, Dk, Dv, 1, int(need_decay), copies))
    else:
        gg.zero_()
    return gq, gk, gv, gg, ginit


def _check_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, state: Tensor) -> None:
    shape, dt = q.shape, q.dtype
    if (len(shape) == 3 and k.shape == shape and v.dim() == 3 and v.shape[:2] == shape[:2] and k.dtype == dt and v.dtype == dt
            and 1 <= shape[2] <= MAX_HEAD_DIM and 1 <= v.shape[2] <= MAX_HEAD_DIM and g.dtype == state_dtype(dt)
            and (g.shape == shape[1:2] or g.shape == shape[:2]) and state.dtype == g.dtype
            and state.shape == (shape[0], shape[1], shape[2], v.shape[2]) and state.is_contiguous()):
        return
    torch._check(q.dim() == 3, lambda: f"q must be 3D (batch, heads, Dk), got {tuple(q.shape)}")
    torch._check(k.shape == q.shape, lambda: f"k must have the shape of q, got {tuple(k.shape)} and {tuple(q.shape)}")
    torch._check(v.dim() == 3 and v.shape[:2] == q.shape[:2],
                 lambda: f"v must be (batch, heads, Dv) beside q {tuple(q.shape)}, got {tuple(v.shape)}")
    B, H, Dk = q.shape
    Dv = v.shape[2]
    torch._check(1 <= Dk <= MAX_HEAD_DIM and 1 <= Dv <= MAX_HEAD_DIM,
                 lambda: f"head sizes Dk = {Dk}, Dv = {Dv}: the kernels cover 1..{MAX_HEAD_DIM}.")
    torch._check(k.dtype == q.dtype and v.dtype == q.dtype,
                 lambda: f"q, k and v must have the same type, got {q.dtype}, {k.dtype}, {v.dtype}")
    wide = state_dtype(q.dtype)
    torch._check(g.dtype == wide, lambda: f"log_decay must be {wide} beside {q.dtype} tensors, got {g.dtype}")
    torch._check(tuple(g.shape) in ((H,), (B, H)),
                 lambda: f"log_decay must be (heads,) or (batch, heads), got {tuple(g.shape)}")
    torch._check(tuple(state.shape) == (B, H, Dk, Dv), lambda: f"state must be {(B, H, Dk, Dv)}, got {tuple(state.shape)}")
    torch._check(state.dtype == wide, lambda: f"state must be {wide} beside {q.dtype} tensors, got {state.dtype}")
    # it is written in place: each (Dk, Dv) matrix dense, no two of them sharing memory
    ok = (state.stride(3) == 1 or Dv == 1) and (state.stride(2) == Dv or Dk == 1)
    room = Dk * Dv
    for stride, size in sorted((state.stride(i), state.shape[i]) for i in (0, 1) if state.shape[i] > 1):
        ok = ok and stride >= room
        room = stride * size
    torch._check(ok or state.numel() == 0, lambda: "state is updated in place: its (Dk, Dv) matrices must be dense and "
                                                   f"apart from one another, got strides {tuple(state.stride())}")


def _linear_attention_step(q, k, v, log_decay, state, scale, wide=False):
    _check_step(q, k, v, log_decay, state)
    dev = _lib.require_cuda(q, k, v, log_decay, state)
    B, H, Dk = q.shape
    Dv = v.shape[2]
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = (state if wide else v).new_empty((B, H, Dv))   # wide: in the sums' type, for a normalisation that follows
    if B and H:
        gs = _array((0, log_decay.stride(0)) if log_decay.dim() == 1 else log_decay.stride())
        entry = lib.ptb_linear_attention_step_sums if wide else lib.ptb_linear_attention_step
        _lib.launch(entry, dev, _code(q), B, H, Dk, Dv, ptr(q), _outer_strides(q), ptr(k), _outer_strides(k), ptr(v), _outer_strides(v),
                    ptr(log_decay), gs, scale, ptr(state), _array(state.stride()[:2]), ptr(o))
        torch.autograd.graph.increment_version(state)
    return o


_LIB.impl("linear_attention", _linear_attention, "CUDA")
_LIB.impl("linear_attention_bwd", _linear_attention_bwd, "CUDA")
_LIB.impl("linear_attention_step", _linear_attention_step, "CUDA")


@torch.library.register_fake("philtorch_b200::linear_attention")
def _(q, k, v, log_decay, init, lengths, scale, want_state, wide=False):
    _check(q, k, v, log_decay, init, lengths)
    B, T, H, Dk = q.shape
    return (log_decay if wide else v).new_empty((B, T, H, v.shape[3])), log_decay.new_empty((B, H, Dk, v.shape[3]) if want_state else (0,))


@torch.library.register_fake("philtorch_b200::linear_attention_bwd")
def _(q, k, v, log_decay, init, lengths, scale, grad_o, grad_state, need_q, need_k, need_v, need_decay, need_init):
    gq, gk, gv = (t.new_empty(t.shape if need else (0,)) for t, need in ((q, need_q), (k, need_k), (v, need_v)))
    B, T, H, Dk = q.shape
    return (gq, gk, gv, log_decay.new_empty(log_decay.shape if need_decay else (0,)),
            log_decay.new_empty((B, H, Dk, v.shape[3]) if need_init else (0,)))


@torch.library.register_fake("philtorch_b200::linear_attention_step")
def _(q, k, v, log_decay, state, scale, wide=False):
    _check_step(q, k, v, log_decay, state)
    return (state if wide else v).new_empty(v.shape)


_ops = torch.ops.philtorch_b200


# ------------------------------------------------------------------------------------------------ autograd
def _forward(q, k, v, log_decay, init, lengths, scale, want_state, wide=False):
    if q.device.type == "cpu":
        _lib.require_cuda(q)
    run = _linear_attention if _lib.eager(q) else _ops.linear_attention
    return run(q, k, v, log_decay, init, lengths, scale, want_state, wide)


def _backward(ctx: Any, grad_o: Optional[Tensor], grad_state: Optional[Tensor]):
    need = ctx.needs_input_grad[:5]
    if (grad_o is None and grad_state is None) or not any(need):
        return (None,) * 8
    q, k, v, log_decay, init, lengths = ctx.saved_tensors
    run = _linear_attention_bwd if _lib.eager(q) else _ops.linear_attention_bwd
    grads = run(q, k, v, log_decay, init, lengths, ctx.scale, grad_o, grad_state, *need)
    return (*(g if n else None for g, n in zip(grads, need)), None, None, None)


_backward_once = once_differentiable(_backward)


class LinearAttention(Function):
    """(q, k, v, log_decay, init or None, lengths or None, scale, want_state) -> (o, final state).  First
    derivatives; the backward pass recomputes the states instead of keeping them."""

    @staticmethod
    def forward(ctx: Any, q, k, v, log_decay, init, lengths, scale: float, want_state: bool):
        o, state = _forward(q, k, v, log_decay, init, lengths, scale, want_state)
        ctx.save_for_backward(q, k, v, log_decay, init, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if not want_state:
            ctx.mark_non_differentiable(state)
        return o, state

    @staticmethod
    def backward(ctx: Any, grad_o: Optional[Tensor], grad_state: Optional[Tensor]):
        # (the guard against second derivatives is only needed, and only paid, where a graph is being recorded)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad_o, grad_state)


def _check_norm(v: Tensor, eps: Optional[float], weight: Optional[Tensor], bias: Optional[Tensor]) -> None:
    """What the norm of the read-out would refuse, before anything runs: a step has moved its state on by then."""
    if eps is None:
        if weight is not None or bias is not None:
            raise ValueError("norm_weight and norm_bias need norm_eps")
    elif v.dim() >= 2:      # (anything else is refused by the operator's own checks)
        check_parameters(v.shape[-2] * v.shape[-1], v.dtype, weight, bias, v.shape[-2])
        if v.is_cuda:
            _lib.require_cuda(v, weight, bias)


def _normalised(o: Tensor, dtype: torch.dtype, eps: float, weight: Optional[Tensor], bias: Optional[Tensor]) -> Tensor:
    H, Dv = o.shape[-2:]
    rows = o.flatten(-2)
    if o.dtype == dtype:
        return layer_norm(rows, weight, bias, eps=eps, groups=H).unflatten(-1, (H, Dv))
    return layer_norm_of_sums(rows, weight, bias, float(eps), H, dtype).unflatten(-1, (H, Dv))


def _norm_differentiable(*params: Optional[Tensor]) -> bool:
    return torch.is_grad_enabled() and any(p is not None and p.requires_grad for p in params)


def attend(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, zi: Optional[Tensor], scale: float,
           lengths: Optional[Tensor], return_state: Optional[bool], norm_eps: Optional[float],
           norm_weight: Optional[Tensor], norm_bias: Optional[Tensor]):
    _lib.refuse_tangents("linear_attention", q, k, v, log_decay, zi, norm_weight, norm_bias)
    _check_norm(v, norm_eps, norm_weight, norm_bias)
    want = (zi is not None) if return_state is None else bool(return_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or (zi is not None and zi.requires_grad)):
        o, state = LinearAttention.apply(q, k, v, log_decay, zi, lengths, float(scale), want)
    else:   # (without gradients the normalisation reads the sums before they are rounded to q's type)
        wide = norm_eps is not None and not _norm_differentiable(norm_weight, norm_bias)
        o, state = _forward(q, k, v, log_decay, zi, lengths, float(scale), want, wide)
    if norm_eps is not None:
        o = _normalised(o, q.dtype, norm_eps, norm_weight, norm_bias)
    return (o, state) if want else o


def attend_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: float,
                norm_eps: Optional[float], norm_weight: Optional[Tensor], norm_bias: Optional[Tensor]) -> Tensor:
    _lib.refuse_tangents("linear_attention_step", q, k, v, log_decay, state, norm_weight, norm_bias)
    _check_norm(v, norm_eps, norm_weight, norm_bias)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad):
        raise RuntimeError("linear_attention_step updates its state in place and is not differentiable: call it under "
                           "torch.no_grad(), or linear_attention for gradients")
    if q.device.type == "cpu":
        _lib.require_cuda(q)
    run = _linear_attention_step if _lib.eager(q) else _ops.linear_attention_step
    wide = norm_eps is not None and not _norm_differentiable(norm_weight, norm_bias)   # (as in attend)
    o = run(q, k, v, log_decay, state, float(scale), wide)
    if norm_eps is not None:
        o = _normalised(o, q.dtype, norm_eps, norm_weight, norm_bias)
    return o
