"""Layer norm over groups of channels: the read-out normalisation of ``linear_attention`` (one group per
head), and the norm over whole rows (one group)."""
from __future__ import annotations

from typing import Any, Optional

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib, ptr
from .ops import _LIB, _TAGS

__all__ = ["LayerNorm", "layer_norm", "MAX_WIDTH"]

MAX_WIDTH = 16384
_CODES = {torch.float32: _lib.PTB_F32, torch.float64: _lib.PTB_F64, torch.float16: _lib.PTB_F16,
          torch.bfloat16: _lib.PTB_BF16}

_LIB.define("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, int groups, ScalarType? out=None) "
            "-> (Tensor, Tensor)",
            tags=_TAGS)
_LIB.define("layer_norm_bwd(Tensor x, Tensor? weight, Tensor? bias, Tensor stats, Tensor grad_y, int groups, "
            "bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)", tags=_TAGS)


def check_parameters(C: int, dtype: torch.dtype, weight: Optional[Tensor], bias: Optional[Tensor], groups: int,
                     out: Optional[torch.dtype] = None) -> None:
    """Whether rows of C channels of ``dtype`` can be normalised with these parameters (results in ``out``)."""
    # the common case in one expression: the explanations below cost more host time than the launch
    dt = dtype if out is None else out
    if (1 <= groups <= 65535 and C and C % groups == 0 and C // groups <= MAX_WIDTH
            and (weight is None or (weight.shape == (C,) and weight.dtype == dt))
            and (bias is None or (bias.shape == (C,) and bias.dtype == dt)) and (out is None or dtype in (dt, torch.float32))):
        return
    torch._check(1 <= groups <= 65535 and C % groups == 0 and C > 0,
                 lambda: f"the last axis ({C}) must be a multiple of groups ({groups}, at most 65535)")
    torch._check(C // groups <= MAX_WIDTH, lambda: f"groups of {C // groups} channels: the kernels cover 1..{MAX_WIDTH}.")
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    torch._check(dt == dtype or (dtype == torch.float32 and dt in (torch.float16, torch.bfloat16)),
                 lambda: f"no results in {dt} of {dtype} tensors")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            torch._check(tuple(p.shape) == (C,), lambda: f"{name} must be ({C},), got {tuple(p.shape)}")
            torch._check(p.dtype in (dt, wide), lambda: f"{name} must be {dt} or {wide}, got {p.dtype}")
    if weight is not None and bias is not None:
        torch._check(weight.dtype == bias.dtype,
                     lambda: f"weight and bias must have the same type, got {weight.dtype} and {bias.dtype}")


def _check(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], groups: int, out: Optional[torch.dtype] = None) -> None:
    torch._check(x.dim() >= 1, lambda: "x must have at least one axis")
    check_parameters(x.shape[-1], x.dtype, weight, bias, groups, out)


def _code(t: Tensor) -> int:
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise RuntimeError(f"layer_norm takes float32, float64, float16 and bfloat16 tensors, got {t.dtype}") from None


def _as_rows(t: Tensor) -> Tensor:
    """(rows, channels) with dense channels; a view where the strides allow it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _wide(weight: Optional[Tensor], bias: Optional[Tensor]) -> int:
    p = weight if weight is not None else bias
    return int(p is not None and p.dtype in (torch.float32, torch.float64))


def _stats_dtype(x: Tensor) -> torch.dtype:
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _layer_norm(x, weight, bias, eps, groups, out=None):
    _check(x, weight, bias, groups, out)
    dev = _lib.require_cuda(x, weight, bias)
    rows = _as_rows(x)
    R, C = rows.shape
    w, b = (None if p is None else p.contiguous() for p in (weight, bias))
    y = x.new_empty(x.shape, dtype=out)
    stats = x.new_empty((2, R, groups), dtype=_stats_dtype(x))
    if R:
        at = stats.data_ptr()
        _lib.launch(lib.ptb_layer_norm_fwd, dev, _code(x), R, groups, C // groups, ptr(rows), rows.stride(0), ptr(w), ptr(b),
                    _wide(weight, bias), eps, _code(y), ptr(y), at, at + R * groups * stats.element_size())
    return y, stats


_ws_bytes: dict = {}


def _layer_norm_bwd(x, weight, bias, stats, grad_y, groups, need_x, need_weight, need_bias):
    dev = _lib.require_cuda(x, weight, bias, stats, grad_y)
    rows, gy = _as_rows(x), _as_rows(grad_y)
    R, C = rows.shape
    w = None if weight is None else weight.contiguous()
    gx = x.new_empty(x.shape if need_x else (0,))
    gw = weight.new_empty((C,)) if need_weight else x.new_empty(0)
    gb = bias.new_empty((C,)) if need_bias else x.new_empty(0)
    if R:
        code, width, ws = _code(x), C // groups, 0
        if need_weight or need_bias:
            key = (code, R, groups, width)
            ws = _ws_bytes.get(key)
            if ws is None:
                if len(_ws_bytes) > 4096:   # a server sees many sizes
                    _ws_bytes.clear()
                ws = _ws_bytes[key] = lib.ptb_layer_norm_bwd_workspace_bytes(code, R, groups, width)
        at = stats.data_ptr()
        _lib.call(lib.ptb_layer_norm_bwd, dev, R, C, code, R, groups, width, ptr(rows), rows.stride(0), ptr(w),
                  _wide(weight, bias), at, at + R * groups * stats.element_size(), ptr(gy), gy.stride(0),
                  ptr(gx) if need_x else None, ptr(gw) if need_weight else None, ptr(gb) if need_bias else None, ws_bytes=ws)
    else:
        gw.zero_()
        gb.zero_()
    return gx, gw, gb


_LIB.impl("layer_norm", _layer_norm, "CUDA")
_LIB.impl("layer_norm_bwd", _layer_norm_bwd, "CUDA")


@torch.library.register_fake("philtorch_b200::layer_norm")
def _(x, weight, bias, eps, groups, out=None):
    _check(x, weight, bias, groups, out)
    return x.new_empty(x.shape, dtype=out), x.new_empty((2, x.numel() // x.shape[-1], groups), dtype=_stats_dtype(x))


@torch.library.register_fake("philtorch_b200::layer_norm_bwd")
def _(x, weight, bias, stats, grad_y, groups, need_x, need_weight, need_bias):
    C = x.shape[-1]
    return (x.new_empty(x.shape if need_x else (0,)), weight.new_empty((C,)) if need_weight else x.new_empty(0),
            bias.new_empty((C,)) if need_bias else x.new_empty(0))


_ops = torch.ops.philtorch_b200


def _forward(x, weight, bias, eps, groups):
    if x.device.type == "cpu":
        _lib.require_cuda(x)
    return (_layer_norm if _lib.eager(x) else _ops.layer_norm)(x, weight, bias, eps, groups)


def _backward(ctx: Any, grad_y: Tensor):
    x, weight, bias, stats = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    run = _layer_norm_bwd if _lib.eager(x) else _ops.layer_norm_bwd
    gx, gw, gb = run(x, weight, bias, stats, grad_y, ctx.groups, *need)
    return gx if need[0] else None, gw if need[1] else None, gb if need[2] else None, None, None


_backward_once = once_differentiable(_backward)


class LayerNorm(Function):
    """(x, weight or None, bias or None, eps, groups) -> y; first derivatives."""

    @staticmethod
    def forward(ctx: Any, x, weight, bias, eps: float, groups: int):
        y, stats = _forward(x, weight, bias, eps, groups)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups = groups
        return y

    @staticmethod
    def backward(ctx: Any, grad_y: Tensor):
        # (the guard against second derivatives is only needed, and only paid, where a graph is being recorded)
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad_y)


def layer_norm_of_sums(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, groups: int,
                       out: torch.dtype) -> Tensor:
    """``layer_norm`` of float32 sums with results (and parameters) in a 2-byte type; no gradients."""
    return (_layer_norm if _lib.eager(x) else _ops.layer_norm)(x, weight, bias, eps, groups, out)[0]


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               groups: int = 1) -> Tensor:
    """Normalises groups of consecutive channels of the last axis to mean zero and variance one, then applies
    a weight and a bias per channel.

    Args:
        x: (..., C), CUDA, float32, float64, float16 or bfloat16 (statistics in float32 or better).
        weight, bias: (C,) of x's type or float32 (float64 beside float64), or None.
        eps: added to the variance.
        groups: the last axis is cut into this many groups of C / groups <= 16384 channels; 1: whole rows.

    Returns:
        Tensor of x's shape and type.  Differentiable once in x, weight and bias; their gradients are sums
        in a fixed order (bit-reproducible).  Forward-mode tangents are refused.
    """
    _lib.refuse_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return LayerNorm.apply(x, weight, bias, float(eps), int(groups))
    return _forward(x, weight, bias, float(eps), int(groups))[0]
