"""Linear attention with a decay per token and head (gated): the recurrence of this package on a matrix state."""
from __future__ import annotations

from typing import Optional

from torch import Tensor

from ..attention import attend, attend_step

__all__ = ["linear_attention", "linear_attention_step"]


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, zi: Optional[Tensor] = None, *,
                     scale: float = 1.0, lengths: Optional[Tensor] = None, return_state: Optional[bool] = None,
                     norm_eps: Optional[float] = None, norm_weight: Optional[Tensor] = None,
                     norm_bias: Optional[Tensor] = None):
    """``S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T``, ``o[t] = scale * q[t]^T S[t]`` for whole sequences.

    Args:
        q, k: (B, T, H, Dk); v: (B, T, H, Dv); one type out of float32, float64, float16, bfloat16 (sums
            and states in float32, or float64 for float64), Dk and Dv at most 128.  The last axis is read dense,
            the others with any strides (views of a fused projection, ``expand``-ed heads).
        log_decay: (B, T, H), the logarithm of a decay per token and head; ``-inf`` starts the sequence anew at that token;
            float32 (float64 beside float64), at most 0; ``lti.linear_attention`` takes one decay per head.
        zi: (B, H, Dk, Dv) initial state of log_decay's type; None: zeros.
        scale: factor of the output.
        lengths: (B,) int32 or int64: tokens from lengths[b] on are not read, leave the state as it was and
            give zeros (a padded batch); values outside 0..T are clamped.
        return_state: whether the state after the last token is returned too; by default when zi is given.
        norm_eps, norm_weight, norm_bias: with norm_eps, the output of each head is normalised by
            ``layer_norm`` (one group of Dv channels per head; weight and bias (H * Dv,)).  Without gradients it
            reads the sums before they are rounded to q's type, with gradients the rounded output (the two operators
            one after the other); the zeros behind a sequence's end become norm_bias.

    bfloat16 tensors of more than 32 tokens run on the tensor cores: weights and states are rounded to bfloat16
    once where they enter a product (sums, states and the decays' gradient are float32), and an infinite value
    counts as NaN.  Infinite and NaN values reach no output before their token and no gradient of q, k, v that does
    not depend on them; in the gradient of log_decay they reach the chunk of tokens (up to 128) that they are in.

    Returns:
        o (B, T, H, Dv), or (o, state).  Differentiable once in q, k, v, log_decay, zi (and the norm's
        parameters); forward-mode tangents are refused.
    """
    if log_decay.dim() != 3:
        raise ValueError(f"log_decay must be (batch, time, heads), got {tuple(log_decay.shape)}")
    return attend(q, k, v, log_decay, zi, scale, lengths, return_state, norm_eps, norm_weight, norm_bias)


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *, scale: float = 1.0,
                          norm_eps: Optional[float] = None, norm_weight: Optional[Tensor] = None,
                          norm_bias: Optional[Tensor] = None) -> Tensor:
    """One token of every sequence: ``state`` (B, H, Dk, Dv) moves on IN PLACE, and the token's output (B, H, Dv)
    is returned.  q, k: (B, H, Dk); v: (B, H, Dv); log_decay: (B, H); the other arguments as in
    ``linear_attention`` (the norm reads the sums before they are rounded).  Not differentiable (serving).
    """
    if log_decay.dim() != 2:
        raise ValueError(f"log_decay must be (batch, heads), got {tuple(log_decay.shape)}")
    return attend_step(q, k, v, log_decay, state, scale, norm_eps, norm_weight, norm_bias)
