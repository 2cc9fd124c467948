"""Linear attention with decays from its recurrence, token by token in float64, with the bounds that the tests' tolerances
count in: every result comes with the sum of the absolute values of its terms."""
import torch


def decays(g, B, T, H, lengths):
    """exp(g) as (B,T,H) float64, 1 behind a sequence's end, and the mask of the tokens that count."""
    a = g.double().exp().expand(B, T, H).clone()
    on = torch.ones(B, T, dtype=torch.bool, device=g.device)
    if lengths is not None:
        on = torch.arange(T, device=g.device)[None] < lengths.to(g.device)[:, None]
    a[~on] = 1.0
    return a, on


def _clean(t, on):
    t = t.double().clone()
    t[~on] = 0.0
    return t


def forward(q, k, v, g, zi, scale, lengths):
    B, T, H, Dk = q.shape
    a, on = decays(g, B, T, H, lengths)
    q, k, v = (_clean(t, on) for t in (q, k, v))
    S = torch.zeros(B, H, Dk, v.shape[-1], dtype=torch.float64, device=q.device) if zi is None else zi.double().clone()
    o = torch.zeros_like(v)
    for t in range(T):
        S = S * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * (q[:, t, :, :, None] * S).sum(-2)
    o[~on] = 0.0
    return o, S


def backward(q, k, v, g, zi, scale, lengths, go, gzf):
    """gq, gk, gv, gg (B,T,H), gzi; gg[t] = <R[t], a[t] S[t-1]>, straight from the two sequences of states."""
    B, T, H, Dk = q.shape
    a, on = decays(g, B, T, H, lengths)
    q, k, v, go = (_clean(t, on) for t in (q, k, v, go))
    S = torch.zeros(B, H, Dk, v.shape[-1], dtype=torch.float64, device=q.device) if zi is None else zi.double().clone()
    gq, decayed = torch.zeros_like(q), []
    for t in range(T):
        S = S * a[:, t, :, None, None]
        decayed.append(S)
        S = S + k[:, t, :, :, None] * v[:, t, :, None, :]
        gq[:, t] = scale * (S * go[:, t, :, None, :]).sum(-1)
    R = torch.zeros_like(S) if gzf is None else gzf.double().clone()
    gk, gv = torch.zeros_like(k), torch.zeros_like(v)
    gg = torch.zeros(B, T, H, dtype=torch.float64, device=q.device)
    for t in range(T - 1, -1, -1):
        R = R + scale * q[:, t, :, :, None] * go[:, t, :, None, :]
        gk[:, t] = (R * v[:, t, :, None, :]).sum(-1)
        gv[:, t] = (R * k[:, t, :, :, None]).sum(-2)
        gg[:, t] = (R * decayed[t]).sum((-1, -2))
        R = R * a[:, t, :, None, None]
    for x in (gq, gk, gv, gg):
        x[~on] = 0.0
    return gq, gk, gv, gg, R


def absolute(*tensors):
    return tuple(None if t is None else t.abs() for t in tensors)


# A result in float32 is a sum of products of at most Dk * T terms in three nested sums (over the head's channels, the
# tokens of a chunk, the chunks): at most D + T roundings meet one term, and its weight, an exponential of a
# difference d of log decays, is off by (|d| + 2) roundings, with |d| <= 104 for any weight float32 can hold.
def roundings(q, v):
    return 2 * max(q.shape[-1], v.shape[-1]) + q.shape[1] + 128


def tolerance(ref, bound, dtype, q, v):
    """Elementwise: one rounding of the result to its type; in a 2-byte type one more of each weight and state that
    enters a product; roundings() of float32 (or float64) arithmetic on the sum of the terms' absolute values."""
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    unit, u = torch.finfo(wide).eps / 2, torch.finfo(dtype).eps / 2
    tol = u * ref.abs() + roundings(q, v) * unit * bound
    if dtype in (torch.float16, torch.bfloat16):
        tol = tol + 1.01 * u * bound + torch.finfo(dtype).tiny
    return tol + torch.finfo(wide).tiny


def decay_bound(q, k, v, g, zi, scale, lengths, go, gzf, window=128):
    """Sum of the absolute terms of gg: the pairs across a token, and, of the sums that start anew in every
    chunk (at most `window` tokens), the pairs around it that cancel."""
    aq, ak, av, azi, ago, agzf = absolute(q, k, v, zi, go, gzf)
    gq, gk, _, gg, _ = backward(aq, ak, av, g, azi, abs(scale), lengths, ago, agzf)
    _, on = decays(g, *q.shape[:3], lengths)
    per = (_clean(aq, on) * gq).sum(-1) + (_clean(ak, on) * gk).sum(-1)
    T = q.shape[1]
    c = torch.cat([torch.zeros_like(per[:, :1]), per.cumsum(1)], 1)
    t = torch.arange(T, device=q.device)
    return gg + c[:, (t + window).clamp(max=T)] - c[:, (t - window).clamp(min=0)]
