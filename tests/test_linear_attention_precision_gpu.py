"""Linear attention: decays near one over long sequences (token by token, and chunk by chunk), and decays of zero in
float64, where a difference of large sums would show."""
import math

import pytest
import torch

import philtorch_b200 as ptb
from test_linear_attention_gpu import check_backward, check_forward, inputs

pytestmark = pytest.mark.gpu

# 16.5 steps of float32 below one: a factor held in a single float32 is off by half a step, 3 % of this decay, always in
# the same direction
HALF_WAY = -16.5 * 2.0 ** -24


def noise(count, largest):
    """What `count` independent roundings of float32 come to: each is off by at most half a step (2^-24 of the largest value
    there), either way; a sum of so many is above six times the root of their number once in 10^7 (Hoeffding)."""
    return 6 * math.sqrt(count) * 2.0 ** -24 * largest


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decays_near_one_token_by_token(dtype, form):
    T, H, D = 4096, 3, 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    q, k, v = randn(1, H, D).to(dtype), (0.01 * randn(T, 1, H, D)).to(dtype), (0.01 * randn(T, 1, H, D)).to(dtype)
    g = torch.tensor([HALF_WAY, 10 * HALF_WAY, 3.5 * HALF_WAY], device="cuda")
    zi = randn(1, H, D, D)
    state = zi.clone()
    step = (ptb.lti if form == "lti" else ptb.lpv).linear_attention_step
    gates = g if form == "lti" else g[None]
    for t in range(T):
        step(q, k[t], v[t], gates, state)
    weight = torch.exp(g.double() * torch.arange(T - 1, -1, -1, device="cuda")[:, None])        # (T, H)
    first = torch.exp(g.double() * T)[:, None, None]
    kw, vd = k[:, 0].double() * weight[..., None], v[:, 0].double()
    ref = first * zi[0].double() + torch.einsum("thm,thn->hmn", kw, vd)
    most = zi[0].double().abs() + torch.einsum("thm,thn->hmn", k[:, 0].double().abs(), vd.abs())
    # a token: the product of key and value, two multiply-adds
    bad = (state[0].double() - ref).abs() > noise(3 * T, most)
    assert not bad.any(), (bad.sum().item(), ((state[0].double() - ref).abs() / most).max().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decays_near_one_chunk_by_chunk(dtype):
    """A state that only decays, forward and (its gradient) backward; so many heads that no time axis is cut."""
    T, H, D, C = 32768, 160, 16, 32
    g = torch.full((H,), HALF_WAY / C, device="cuda")     # a chunk's factor lies half-way between two floats
    g[1::2] *= 5
    zero = torch.zeros(1, T, 1, D, device="cuda", dtype=dtype).expand(1, T, H, D)
    gen = torch.Generator(device="cuda").manual_seed(2)
    zi = torch.randn(1, H, D, D, generator=gen, device="cuda").requires_grad_()
    gS = torch.randn(1, H, D, D, generator=gen, device="cuda")
    _, S = ptb.lti.linear_attention(zero, zero, zero, g, zi)
    (gzi,) = torch.autograd.grad(S, zi, gS)
    factor = torch.exp(g.double() * T)[:, None, None]
    # A chunk rounds a state twice, by at most 2^-24 of it, and while nothing is added the mantissa hardly moves: the second rounding
    # may be the same in every chunk.  So one state may be off by 2 T / C roundings; but which way goes by its mantissa, that is, by
    # chance, and the mean over a head's kind of n states is below six times that over the root of n (Hoeffding): 5e-6.  A factor
    # rounded to one float moves all of them the same way, by half a step a chunk: 3e-5.
    most = 2 * (T // C) * 2.0 ** -24
    for got, start in ((S.detach(), zi.detach()), (gzi, gS)):
        off = got[0].double() / (factor * start[0].double()) - 1
        assert off.abs().max() <= 1.01 * most
        for kind in (off[::2], off[1::2]):
            assert abs(kind.mean().item()) <= 6 * most / math.sqrt(kind.numel())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_an_infinite_state_stays_infinite(dtype):
    q, k, v, _, zi, _ = inputs((1, 70, 3, 16, 16), dtype, "lti", seed=3)
    zi[0, :, 2, 3], zi[0, :, 4, 5] = float("inf"), -float("inf")
    g = torch.tensor([0.0, -1e-3, -2.5], device="cuda")
    state = zi.clone()
    for t in range(70):
        ptb.lti.linear_attention_step(q[:, t], k[:, t], v[:, t], g, state)
    _, S = ptb.lti.linear_attention(q, k, v, g, zi)
    for got in (state[0], S[0, :2]):      # (a whole chunk's decay of exp(-80) times infinity is not asked for)
        assert (got[:, 2, 3] == float("inf")).all() and (got[:, 4, 5] == -float("inf")).all()
        assert got.isfinite().sum() == got.numel() - 2 * len(got)


@pytest.mark.parametrize("zero", [-float("inf"), -1e4])
def test_decay_of_zero_in_float64(zero):
    """Weights behind a decay of zero are exponentials of differences of small sums: nothing of it is left in them."""
    q, k, v, g, zi, scale = inputs((1, 300, 2, 64, 64), torch.float64, "lpv", seed=5)
    for t in (0, 40, 41, 64, 128, 250):
        g[:, t] = zero
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = ptb.lpv.linear_attention(*leaves, scale=scale)
    det = [t.detach() for t in leaves]
    check_forward((o.detach(), S.detach()), *det, scale)
    gen = torch.Generator(device="cuda").manual_seed(6)
    go = torch.randn(o.shape, generator=gen, device="cuda", dtype=torch.float64)
    gS = torch.randn(S.shape, generator=gen, device="cuda", dtype=torch.float64)
    check_backward("lpv", torch.autograd.grad([o, S], leaves, [go, gS]), *det, scale, None, go, gS)
