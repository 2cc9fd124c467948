"""The single-token form: what it refuses leaves the state alone, and its normalised read-out is that of a prompt."""
import pytest
import torch

import philtorch_b200 as ptb
import linear_attention_common as la
from test_linear_attention_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["lti", "lpv"])
def test_a_refused_step_leaves_the_state(form):
    q, k, v, g, zi, _ = inputs((2, 1, 3, 16, 8), torch.bfloat16, form, seed=61)
    side = ptb.lti if form == "lti" else ptb.lpv
    w = torch.ones(24, device="cuda", dtype=torch.bfloat16)
    token = [t[:, 0] for t in (q, k, v)] + [g if form == "lti" else g[:, 0]]
    for norm, error in ((dict(norm_weight=w), ValueError), (dict(norm_bias=w), ValueError),
                        (dict(norm_eps=1e-5, norm_weight=w[:23]), RuntimeError), (dict(norm_eps=1e-5, norm_bias=w.half()), RuntimeError),
                        (dict(norm_eps=1e-5, norm_weight=w.cpu()), RuntimeError),
                        (dict(norm_eps=1e-5, norm_weight=w, norm_bias=w.float()), RuntimeError)):
        state = zi.clone()
        with pytest.raises(error):
            side.linear_attention_step(*token, state, **norm)
        assert torch.equal(state, zi)
        with pytest.raises(error):
            side.linear_attention(q, k, v, g, zi, **norm)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("size", [(3, 70, 2, 64, 64), (2, 9, 3, 33, 21)])
def test_normalised_tokens(size, dtype):
    """A padded batch of prompts, then token by token, read-out normalised: the norm reads the sums before they are rounded.
    An error d of o moves a normalised value xh by at most r (d + mean d + |xh| mean(|xh| d)) in first order; the fifth on top
    is for what is of second order."""
    B, T, H, Dk, Dv = size
    more = 5
    q, k, v, g, _, scale = inputs((B, T + more, H, Dk, Dv), dtype, "lpv", seed=62, state=False)
    gen = torch.Generator(device="cuda").manual_seed(63)
    w = (1 + torch.rand(H * Dv, generator=gen, device="cuda", dtype=torch.float64)).to(dtype)
    b = torch.randn(H * Dv, generator=gen, device="cuda", dtype=torch.float64).to(dtype)
    _, state = ptb.lpv.linear_attention(q[:, :T], k[:, :T], v[:, :T], g[:, :T], scale=scale, return_state=True)
    u, unit = torch.finfo(dtype).eps / 2, torch.finfo(state.dtype).eps / 2
    wide, bias = w.double().view(H, Dv), b.double().view(H, Dv)
    for t in range(T, T + more):
        before = state.clone()
        token = [x[:, t] for x in (q, k, v, g)]
        o = ptb.lpv.linear_attention_step(*token, state, scale=scale, norm_eps=1e-3, norm_weight=w, norm_bias=b)
        assert o.dtype == dtype and o.shape == (B, H, Dv)
        one = [x.unsqueeze(1) for x in token]
        ro, _ = la.forward(*one, before, scale, None)
        bo, _ = la.forward(*la.absolute(*one[:3]), one[3], before.abs(), scale, None)
        d = la.roundings(*one[1:3]) * unit * bo        # no rounding to the type
        c = ro - ro.mean(-1, keepdim=True)
        r = (c.square().mean(-1, keepdim=True) + 1e-3).rsqrt()
        xh = c * r
        ref = xh * wide + bias
        moved = r * (d + d.mean(-1, keepdim=True) + xh.abs() * (xh.abs() * d).mean(-1, keepdim=True))
        tol = u * ref.abs() + 1.2 * wide * moved + (Dv + 16) * unit * (wide * (xh.abs() + r * ro.abs().mean(-1, keepdim=True)) + ref.abs())
        bad = (o.unsqueeze(1).double() - ref).abs() > tol + torch.finfo(dtype).tiny
        assert not bad.any(), ((o.unsqueeze(1).double() - ref).abs() / tol).max().item()
        plain = ptb.lpv.linear_attention_step(*token, before, scale=scale)
        assert torch.equal(before, state) and plain.dtype == dtype
