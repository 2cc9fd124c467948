"""The single-token form: what it refuses leaves the state alone."""
import pytest
import torch

import philtorch_b200 as ptb
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
