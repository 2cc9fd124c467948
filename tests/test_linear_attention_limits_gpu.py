"""Linear attention at the ends of its ranges: very many sequences or heads, no tokens, graphs that share their memory, transforms
that would write a state more than once."""
import pytest
import torch

import philtorch_b200 as ptb
from test_linear_attention_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("axis", ["batch", "heads"])
@pytest.mark.parametrize("T", [20, 40])
def test_more_than_65535(axis, T):
    n, D = 70_000, 8
    gen = torch.Generator(device="cuda").manual_seed(91)
    x = torch.randn(n, T, D, generator=gen, device="cuda").bfloat16()
    few = torch.tensor([0, 1, 65_535, 65_536, n - 1], device="cuda")

    def run(x):
        count = len(x)
        a = x[:, :, None] if axis == "batch" else x.transpose(0, 1)[None]
        a = a.contiguous().requires_grad_()
        g = torch.full((1 if axis == "batch" else count,), -0.1, device="cuda", requires_grad=True)
        o, S = ptb.lti.linear_attention(a, a, a, g, return_state=True)
        (ga,) = torch.autograd.grad([o, S], a, [torch.ones_like(o), torch.ones_like(S)])
        state = S.detach().clone()
        with torch.no_grad():
            y = ptb.lti.linear_attention_step(a[:, 0], a[:, 0], a[:, 0], g, state)
        if axis == "batch":
            return [t.detach() for t in (o, S, ga, state, y)]
        return [o.detach()[0].transpose(0, 1), S.detach()[0], ga[0].transpose(0, 1), state[0], y[0]]

    for whole, part in zip(run(x), run(x[few])):
        assert torch.equal(whole[few], part)
    ptb.check_errors()


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_no_tokens(dtype, form):
    q, k, v, g, zi, _ = inputs((2, 0, 3, 16, 8), dtype, form)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = (ptb.lti if form == "lti" else ptb.lpv).linear_attention(*leaves)
    grads = torch.autograd.grad([o, S], leaves, [torch.ones_like(o), 2 * torch.ones_like(S)])
    assert all(t.shape == x.shape and (t == 0).all() for t, x in zip(grads[:4], leaves)) and (grads[4] == 2).all()


def test_two_graphs_of_one_memory_pool():
    sets = [inputs(size, torch.bfloat16, "lpv", seed=s) for size, s in (((1, 1300, 2, 64, 64), 92), ((2, 200, 3, 60, 33), 93))]
    gos = [torch.randn(s[2].shape, device="cuda").bfloat16() for s in sets]

    def step(s, go):
        leaves = [t.detach().requires_grad_() for t in s[:5]]
        o, S = ptb.lpv.linear_attention(*leaves, scale=s[5])
        return [o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [go, torch.ones_like(S)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(s, go) for s, go in zip(sets, gos)]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s, go in zip(sets, gos):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(step(s, go))
    for _ in range(3):
        for gr, out, w in zip(graphs, outs, want):
            for t in out:
                t.fill_(7)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    ptb.check_errors()


def test_a_step_under_vmap_is_refused():
    q, k, v, g, zi, _ = inputs((2, 1, 3, 16, 8), torch.float32, "lpv")
    states = torch.stack([zi, zi])
    before = states.clone()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: ptb.lpv.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], s))(states)
    with pytest.raises(RuntimeError):      # one state, several tokens: written more than once
        torch.func.vmap(lambda x: ptb.lpv.linear_attention_step(x, k[:, 0], v[:, 0], g[:, 0], zi))(torch.stack([q[:, 0]] * 2))
    assert torch.equal(states, before) and torch.equal(zi, before[0])
