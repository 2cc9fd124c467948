"""Padded batches of long rows: the time axis is cut, and whole segments lie behind a sequence's end."""
import pytest
import torch

import philtorch_b200 as ptb
from test_linear_attention_gpu import check_backward, check_forward, inputs

pytestmark = pytest.mark.gpu


def poison():
    """Freed memory full of NaN, large blocks and small ones: workspace that is read before it is written shows."""
    kept = [torch.full((1 << 28,), float("nan"), device="cuda")]
    kept += [torch.full((1 << n,), float("nan"), device="cuda") for n in range(8, 18) for _ in range(8)]
    torch.cuda.synchronize()
    del kept


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("size,dtype", [((6, 2500, 2, 64, 64), torch.bfloat16), ((6, 2500, 1, 128, 72), torch.bfloat16),
                                        ((6, 2300, 1, 20, 33), torch.bfloat16), ((6, 700, 2, 64, 40), torch.float32),
                                        ((6, 700, 1, 33, 128), torch.float16), ((6, 700, 1, 16, 24), torch.float64)])
def test_whole_segments_behind_the_end(size, dtype, form):
    B, T, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs(size, dtype, form, seed=31)
    lengths = torch.tensor([T, 0, 1, 130, T // 2, T // 3 + 1], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(32)
    go = torch.randn(B, T, H, Dv, generator=gen, device="cuda").to(dtype)
    gS = torch.randn(zi.shape, generator=gen, device="cuda").to(zi.dtype)
    clean = [t.clone() for t in (q, k, v, g)]
    clean_go = go.clone()
    for t in (q, k, v, go) + ((g,) if form == "lpv" else ()):
        for b, n in enumerate(lengths.tolist()):
            t[b, n:] = float("nan")
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    side = ptb.lti if form == "lti" else ptb.lpv
    poison()
    o, S = side.linear_attention(*leaves, scale=scale, lengths=lengths)
    check_forward((o.detach(), S.detach()), *clean, zi.detach(), scale, lengths)
    assert torch.equal(S[1], zi[1])
    for b, n in enumerate(lengths.tolist()):
        assert (o[b, n:] == 0).all()
    poison()
    grads = torch.autograd.grad([o, S], leaves, [go, gS], retain_graph=True)
    check_backward(form, grads, *clean, zi.detach(), scale, lengths, clean_go, gS)
    for t in grads[:3] + ((grads[3],) if form == "lpv" else ()):
        for b, n in enumerate(lengths.tolist()):
            assert (t[b, n:] == 0).all()
    poison()
    some = torch.autograd.grad([o, S], leaves[:3] + leaves[4:], [go, gS])     # without the decays' gradient: other kernels
    check_backward(form, [*some[:3], None, some[3]], *clean, zi.detach(), scale, lengths, clean_go, gS)
    ptb.check_errors()
