"""The tensor-core kernels under the shortest limit for their waits: a load or a product takes microseconds, so nothing gives up, and the
results are those of the default limit."""
import pytest
import torch

import philtorch_b200 as ptb
from philtorch_b200 import _lib
from test_linear_attention_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [(2, 300, 2, 64, 72), (1, 5000, 2, 128, 128), (2, 2000, 40, 16, 64)])
def test_shortest_limit(size):
    q, k, v, g, zi, scale = inputs(size, torch.bfloat16, "lpv", seed=81)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]

    def run():
        o, S = ptb.lpv.linear_attention(*leaves, scale=scale)
        return [o, S, *torch.autograd.grad([o, S], leaves, [torch.ones_like(o), torch.ones_like(S)])]

    want = run()
    assert _lib.lib.ptb_set_wait_limit_ms(1) == 0
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        assert _lib.lib.ptb_set_wait_limit_ms(2000) == 0
    ptb.check_errors()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
