"""Calls from threads that have made no CUDA call yet: an autograd thread, or a server's worker, whose memory all comes from the
allocator's cache."""
import threading

import pytest
import torch

import philtorch_b200 as ptb

pytestmark = pytest.mark.gpu


def in_fresh_threads(fn, count=1):
    got, failed = [], []

    def body():
        try:
            got.append(fn())
        except Exception as e:   # noqa: BLE001  shown by the test
            failed.append(e)

    threads = [threading.Thread(target=body) for _ in range(count)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("count", [1, 3])
def test_linear_attention(count):
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, go = (torch.randn(1, 300, 2, 64, generator=gen, device="cuda").bfloat16() for _ in range(4))
    g = -torch.rand(1, 300, 2, generator=gen, device="cuda")

    def both():
        o, S = torch.ops.philtorch_b200.linear_attention(q, k, v, g, None, None, 0.5, True)
        return [o, S, *torch.ops.philtorch_b200.linear_attention_bwd(q, k, v, g, None, None, 0.5, go, None, *[True] * 4, False)]

    want = both()
    kept = [both() for _ in range(4)]   # room for every thread in the allocator's cache
    torch.cuda.synchronize()
    del kept
    for got in in_fresh_threads(both, count):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_comb_filter():
    x = torch.randn(16, 38400, device="cuda")
    c = torch.rand(16, device="cuda") * 1.8 - 0.9
    want = ptb.lti.comb_filter(c, 600, x)
    kept = [ptb.lti.comb_filter(c, 600, x) for _ in range(2)]
    torch.cuda.synchronize()
    del kept
    (got,) = in_fresh_threads(lambda: ptb.lti.comb_filter(c, 600, x))
    assert torch.equal(got, want)
