"""Linear attention: an infinite or NaN value reaches what the recurrence lets it reach, and nothing else: no output before its
token, no gradient behind it, no other column and no other head."""
import pytest
import torch

import philtorch_b200 as ptb
from test_linear_attention_gpu import inputs

pytestmark = pytest.mark.gpu

# one short sequence, several chunks, a row cut into segments, two slices of columns, rows off the 16-byte boundaries
SIZES = [(1, 20, 2, 16, 24), (1, 300, 2, 64, 72), (1, 1500, 2, 128, 128), (1, 200, 2, 33, 65)]


def places(T):
    return sorted({0, 5, 15, T // 2 + 3, T - 2, T - 1} | {s for s in (31, 33, 100, 127, 128, 131) if s < T})


def same(got, clean):
    assert torch.equal(got, clean)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs(dtype, size, value):
    B, T, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs(size, dtype, "lpv", seed=41)
    run = lambda *a: ptb.lpv.linear_attention(*a, zi, scale=scale)   # noqa: E731
    clean, clean_state = run(q, k, v, g)
    for s in places(T):
        for name in ("q", "k", "v", "g"):
            args = dict(q=q, k=k, v=v, g=g)
            at = args[name] = args[name].clone()
            c = 7
            if name == "g":
                at[0, s, 0] = float("nan")
            else:
                at[0, s, 0, c] = value
            o, S = run(*args.values())
            same(o[:, :, 1], clean[:, :, 1])
            same(S[:, 1], clean_state[:, 1])
            same(o[:, :s, 0], clean[:, :s, 0])
            if name == "q":
                same(o[:, s + 1:], clean[:, s + 1:])
                same(S, clean_state)
                assert not o[0, s, 0].isfinite().any()
            elif name == "v":
                others = [n for n in range(Dv) if n != c]
                same(o[..., others], clean[..., others])
                same(S[..., others], clean_state[..., others])
                assert not o[0, s:, 0, c].isfinite().any() and not S[0, 0, :, c].isfinite().any()
            else:
                assert not o[0, s:, 0].isfinite().any()
                assert not (S[0, 0, c] if name == "k" else S[0, 0]).isfinite().any()
    ptb.check_errors()


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(dtype, size, decay):
    """decay: with the gradient of the log decays (other kernels), whose sums over a chunk are not separated by token."""
    B, T, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs(size, dtype, "lpv", seed=42)
    gen = torch.Generator(device="cuda").manual_seed(43)
    go = torch.randn(B, T, H, Dv, generator=gen, device="cuda").to(dtype)

    def run(q, k, v, go):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, g)[:4 if decay else 3]]
        o = ptb.lpv.linear_attention(*leaves, *([] if decay else [g]), scale=scale)
        return torch.autograd.grad(o, leaves, go)

    clean = run(q, k, v, go)
    c = 7
    for s in places(T):
        for name in ("q", "k", "v", "go"):
            args = dict(q=q, k=k, v=v, go=go)
            at = args[name] = args[name].clone()
            at[0, s, 0, c] = float("nan")
            got = run(*args.values())
            for a, b in zip(got, clean):
                same(a[:, :, 1], b[:, :, 1])
            (dq, dk, dv), (cq, ck, cv) = got[:3], clean[:3]
            rest_k, rest_v = [m for m in range(Dk) if m != c], [n for n in range(Dv) if n != c]
            if name == "q":
                same(dq, cq)
                same(dk[..., rest_k], ck[..., rest_k])
                same(dk[:, s + 1:], ck[:, s + 1:])
                same(dv[:, s + 1:], cv[:, s + 1:])
                assert dk[0, :s + 1, 0, c].isnan().all() and dv[0, :s + 1, 0].isnan().all()
            elif name == "k":
                same(dk, ck)
                same(dq[..., rest_k], cq[..., rest_k])
                same(dq[:, :s], cq[:, :s])
                same(dv[:, :s], cv[:, :s])
                same(dv[:, s + 1:], cv[:, s + 1:])
                assert dq[0, s:, 0, c].isnan().all() and dv[0, s, 0].isnan().all()
            elif name == "v":
                same(dv, cv)
                same(dq[:, :s], cq[:, :s])
                same(dk[:, :s], ck[:, :s])
                same(dk[:, s + 1:], ck[:, s + 1:])
                assert dq[0, s:, 0].isnan().all() and dk[0, s, 0].isnan().all()
            else:
                same(dq[:, :s], cq[:, :s])
                same(dq[:, s + 1:], cq[:, s + 1:])
                same(dk[:, s + 1:], ck[:, s + 1:])
                same(dv[..., rest_v], cv[..., rest_v])
                same(dv[:, s + 1:], cv[:, s + 1:])
                assert dq[0, s, 0].isnan().all() and dk[0, :s + 1, 0].isnan().all() and dv[0, :s + 1, 0, c].isnan().all()
    ptb.check_errors()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("size", [(2, 1500, 3, 64, 128), (3, 1300, 32, 16, 128), (2, 700, 40, 128, 20)])
def test_many_at_once(size, norm):
    """NaN in many chunks and columns, lengths that end inside a chunk: each column of a head is as it was up to its first one."""
    B, T, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs(size, torch.bfloat16, "lpv", seed=44)
    lengths = torch.tensor([T, T - 130, T - 1][:B], device="cuda")
    run = lambda v: ptb.lpv.linear_attention(q, k, v, g, zi, scale=scale, lengths=lengths)   # noqa: E731
    clean, clean_state = run(v)
    gen = torch.Generator(device="cuda").manual_seed(45)
    odd = torch.rand(B, T, H, Dv, generator=gen, device="cuda") < 4 / T      # about four in a column
    odd &= torch.arange(T, device="cuda")[None, :, None, None] < lengths[:, None, None, None]
    o, S = run(torch.where(odd, torch.full_like(v, float("nan")), v))
    seen = odd.int().cumsum(1) > 0
    behind = torch.arange(T, device="cuda")[None, :, None, None] >= lengths[:, None, None, None]
    want = torch.where(seen & ~behind, torch.full_like(clean, float("nan")), clean)
    assert torch.equal(o.isnan(), want.isnan()) and torch.equal(o.nan_to_num(), want.nan_to_num())
    column = seen[:, -1][:, :, None].expand_as(S)
    assert S[column].isnan().all() and torch.equal(S[~column], clean_state[~column])
    if norm:      # a normalised row is NaN where one of its channels is
        run = lambda v: ptb.lpv.linear_attention(q, k, v, g, zi, scale=scale, lengths=lengths, norm_eps=1e-5)[0]   # noqa: E731
        y, plain = run(torch.where(odd, torch.full_like(v, float("nan")), v)), run(v)
        rows = (seen & ~behind).any(-1)
        assert y[rows].isnan().all() and torch.equal(y[~rows], plain[~rows])
    ptb.check_errors()
