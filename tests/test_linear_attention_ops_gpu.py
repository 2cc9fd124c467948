"""The ops of linear attention and layer norm under the machinery of torch: schemas and shape rules, a compiler, vmap, and the
transforms that are refused."""
import pytest
import torch

import philtorch_b200 as ptb

pytestmark = pytest.mark.gpu


def tensors(dtype=torch.bfloat16, T=70):
    gen = torch.Generator(device="cuda").manual_seed(51)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")   # noqa: E731
    q, k, v = randn(2, T, 3, 16).to(dtype), randn(2, T, 3, 16).to(dtype), randn(2, T, 3, 24).to(dtype)
    return q, k, v, -torch.rand(2, T, 3, generator=gen, device="cuda"), randn(2, 3, 16, 24), randn(72).to(dtype), randn(72).to(dtype)


def test_opcheck():
    ops, tests = torch.ops.philtorch_b200, ("test_schema", "test_faketensor")
    q, k, v, g, zi, w, b = tensors()
    n = torch.tensor([70, 11], device="cuda")
    check = lambda op, *args: torch.library.opcheck(op, args, test_utils=tests)   # noqa: E731
    for init, lengths, want, wide in ((None, None, False, False), (zi, n, True, False), (zi, None, True, True)):
        check(ops.linear_attention, q, k, v, g, init, lengths, 0.5, want, wide)
    for need in ((True,) * 5, (True, False, True, False, False), (False, False, False, True, True)):
        check(ops.linear_attention_bwd, q, k, v, g, zi, n, 0.5, v, zi, *need)
    check(ops.linear_attention_bwd, q, k, v, g[0, 0], None, None, 0.5, v, None, True, True, True, True, False)
    check(ops.linear_attention_step, q[:, 0], k[:, 0], v[:, 0], g[:, 0], zi.clone(), 0.5)
    x = v.flatten(-2)
    for weight, bias in ((w, b), (None, None), (w.float(), None)):
        check(ops.layer_norm, x, weight, bias, 1e-5, 3)
    check(ops.layer_norm, x.float(), w, b, 1e-5, 3, torch.bfloat16)
    _, stats = ops.layer_norm(x, w, b, 1e-5, 3)
    for need in ((True, True, True), (True, False, False), (False, True, False)):
        check(ops.layer_norm_bwd, x, w, b, stats, x, 3, *need)
    ptb.check_errors()


def test_compiled_step():
    """A training step and a token under torch.compile: the values of the eager calls."""
    q, k, v, g, zi, w, b = tensors()
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi, w, b)]

    def step(q, k, v, g, zi, w, b):
        return ptb.lpv.linear_attention(q, k, v, g, zi, scale=0.5, norm_eps=1e-5, norm_weight=w, norm_bias=b)

    def both(fn):
        o, S = fn(*leaves)
        return [o, S, *torch.autograd.grad([o, S], leaves, [torch.ones_like(o), torch.ones_like(S)])]

    eager = both(step)
    got = both(torch.compile(step, backend="aot_eager"))
    assert all(torch.equal(a, c) for a, c in zip(eager, got))
    with torch.no_grad():
        token = lambda state: ptb.lpv.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, scale=0.5)   # noqa: E731
        one, two = zi.clone(), zi.clone()
        a, c = token(one), torch.compile(token, backend="aot_eager")(two)
        assert torch.equal(a, c) and torch.equal(one, two) and not torch.equal(one, zi)


def test_vmap():
    q, k, v, g, zi, w, b = tensors()
    stack = lambda t: torch.stack([t, 2 * t, -t])   # noqa: E731
    o = torch.func.vmap(lambda x: ptb.lpv.linear_attention(q, k, x, g, scale=0.5))(stack(v))
    for got, one in zip(o, stack(v)):
        assert torch.equal(got, ptb.lpv.linear_attention(q, k, one, g, scale=0.5))
    x = v.flatten(-2)
    y = torch.func.vmap(lambda t: ptb.layer_norm(t, w, b, groups=3))(stack(x))
    for got, one in zip(y, stack(x)):
        assert torch.equal(got, ptb.layer_norm(one, w, b, groups=3))


def test_functional_gradients_are_refused():
    q, k, v, g, zi, w, b = tensors()
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ptb.lpv.linear_attention(t, k, v, g).float().sum())(q)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: ptb.layer_norm(t).float().sum())(v)
