"""Linear attention: sizes at which its kernels change over, the normalised read-out, and the ways a program runs it
(side by side, in inference mode, captured, on a long row)."""
import pytest
import torch

import philtorch_b200 as ptb
import linear_attention_common as la
from test_linear_attention_gpu import check_backward, check_forward, entry, inputs

pytestmark = pytest.mark.gpu

# head sizes of eight channels to 128, aligned and not; one token more than the short sequences, chunks of 128 and
# one more or less, two and more segments
SIZES = [(2, 33, 2, 64, 64), (2, 200, 2, 16, 8), (1, 700, 1, 8, 128), (1, 300, 3, 128, 8), (1, 450, 2, 72, 120), (2, 128, 1, 64, 72),
         (1, 257, 2, 65, 64), (1, 1500, 1, 128, 128), (1, 3200, 1, 64, 33)]


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sizes(dtype, size, form):
    q, k, v, g, zi, scale = inputs(size, dtype, form, seed=21)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = entry(form)(q, k, v, g, zi, scale=scale)
    det = [t.detach() for t in leaves]
    check_forward((o.detach(), S.detach()), *det, scale)
    gen = torch.Generator(device="cuda").manual_seed(22)
    go = torch.randn(o.shape, generator=gen, device="cuda").to(dtype)
    gS = torch.randn(S.shape, generator=gen, device="cuda").to(S.dtype)
    check_backward(form, torch.autograd.grad([o, S], leaves, [go, gS], retain_graph=True), *det, scale, None, go, gS)
    some = torch.autograd.grad([o, S], leaves[:3], [go, gS])     # without the decays' gradient: other kernels
    check_backward(form, list(some) + [None, None], *det, scale, None, go, gS)


def place(t, how):
    """The values of t (B,T,H,D) on rows that do not start on 16 bytes, or whose strides say so."""
    B, T, H, D = t.shape
    if how == "shifted":
        return t.new_empty(t.numel() + 1)[1:].view(t.shape).copy_(t)
    if how == "even":            # rows on 4 bytes
        return t.new_empty(B, T, H, D + 2)[..., 2:].copy_(t)
    if how == "heads first":     # memory order (H, B, T), an odd step from token to token
        return t.new_empty(H, B, T, D + 3)[..., :D].permute(1, 2, 0, 3).copy_(t)
    if how == "one token":
        return t[:, :1].expand(B, T, H, D)
    return t


@pytest.mark.parametrize("forms", [("shifted", "", "", ""), ("", "even", "heads first", ""), ("one token", "", "shifted", "even"),
                                   ("", "one token", "", "heads first"), ("even", "even", "even", "even"), ("", "", "", "one token")])
@pytest.mark.parametrize("size", [(2, 140, 3, 64, 64), (1, 33, 1, 128, 72), (2, 400, 2, 36, 100), (1, 1200, 2, 7, 65)])
def test_rows_off_the_boundaries(size, forms):
    q, k, v, g, zi, scale = inputs(size, torch.bfloat16, "lpv", seed=26)
    B, T, H, _ = q.shape
    lengths = torch.tensor([T - 9] * B, device="cuda")
    q, k, v = (place(t, how) for t, how in zip((q, k, v), forms))
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = ptb.lpv.linear_attention(*leaves, scale=scale, lengths=lengths)
    det = [t.detach() for t in leaves]
    check_forward((o.detach(), S.detach()), *det, scale, lengths)
    gen = torch.Generator(device="cuda").manual_seed(27)
    go = place(torch.randn(o.shape, generator=gen, device="cuda").to(o.dtype), forms[3])
    gS = torch.randn(S.shape, generator=gen, device="cuda").to(S.dtype)
    check_backward("lpv", torch.autograd.grad([o, S], leaves, [go, gS], retain_graph=True), *det, scale, lengths, go, gS)
    some = torch.autograd.grad([o, S], leaves[1:3], [go, gS])
    check_backward("lpv", [None] + list(some) + [None, None], *det, scale, lengths, go, gS)
    again = torch.autograd.grad(ptb.lpv.linear_attention(*leaves, scale=scale, lengths=lengths), leaves, [go, gS])
    plain = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in leaves]
    same = torch.autograd.grad(ptb.lpv.linear_attention(*plain, scale=scale, lengths=lengths), plain, [go.contiguous(), gS])
    assert all(torch.equal(a, b) for a, b in zip(again, same))     # where the rows lie changes no bit


def test_padded_batch_off_the_boundaries():
    """Sequences of no token, of one, up to a chunk's end and behind it, NaN behind their ends; captured and replayed."""
    q, k, v, g, zi, scale = inputs((5, 400, 2, 60, 33), torch.bfloat16, "lpv", seed=28)
    lengths = torch.tensor([0, 1, 128, 129, 400], device="cuda")
    clean = [t.clone() for t in (q, k, v, g)]
    for t in (q, k, v, g):
        for b, n in enumerate(lengths.tolist()):
            t[b, n:] = float("nan")
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    gen = torch.Generator(device="cuda").manual_seed(29)
    go = torch.randn(v.shape, generator=gen, device="cuda").to(v.dtype)
    gS = torch.randn(zi.shape, generator=gen, device="cuda")

    def step():
        o, S = ptb.lpv.linear_attention(*leaves, scale=scale, lengths=lengths)
        return (o.detach(), S.detach()) + torch.autograd.grad([o, S], leaves, [go, gS])

    first = step()
    check_forward(first[:2], *clean, zi.detach(), scale, lengths)
    check_backward("lpv", first[2:], *clean, zi.detach(), scale, lengths, go, gS)
    with torch.no_grad():
        y = ptb.lpv.linear_attention(*leaves[:4], scale=scale, lengths=lengths, norm_eps=1e-5)
        for b, n in enumerate(lengths.tolist()):
            assert (y[b, n:] == 0).all() and y[b, :n].isfinite().all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    del first
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        for t in out:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("params", [True, False])
@pytest.mark.parametrize("size", [(2, 20, 2, 32, 48), (2, 150, 3, 64, 128), (2, 90, 2, 33, 21), (1, 1500, 2, 128, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_normalised_read_out(dtype, size, params):
    """The norm reads the sums before they are rounded: first order, an error d of o moves a normalised value xh by at
    most r (d + mean d + |xh| mean(|xh| d)); the fifth on top is for what is of second order."""
    B, T, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs(size, dtype, "lpv", seed=23)
    gen = torch.Generator(device="cuda").manual_seed(24)
    w = (1 + torch.rand(H * Dv, generator=gen, device="cuda", dtype=torch.float64)).to(dtype) if params else None
    b = torch.randn(H * Dv, generator=gen, device="cuda", dtype=torch.float64).to(dtype) if params else None
    lengths = torch.tensor([T - 5] * B, device="cuda")
    o, S = ptb.lpv.linear_attention(q, k, v, g, zi, scale=scale, lengths=lengths, norm_eps=1e-3, norm_weight=w, norm_bias=b)
    assert o.dtype == dtype and o.shape == (B, T, H, Dv)
    ro, rS = la.forward(q, k, v, g, zi, scale, lengths)
    bo, bS = la.forward(*la.absolute(q, k, v), g, zi.abs(), scale, lengths)
    assert ((S.double() - rS).abs() <= la.tolerance(rS, bS, S.dtype, q, v)).all()
    u = torch.finfo(dtype).eps / 2
    d = la.tolerance(ro, bo, dtype, q, v) - u * ro.abs()
    c = ro - ro.mean(-1, keepdim=True)
    r = (c.square().mean(-1, keepdim=True) + 1e-3).rsqrt()
    xh = c * r
    wide = torch.ones(H, Dv, dtype=torch.float64, device="cuda") if w is None else w.double().view(H, Dv)
    ref = xh * wide + (0 if b is None else b.double().view(H, Dv))
    moved = r * (d + d.mean(-1, keepdim=True) + xh.abs() * (xh.abs() * d).mean(-1, keepdim=True))
    unit = torch.finfo(S.dtype).eps / 2
    tol = u * ref.abs() + 1.2 * wide * moved + (Dv + 16) * unit * (wide * (xh.abs() + r * ro.abs().mean(-1, keepdim=True)) + ref.abs())
    bad = (o.double() - ref).abs() > tol + torch.finfo(dtype).tiny
    assert not bad.any(), ((o.double() - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_normalised_read_out_with_gradients(dtype):
    """With gradients it is the two operators one after the other, bit for bit."""
    size = (2, 90, 2, 64, 32)
    q, k, v, g, zi, scale = inputs(size, dtype, "lti", seed=25)
    w = torch.ones(64, device="cuda", dtype=dtype)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi, w)]
    y, S = ptb.lti.linear_attention(q, k, v, g, zi, scale=scale, norm_eps=1e-5, norm_weight=w)
    o, S2 = ptb.lti.linear_attention(q, k, v, g, zi, scale=scale)
    z = ptb.layer_norm(o.flatten(-2), w, None, groups=2).unflatten(-1, (2, 32))
    assert torch.equal(y, z) and torch.equal(S, S2)
    gy = torch.randn_like(y)
    for a, c in zip(torch.autograd.grad(y, leaves, gy), torch.autograd.grad(z, leaves, gy)):
        assert torch.equal(a, c)
    fixed = [t.detach() for t in (q, k, v, g, zi)]      # only the norm's weight is learned: its gradient is there
    y, _ = ptb.lti.linear_attention(*fixed, scale=scale, norm_eps=1e-5, norm_weight=w)
    z = ptb.layer_norm(ptb.lti.linear_attention(*fixed, scale=scale)[0].flatten(-2), w, None, groups=2)
    assert torch.equal(torch.autograd.grad(y, w, gy)[0], torch.autograd.grad(z, w, gy.flatten(-2))[0])


def test_two_calls_at_once():
    """Two streams, both directions at the same time: the results of one call after the other."""
    sets = [inputs((1, 2000, 3, 128, 64), torch.bfloat16, "lpv", seed=s) for s in (26, 27)]
    for s in sets:
        for t in s[:5]:
            t.requires_grad_()
    gos = [torch.randn(1, 2000, 3, 64, device="cuda").bfloat16() for _ in sets]

    def both(s, go):
        o, S = ptb.lpv.linear_attention(*s[:5], scale=s[5])
        return [o, S, *torch.autograd.grad([o, S], s[:5], [go, torch.ones_like(S)])]

    one = [both(s, go) for s, go in zip(sets, gos)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    two = []
    for _ in range(3):
        for st, s, go in zip(streams, sets, gos):
            with torch.cuda.stream(st):
                two.append(both(s, go))
    torch.cuda.synchronize()
    for i, got in enumerate(two):
        assert all(torch.equal(a, b) for a, b in zip(got, one[i % 2]))
    ptb.check_errors()


def test_inference_mode_and_captured_step():
    """A server in inference mode: the prompt, then the step captured once and replayed on new tokens."""
    B, T, H, D = 3, 140, 2, 64
    with torch.inference_mode():
        q, k, v, g, _, scale = inputs((B, T + 4, H, D, D), torch.bfloat16, "lpv", seed=28, state=False)
        _, state = ptb.lpv.linear_attention(q[:, :T], k[:, :T], v[:, :T], g[:, :T], scale=scale, return_state=True)
        eager = state.clone()
        buf = [x[:, T].clone() for x in (q, k, v, g)]
        ptb.lpv.linear_attention_step(*buf, state.clone(), scale=scale)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = ptb.lpv.linear_attention_step(*buf, state, scale=scale)
        for t in range(T, T + 4):
            for dst, src in zip(buf, (q, k, v, g)):
                dst.copy_(src[:, t])
            graph.replay()
            want = ptb.lpv.linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], eager, scale=scale)
            assert torch.equal(o, want) and torch.equal(state, eager)


def test_a_row_whose_offsets_pass_32_bits():
    """2.3e9 outputs: the heads share q, k, v (stride zero), the end of the row equals a call that starts from the
    state before it."""
    T, H, D = 140_000, 128, 128
    gen = torch.Generator(device="cuda").manual_seed(29)
    q, k, v = (torch.randn(1, T, 1, D, generator=gen, device="cuda").bfloat16().expand(1, T, H, D) for _ in range(3))
    g = torch.full((H,), -0.02, device="cuda")
    o, S = ptb.lti.linear_attention(q, k, v, g, scale=0.1, return_state=True)
    assert o.numel() > 2 ** 31
    cut = 128 * 1090
    _, before = ptb.lti.linear_attention(q[:, :cut, :1], k[:, :cut, :1], v[:, :cut, :1], g[:1], scale=0.1, return_state=True)
    tail = [t[:, cut:, :1] for t in (q, k, v)]
    for h in (0, H - 1):
        check_forward((o[:, cut:, h:h + 1].contiguous(), S[:, h:h + 1]), *tail, g[:1], before, 0.1)
    assert torch.equal(o[:, :, 0], o[:, :, H - 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_are_not_written_and_nothing_else_is(dtype):
    """The output, its gradients and the states are whole tensors of their own: neighbours in memory keep their values."""
    q, k, v, g, zi, scale = inputs((1, 130, 2, 64, 64), dtype, "lti", seed=30)
    kept = [t.clone() for t in (q, k, v, g, zi)]
    lengths = torch.tensor([70], device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = ptb.lti.linear_attention(*leaves, scale=scale, lengths=lengths)
    torch.autograd.grad([o, S], leaves, [torch.ones_like(o), torch.ones_like(S)])
    assert all(torch.equal(a.detach(), b) for a, b in zip(leaves, kept))
    assert (o[:, 70:] == 0).all() and (lengths == 70).all()
