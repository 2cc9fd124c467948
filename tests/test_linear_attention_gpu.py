"""Linear attention with decays (lti: per head, lpv: per token and head) and its single-token form against the
recurrence in float64; sizes and masks where tiles, chunks and segments end."""
import pytest
import torch

import philtorch_b200 as ptb
import linear_attention_common as la

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
# (B, T, H, Dk, Dv): single tokens, chunks of 32 / 64 / 128 and one more or less, odd and unaligned head sizes, rows
# long enough to be cut into segments
SIZES = [(1, 1, 1, 1, 1), (2, 3, 2, 5, 7), (2, 31, 3, 16, 16), (1, 32, 2, 64, 64), (2, 33, 2, 33, 65), (3, 64, 1, 128, 128),
         (1, 65, 2, 80, 48), (2, 127, 1, 96, 128), (1, 129, 3, 72, 100), (2, 300, 2, 128, 64), (1, 1100, 1, 64, 128),
         (1, 2500, 2, 40, 24)]


def inputs(size, dtype, form, seed=0, state=True):
    B, T, H, Dk, Dv = size
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=torch.float64)   # noqa: E731
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    q, k, v = randn(B, T, H, Dk).to(dtype), randn(B, T, H, Dk).to(dtype), randn(B, T, H, Dv).to(dtype)
    if form == "lti":
        g = torch.log1p(-torch.exp2(-(1.0 + 7 * torch.rand(H, generator=gen, device="cuda", dtype=torch.float64))))
    else:
        g = torch.nn.functional.logsigmoid(3 * randn(B, T, H) + 2)
    zi = randn(B, H, Dk, Dv).to(wide) if state else None
    return q, k, v, g.to(wide), zi, Dk ** -0.5


def entry(form):
    return (ptb.lti if form == "lti" else ptb.lpv).linear_attention


def check_forward(out, q, k, v, g, zi, scale, lengths=None):
    o, S = out
    ro, rS = la.forward(q, k, v, g, zi, scale, lengths)
    bo, bS = la.forward(*la.absolute(q, k, v), g, *la.absolute(zi), abs(scale), lengths)
    assert o.dtype == q.dtype and o.is_contiguous()
    assert ((o.double() - ro).abs() <= la.tolerance(ro, bo, q.dtype, q, v)).all()
    assert ((S.double() - rS).abs() <= la.tolerance(rS, bS, S.dtype, q, v)).all()


def check_backward(form, grads, q, k, v, g, zi, scale, lengths, go, gzf):
    ref = la.backward(q, k, v, g, zi, scale, lengths, go, gzf)
    aq, ak, av, azi, ago, agzf = la.absolute(q, k, v, zi, go, gzf)
    bound = list(la.backward(aq, ak, av, g, azi, abs(scale), lengths, ago, agzf))
    bound[3] = la.decay_bound(q, k, v, g, zi, scale, lengths, go, gzf)
    ref = list(ref)
    if form == "lti":
        ref[3], bound[3] = ref[3].sum((0, 1)), bound[3].sum((0, 1))
    names = ["q", "k", "v", "log_decay", "zi"]
    for name, got, r, b in zip(names, grads, ref, bound):
        if got is None:
            continue
        bad = (got.double() - r).abs() > la.tolerance(r, b, got.dtype, q, v)
        assert not bad.any(), (name, bad.sum().item(), (got.double() - r).abs().max().item())


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward(dtype, size, form):
    q, k, v, g, zi, scale = inputs(size, dtype, form)
    check_forward(entry(form)(q, k, v, g, zi, scale=scale), q, k, v, g, zi, scale)
    o, S = entry(form)(q, k, v, g, scale=scale, return_state=True)
    check_forward((o, S), q, k, v, g, None, scale)
    only = entry(form)(q, k, v, g, scale=scale)      # without the state: one tensor, the same values to rounding
    check_forward((only, S), q, k, v, g, None, scale)


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward(dtype, size, form):
    q, k, v, g, zi, scale = inputs(size, dtype, form, seed=1)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = entry(form)(q, k, v, g, zi, scale=scale)
    gen = torch.Generator(device="cuda").manual_seed(2)
    go = torch.randn(o.shape, generator=gen, device="cuda").to(dtype)
    gS = torch.randn(S.shape, generator=gen, device="cuda").to(S.dtype)
    grads = torch.autograd.grad([o, S], leaves, [go, gS])
    det = [t.detach() for t in (q, k, v, g, zi)]
    check_backward(form, grads, *det, scale, None, go, gS)


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (4,), (0, 1, 2), (0, 3), (2, 4)])
def test_backward_of_some_inputs(wanted):
    """Only the gradients asked for, from o alone, from the state alone and from both."""
    q, k, v, g, zi, scale = inputs((2, 150, 2, 64, 64), torch.bfloat16, "lpv", seed=3)
    args = [q, k, v, g, zi]
    for i in wanted:
        args[i].requires_grad_()
    o, S = ptb.lpv.linear_attention(*args, scale=scale)
    go, gS = torch.randn_like(o), torch.randn_like(S)
    det = [t.detach() for t in args]
    for use_o, use_S in ((True, True), (True, False), (False, True)):
        outs, gos = [o] * use_o + [S] * use_S, [go] * use_o + [gS] * use_S
        got = torch.autograd.grad(outs, [args[i] for i in wanted], gos, retain_graph=True, allow_unused=True)
        full = [None] * 5
        for i, t in zip(wanted, got):
            full[i] = t
        check_backward("lpv", full, *det, scale, None, go if use_o else torch.zeros_like(go), gS if use_S else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padded_batch(dtype):
    """Lengths of zero, one, a chunk and the whole; what lies behind a sequence's end is NaN and never read."""
    size = (6, 200, 2, 64, 80)
    q, k, v, g, zi, scale = inputs(size, dtype, "lpv", seed=4)
    lengths = torch.tensor([200, 0, 1, 64, 65, 199], device="cuda")
    for t in (q, k, v, g):
        for b, n in enumerate(lengths.tolist()):
            t[b, n:] = float("nan")
    clean = torch.where(torch.isnan(g), torch.zeros_like(g), g)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    for kind in (torch.int64, torch.int32):
        o, S = ptb.lpv.linear_attention(q, k, v, g, zi, scale=scale, lengths=lengths.to(kind))
        with torch.no_grad():
            check_forward((o, S), q.nan_to_num(), k.nan_to_num(), v.nan_to_num(), clean, zi, scale, lengths)
            assert torch.equal(S[1], zi[1])
            assert (o[1] == 0).all() and (o[2, 1:] == 0).all()
        go, gS = torch.randn_like(o), torch.randn_like(S)
        for b, n in enumerate(lengths.tolist()):
            go[b, n:] = float("nan")
        grads = torch.autograd.grad([o, S], leaves, [go, gS])
        assert all(torch.isfinite(t).all() for t in grads)
        det = [t.detach().nan_to_num() for t in (q, k, v)] + [clean.detach(), zi.detach()]
        check_backward("lpv", grads, *det, scale, lengths, go.nan_to_num(), gS)


def test_lengths_out_of_range_are_clamped():
    q, k, v, g, zi, scale = inputs((2, 50, 1, 16, 16), torch.float32, "lti")
    o, S = ptb.lti.linear_attention(q, k, v, g, zi, scale=scale, lengths=torch.tensor([-3, 2 ** 40], device="cuda"))
    assert (o[0] == 0).all() and torch.equal(S[0], zi[0])
    whole, T = ptb.lti.linear_attention(q, k, v, g, zi, scale=scale)
    assert torch.equal(o[1], whole[1]) and torch.equal(S[1], T[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_of_zero_starts_anew(dtype):
    """-inf at a token: nothing before it reaches what comes after, forward or backward, inside a chunk and across."""
    q, k, v, g, zi, scale = inputs((1, 300, 2, 64, 64), dtype, "lpv", seed=5)
    for t in (0, 40, 41, 64, 128, 250):
        g[:, t] = -float("inf")
    o, S = ptb.lpv.linear_attention(q, k, v, g, zi, scale=scale)
    check_forward((o, S), q, k, v, g, zi, scale)
    o2, S2 = ptb.lpv.linear_attention(q[:, 250:], k[:, 250:], v[:, 250:], g[:, 250:], zi, scale=scale)
    check_forward((o[:, 250:].contiguous(), S), q[:, 250:], k[:, 250:], v[:, 250:], g[:, 250:], None, scale)
    assert torch.isfinite(o2).all() and torch.isfinite(S2).all()
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = ptb.lpv.linear_attention(*leaves, scale=scale)
    go, gS = torch.randn_like(o), torch.randn_like(S)
    grads = torch.autograd.grad([o, S], leaves, [go, gS])
    check_backward("lpv", grads, *(t.detach() for t in leaves), scale, None, go, gS)
    assert (grads[4] == 0).all()


def test_no_decay_and_strong_decay():
    for value in (0.0, -30.0, -1e4):
        q, k, v, g, zi, scale = inputs((1, 260, 2, 32, 32), torch.bfloat16, "lti", seed=6)
        g = torch.full_like(g, value)
        check_forward(ptb.lti.linear_attention(q, k, v, g, zi, scale=scale), q, k, v, g, zi, scale)


def test_strides_of_a_fused_projection_and_shared_heads():
    """Views of one (B,T,H,3D) tensor, an unaligned view, heads shared by expand (their gradient is the sum)."""
    B, T, H, D = 2, 90, 4, 64
    gen = torch.Generator(device="cuda").manual_seed(7)
    fused = torch.randn(B, T, H, 3 * D + 1, generator=gen, device="cuda").bfloat16()
    g = -0.1 * torch.rand(B, H, T, generator=gen, device="cuda").transpose(1, 2)
    for at in (0, 1):
        q, k, v = (fused[..., at + i * D:at + (i + 1) * D] for i in range(3))
        check_forward(ptb.lpv.linear_attention(q, k, v, g, return_state=True, scale=0.2), q, k, v, g, None, 0.2)
    t_first = fused[..., :D].permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)   # memory order (T, B, H, D)
    check_forward(ptb.lpv.linear_attention(t_first, k, v, g, return_state=True), t_first, k, v, g, None, 1.0)
    one_k = fused[:, :, :1, :D].clone().requires_grad_()
    shared = one_k.expand(B, T, H, D)
    o = ptb.lpv.linear_attention(q, shared, v, g, scale=0.2)
    go = torch.randn_like(o)
    got = torch.autograd.grad(o, one_k, go)[0]
    dense = one_k.detach().expand(B, T, H, D).contiguous()
    _, rk, _, _, _ = la.backward(q, dense, v, g, None, 0.2, None, go, None)
    _, bk, _, _, _ = la.backward(*la.absolute(q, dense, v), g, None, 0.2, None, go.abs(), None)
    tol = la.tolerance(rk, bk, torch.bfloat16, q, v).sum(2) + torch.finfo(torch.bfloat16).eps / 2 * H * rk.abs().sum(2)
    assert ((got[:, :, 0].double() - rk.sum(2)).abs() <= tol).all()


def test_gradient_against_differences():
    for form in ("lti", "lpv"):
        q, k, v, g, zi, scale = inputs((2, 37, 2, 3, 4), torch.float64, form, seed=8)
        lengths = torch.tensor([37, 20], device="cuda")
        leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
        fn = lambda *a: entry(form)(*a, scale=0.7, lengths=lengths)   # noqa: E731
        assert torch.autograd.gradcheck(fn, leaves, eps=1e-6, atol=1e-6, nondet_tol=0.0)
        with pytest.raises(RuntimeError):      # first derivatives only
            (gq,) = torch.autograd.grad(fn(*leaves)[0].sum(), leaves[0], create_graph=True)
            gq.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_repeat_bit_for_bit(dtype):
    q, k, v, g, zi, scale = inputs((1, 2500, 2, 64, 64), dtype, "lpv", seed=9)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    runs = []
    for _ in range(3):
        o, S = ptb.lpv.linear_attention(*leaves, scale=scale)
        runs.append([o, S, *torch.autograd.grad([o, S], leaves, [torch.ones_like(o), torch.ones_like(S)])])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_empty_sizes():
    q, k, v, g, zi, scale = inputs((2, 0, 3, 16, 8), torch.float32, "lpv")
    o, S = ptb.lpv.linear_attention(q, k, v, g, zi)
    assert o.shape == (2, 0, 3, 8) and torch.equal(S, zi)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    o, S = ptb.lpv.linear_attention(*leaves)
    gs = torch.autograd.grad(S, leaves, torch.ones_like(S), allow_unused=True)
    assert (gs[4] == 1).all()
    q, k, v, g, zi, scale = inputs((0, 5, 3, 16, 8), torch.float32, "lti")
    o, S = ptb.lti.linear_attention(q, k, v, g, zi)
    assert o.shape == (0, 5, 3, 8) and S.shape == (0, 3, 16, 8)


STEP_SIZES = [(1, 1, 1, 1), (1, 16, 128, 128), (7, 5, 33, 65), (3, 2, 128, 40), (64, 3, 64, 64), (2, 3, 17, 2)]


@pytest.mark.parametrize("form", ["lti", "lpv"])
@pytest.mark.parametrize("size", STEP_SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_step(dtype, size, form):
    B, H, Dk, Dv = size
    q, k, v, g, zi, scale = inputs((B, 4, H, Dk, Dv), dtype, form, seed=10)
    state = zi.clone()
    side = ptb.lti if form == "lti" else ptb.lpv
    outs = [side.linear_attention_step(q[:, t], k[:, t], v[:, t], g if form == "lti" else g[:, t], state, scale=scale)
            for t in range(4)]
    assert outs[0].shape == (B, H, Dv) and outs[0].dtype == dtype
    check_forward((torch.stack(outs, 1), state), q, k, v, g, zi, scale)


def test_step_in_a_cache_and_with_a_reset():
    """States that are views of a larger cache: their neighbours stay as they were."""
    B, H, D = 3, 4, 64
    cache = torch.randn(B + 2, H + 1, D, D, device="cuda")
    before = cache.clone()
    state = cache[1:1 + B, :H]
    q, k, v = (torch.randn(B, H, D, device="cuda") for _ in range(3))
    g = -torch.rand(B, H, device="cuda")
    g[1] = -float("inf")
    state_before = state.clone()
    version = cache._version
    o = ptb.lpv.linear_attention_step(q, k, v, g, state, scale=0.5)
    assert cache._version > version
    args = [t.unsqueeze(1) for t in (q, k, v, g)]
    check_forward((o.unsqueeze(1), state), *args, state_before, 0.5)
    outside = torch.ones(B + 2, H + 1, dtype=torch.bool, device="cuda")
    outside[1:1 + B, :H] = False
    assert torch.equal(cache[outside], before[outside])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    """As a server runs them: a padded batch of prompts, then token by token from its states, read-out normalised;
    equal to the whole sequences at once."""
    B, T, H, D, more = 3, 70, 2, 64, 5
    q, k, v, g, _, scale = inputs((B, T + more, H, D, D), dtype, "lpv", seed=11, state=False)
    w, b = torch.randn(H * D, device="cuda").to(dtype), torch.randn(H * D, device="cuda").to(dtype)
    lengths = torch.tensor([T, 13, 64], device="cuda")
    norm = dict(norm_eps=1e-5, norm_weight=w, norm_bias=b)
    _, state = ptb.lpv.linear_attention(q[:, :T], k[:, :T], v[:, :T], g[:, :T], scale=scale, lengths=lengths,
                                        return_state=True, **norm)
    for t in range(T, T + more):
        o = ptb.lpv.linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], state, scale=scale, **norm)
    for i, n in enumerate(lengths.tolist()):
        sel = torch.cat([torch.arange(n), torch.arange(T, T + more)]).cuda()
        whole, S = ptb.lpv.linear_attention(q[i:i + 1, sel], k[i:i + 1, sel], v[i:i + 1, sel], g[i:i + 1, sel],
                                            scale=scale, return_state=True, **norm)
        ro, rS = la.forward(q[i:i + 1, sel], k[i:i + 1, sel], v[i:i + 1, sel], g[i:i + 1, sel], None, scale, None)
        _, bS = la.forward(*la.absolute(q[i:i + 1, sel], k[i:i + 1, sel], v[i:i + 1, sel]), g[i:i + 1, sel], None, scale, None)
        tol = la.tolerance(rS, bS, S.dtype, q, v)
        assert ((S - rS).abs() <= tol).all() and ((state[i:i + 1] - rS).abs() <= tol).all()
        ref = torch.nn.functional.layer_norm(ro[0, -1], (D,), eps=1e-5) * w.view(H, D).double() + b.view(H, D).double()
        assert (whole[0, -1] - ref).abs().max() <= 0.05 * ref.abs().max()
        assert (o[i] - ref).abs().max() <= 0.05 * ref.abs().max()


def test_other_stream_and_graph():
    """On a stream of its own; captured with its backward pass and replayed on new inputs, twice side by side."""
    q, k, v, g, zi, scale = inputs((1, 1100, 2, 64, 64), torch.bfloat16, "lpv", seed=12)
    leaves = [t.requires_grad_() for t in (q, k, v, g, zi)]
    gen = torch.Generator(device="cuda").manual_seed(13)
    go = torch.randn(1, 1100, 2, 64, generator=gen, device="cuda").bfloat16()

    def step():
        o, S = ptb.lpv.linear_attention(*leaves, scale=scale)
        return [o, S, *torch.autograd.grad([o, S], leaves, [go, torch.ones_like(S)])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            on_stream = step()
    torch.cuda.current_stream().wait_stream(s)
    eager = step()
    assert all(torch.equal(a, b) for a, b in zip(on_stream, eager))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    new = inputs((1, 1100, 2, 64, 64), torch.bfloat16, "lpv", seed=14)
    with torch.no_grad():
        for t, n in zip(leaves, new):
            t.copy_(n)
    for gr in graphs:
        gr.replay()
    eager = step()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals():
    q, k, v, g, zi, _ = inputs((2, 9, 3, 16, 8), torch.float32, "lpv")
    bad = [
        (dict(k=k[..., :8]), "shape of q"), (dict(v=v[:, :5]), "v must be"), (dict(q=q.half()), "same type"),
        (dict(log_decay=g.double()), "log_decay must be"), (dict(log_decay=g[:, :4]), "log_decay must be"),
        (dict(zi=zi[:, :1]), "initial state"), (dict(zi=zi.half()), "initial state"),
        (dict(lengths=torch.zeros(3, dtype=torch.int64, device="cuda")), "lengths"),
        (dict(lengths=torch.zeros(2, device="cuda")), "lengths"), (dict(q=q.cpu()), "CUDA"),
        (dict(q=torch.zeros(2, 9, 3, 129, device="cuda"), k=torch.zeros(2, 9, 3, 129, device="cuda"), zi=None), "head sizes"),
    ]
    for change, match in bad:
        args = dict(q=q, k=k, v=v, log_decay=g, zi=zi)
        args.update(change)
        with pytest.raises(RuntimeError, match=match):
            ptb.lpv.linear_attention(**args)
    with pytest.raises(ValueError, match="log_decay"):
        ptb.lti.linear_attention(q, k, v, g)
    with pytest.raises(ValueError, match="norm_eps"):
        ptb.lpv.linear_attention(q, k, v, g, norm_weight=torch.ones(24, device="cuda"))
    step = [t[:, 0] for t in (q, k, v, g)]
    with pytest.raises(RuntimeError, match="in place"):
        ptb.lpv.linear_attention_step(*step, zi[:, :, :1].expand(2, 3, 16, 8))
    with pytest.raises(RuntimeError, match="in place"):
        ptb.lpv.linear_attention_step(*step, zi[:1].expand(2, 3, 16, 8))
    with pytest.raises(RuntimeError, match="in place"):
        ptb.lpv.linear_attention_step(*step, zi.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError, match="differentiable"):
        ptb.lpv.linear_attention_step(*step, zi.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="state must be"):
        ptb.lpv.linear_attention_step(*step, zi.double())
