"""Layer norm over groups of channels, forward and backward, against its formula in float64."""
import pytest
import torch

import philtorch_b200 as ptb

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float64, torch.float16, torch.bfloat16]
# (rows, C, groups): one channel, widths around each kernel's lanes, odd widths, wide rows, many and few rows
SIZES = [(1, 1, 1), (3, 7, 1), (5, 32, 4), (300, 128, 1), (33, 2048, 16), (17, 96, 3), (9, 777, 1), (1000, 64, 1), (4, 1024, 1),
         (2, 1032, 1), (3, 4096, 1), (2, 5001, 1), (2, 16384, 1), (1, 16383, 1), (50, 12 * 80, 12), (7, 2000, 1)]


def reference(x, w, b, gy, eps, groups):
    x, gy = x.double(), gy.double()
    R, C = x.shape
    n = C // groups
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    xg = x.view(R, groups, n)
    c = xg - xg.mean(2, keepdim=True)
    r = (c.square().mean(2, keepdim=True) + eps).rsqrt()
    xh = c * r
    gu = (gy * w).view(R, groups, n)
    m0, m1 = gu.mean(2, keepdim=True), (gu * xh).mean(2, keepdim=True)
    gx = r * (gu - m0 - xh * m1)
    y, xh2 = xh.reshape(R, C) * w + b, xh.reshape(R, C)
    # sums of absolute terms; the mean is off by n roundings of mean |x|, which reaches xh times r, and the
    # variance by as much relative to it
    spread = (r * xg.abs().mean(2, keepdim=True)).expand_as(xg).reshape(R, C)
    by = w.abs() * (xh2.abs() + spread) * (1 + spread) + b.abs()
    bu = (gu.abs() + gu.abs().mean(2, keepdim=True) + xh.abs() * (gu * xh).abs().mean(2, keepdim=True))
    bgx = (r * bu).reshape(R, C) * (1 + spread) ** 2 + (r * gu.abs().mean(2, keepdim=True)).expand_as(xg).reshape(R, C) * (1 + spread) ** 2
    bw = (gy.abs() * (xh2.abs() + spread) * (1 + spread)).sum(0)
    return [y, gx.reshape(R, C), (gy * xh2).sum(0), gy.sum(0)], [by, bgx, bw, gy.abs().sum(0)]


def close(got, ref, bound, dtype, roundings):
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + roundings * torch.finfo(wide).eps / 2 * bound + torch.finfo(got.dtype).tiny
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (bad.sum().item(), (got.double() - ref).abs().max().item())


@pytest.mark.parametrize("params", ["type", "wide", "weight", "none"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_and_backward(dtype, size, params):
    R, C, groups = size
    gen = torch.Generator(device="cuda").manual_seed(R * C)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=torch.float64)   # noqa: E731
    x, gy = (2 * randn(R, C) + 1).to(dtype), randn(R, C).to(dtype)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    ptype = wide if params == "wide" else dtype
    w = None if params == "none" else (1 + 0.3 * randn(C)).to(ptype)
    b = None if params in ("none", "weight") else randn(C).to(ptype)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = ptb.layer_norm(x, w, b, eps=1e-5, groups=groups)
    grads = torch.autograd.grad(y, leaves, gy)
    ref, bound = reference(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), gy, 1e-5, groups)
    n = C // groups
    close(y.detach(), ref[0], bound[0], dtype, n + 8)
    close(grads[0], ref[1], bound[1], dtype, 3 * n + 16)
    if w is not None:
        assert grads[1].dtype == ptype
        close(grads[1], ref[2], bound[2], dtype, n + R + 16)
    if b is not None:
        close(grads[2], ref[3], bound[3], dtype, R + 16)
    plain = ptb.layer_norm(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), groups=groups)
    assert torch.equal(plain, y.detach())


def test_strides_and_shapes():
    gen = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(4, 6, 3 * 128 + 1, generator=gen, device="cuda").bfloat16()
    for x in (base[..., :128], base[..., 1:129], base[:, ::2, 128:256], base.transpose(0, 1)[..., :120], base[..., ::3][..., :64],
              base[0, 0, :64], base[:0, :, :64]):
        C = x.shape[-1]
        w = torch.randn(C, generator=gen, device="cuda").bfloat16()
        y = ptb.layer_norm(x, w, None, groups=2)
        assert y.shape == x.shape
        if x.numel():
            flat = x.reshape(-1, C)
            ref, bound = reference(flat, w, None, torch.zeros_like(flat), 1e-5, 2)
            close(y.reshape(-1, C), ref[0], bound[0], torch.bfloat16, C + 8)
    x = torch.randn(5, 64, device="cuda", requires_grad=True)
    (gx,) = torch.autograd.grad(ptb.layer_norm(x).sum(), x)     # a broadcast gradient: stride zero
    assert gx.abs().max() < 1e-4
    e = torch.randn(0, 64, device="cuda", requires_grad=True)
    w = torch.randn(64, device="cuda", requires_grad=True)
    ge, gw = torch.autograd.grad(ptb.layer_norm(e, w).sum(), (e, w))
    assert ge.shape == (0, 64) and (gw == 0).all()


def test_constant_rows_and_large_offsets():
    x = torch.full((3, 256), 7.0, device="cuda", requires_grad=True)
    b = torch.randn(256, device="cuda")
    y = ptb.layer_norm(x, None, b)
    assert torch.equal(y, b.expand(3, 256))
    (gx,) = torch.autograd.grad(y, x, torch.randn_like(y))
    assert torch.isfinite(gx).all()
    x = (1e4 + torch.randn(64, 512, device="cuda", dtype=torch.float64)).float()   # the mean far above the deviation
    ref, bound = reference(x, None, None, torch.zeros_like(x), 1e-5, 1)
    close(ptb.layer_norm(x), ref[0], bound[0], torch.float32, 512 + 8)
    bad = torch.randn(4, 64, device="cuda")
    bad[2, 5] = float("nan")
    y = ptb.layer_norm(bad)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()


def test_many_rows_repeat_bit_for_bit():
    x = torch.randn(20011, 192, device="cuda").bfloat16().requires_grad_()
    w, b = (torch.randn(192, device="cuda", requires_grad=True) for _ in range(2))
    gy = torch.randn(20011, 192, device="cuda").bfloat16()
    runs = [torch.autograd.grad(ptb.layer_norm(x, w, b, groups=3), (x, w, b), gy) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))
    ref, bound = reference(x.detach(), w.detach(), b.detach(), gy, 1e-5, 3)
    close(runs[0][1], ref[2], bound[2], torch.bfloat16, 64 + 20011)
    close(runs[0][2], ref[3], bound[3], torch.bfloat16, 20011)


def test_gradient_against_differences():
    x = torch.randn(5, 24, device="cuda", dtype=torch.float64, requires_grad=True)
    w, b = (torch.randn(24, device="cuda", dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda *a: ptb.layer_norm(*a, groups=3), (x, w, b), eps=1e-6, atol=1e-6)


def test_graph_replay():
    x = torch.randn(300, 256, device="cuda").bfloat16().requires_grad_()
    w, b = (torch.randn(256, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    gy = torch.randn(300, 256, device="cuda").bfloat16()
    step = lambda: torch.autograd.grad(ptb.layer_norm(x, w, b, groups=2), (x, w, b), gy)   # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn(300, 256, device="cuda"))
    graph.replay()
    eager = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, eager))


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    for kw, match in ((dict(groups=3), "multiple of groups"), (dict(groups=0), "multiple of groups"),
                      (dict(weight=torch.ones(63, device="cuda")), "weight must be"),
                      (dict(weight=torch.ones(64, device="cuda").half()), "weight must be"),
                      (dict(weight=torch.ones(64)), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            ptb.layer_norm(x, **kw)
    with pytest.raises(RuntimeError, match="16384"):
        ptb.layer_norm(torch.randn(1, 16385, device="cuda"))
    with pytest.raises(RuntimeError, match="same type"):
        ptb.layer_norm(x.half(), torch.ones(64, device="cuda").half(), torch.ones(64, device="cuda"))
    with pytest.raises(RuntimeError, match="takes float32"):
        ptb.layer_norm(torch.ones(4, 64, device="cuda", dtype=torch.int32))
