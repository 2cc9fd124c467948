"""Layer norm over many rows: sums over the rows that a single lost, doubled or misplaced row would change."""
import pytest
import torch

import philtorch_b200 as ptb
from test_layer_norm_gpu import close, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,C,groups", [(20011, 192, 3), (5003, 2048, 16), (4099, 777, 1), (1201, 4096, 1), (301, 16384, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parameter_gradients_count_every_row(dtype, rows, C, groups):
    """x = +-1 in equal numbers per group (one odd channel: 0) and whole numbers for gy: the bias's gradient is an exact whole
    number, the weight's a whole number times r."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    n = C // groups
    sign = torch.ones(n, device="cuda")
    sign[n // 2:] = -1
    if n % 2:
        sign[-1] = 0
    order = torch.rand(rows, groups, n, generator=gen, device="cuda").argsort(-1)
    x = sign[order].reshape(rows, C).to(dtype).requires_grad_()
    gy = torch.randint(-2, 3, (rows, C), generator=gen, device="cuda").to(dtype)
    w, b = (torch.randn(C, generator=gen, device="cuda").requires_grad_() for _ in range(2))
    _, gw, gb = torch.autograd.grad(ptb.layer_norm(x, w, b, eps=0.25, groups=groups), (x, w, b), gy)
    assert torch.equal(gb.double(), gy.double().sum(0))
    r = ((n - n % 2) / n + 0.25) ** -0.5
    whole = (gy.double() * x.detach().double()).sum(0)
    # the mean is zero exactly and r the same few roundings off in every row; a term meets the additions of its lane (a CTA's share
    # of the rows over its lanes, at most 14), of the lanes (32), of the partial rows (at most 296 in 8 parts): below 100 roundings
    tol = 100 * 2.0 ** -24 * r * gy.double().abs().sum(0)
    assert tol.max() < 0.5 * r      # a row that is lost or counted twice changes r |gy| >= r
    bad = (gw.double() - r * whole).abs() > tol
    assert not bad.any(), (gw.double() - r * whole).abs().max().item()


def test_gradient_of_many_rows():
    gen = torch.Generator(device="cuda").manual_seed(71)
    x = torch.randn(20011, 192, generator=gen, device="cuda").bfloat16().requires_grad_()
    w, b = (torch.randn(192, generator=gen, device="cuda") for _ in range(2))
    gy = torch.randn(20011, 192, generator=gen, device="cuda").bfloat16()
    (gx,) = torch.autograd.grad(ptb.layer_norm(x, w, b, groups=3), x, gy)
    ref, bound = reference(x.detach(), w, b, gy, 1e-5, 3)
    close(gx, ref[1], bound[1], torch.bfloat16, 3 * 64 + 16)
