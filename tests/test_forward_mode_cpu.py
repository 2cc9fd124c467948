"""Forward-mode derivatives: no tangent is lost without a word (no device: meta tensors go through the same calls)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import philtorch_b200 as ptb


def meta(*s):
    return torch.zeros(*s, device="meta")


def arguments(step):
    lead = (2, 3) if step else (2, 5, 3)
    return dict(q=meta(*lead, 8), k=meta(*lead, 8), v=meta(*lead, 4), log_decay=meta(*lead), zi=meta(2, 3, 8, 4),
                norm_weight=meta(12), norm_bias=meta(12))


def attention(a):
    return ptb.lpv.linear_attention(a["q"], a["k"], a["v"], a["log_decay"], a["zi"], norm_eps=1e-5, norm_weight=a["norm_weight"],
                                    norm_bias=a["norm_bias"])


def step(a):
    return ptb.lpv.linear_attention_step(a["q"], a["k"], a["v"], a["log_decay"], a["zi"], norm_eps=1e-5,
                                         norm_weight=a["norm_weight"], norm_bias=a["norm_bias"])


@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "zi", "norm_weight", "norm_bias"])
@pytest.mark.parametrize("call", [attention, step])
def test_dual_tensors_are_refused(call, name):
    a = arguments(call is step)
    assert call(a) is not None
    with fwAD.dual_level():
        assert call(a) is not None          # a level alone changes nothing
        a[name] = fwAD.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(a)


@pytest.mark.parametrize("name", ["x", "weight", "bias"])
def test_dual_tensors_are_refused_by_layer_norm(name):
    a = dict(x=meta(4, 12), weight=meta(12), bias=meta(12))
    with fwAD.dual_level():
        assert ptb.layer_norm(**a).shape == (4, 12)
        a[name] = fwAD.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ptb.layer_norm(**a)
        a[name].requires_grad_()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ptb.layer_norm(**a)


def test_functional_jvp_is_refused():
    a = arguments(False)
    one = torch.ones_like(a["q"])
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda q: attention({**a, "q": q}), (a["q"],), (one,))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: ptb.layer_norm(x), (meta(4, 12),), (meta(4, 12),))
    b = arguments(True)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda q: step({**b, "q": q}), (b["q"],), (meta(2, 3, 8),))
