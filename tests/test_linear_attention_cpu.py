"""Argument checks, shape contracts and the C entry points' refusals of linear attention and layer norm (no device)."""
import ctypes

import pytest
import torch

import philtorch_b200 as ptb
from philtorch_b200 import _lib

lib = _lib.lib
I3, I2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2


def meta(*s, dtype=torch.float32):
    return torch.empty(*s, device="meta", dtype=dtype)


def test_shapes_on_meta_tensors():
    ops = torch.ops.philtorch_b200
    q, v, g = meta(2, 9, 3, 16, dtype=torch.bfloat16), meta(2, 9, 3, 8, dtype=torch.bfloat16), meta(3)
    o, S = ops.linear_attention(q, q, v, g, None, None, 1.0, True)
    assert o.shape == (2, 9, 3, 8) and o.dtype == torch.bfloat16
    assert S.shape == (2, 3, 16, 8) and S.dtype == torch.float32
    grads = ops.linear_attention_bwd(q, q, v, g, None, None, 1.0, v, None, True, False, True, True, False)
    assert [tuple(t.shape) for t in grads] == [(2, 9, 3, 16), (0,), (2, 9, 3, 8), (3,), (0,)]
    assert ops.linear_attention_step(q[:, 0], q[:, 0], v[:, 0], g, meta(2, 3, 16, 8), 1.0).shape == (2, 3, 8)
    y, stats = ops.layer_norm(meta(2, 5, 24), None, None, 1e-5, 3)
    assert y.shape == (2, 5, 24) and stats.shape == (2, 10, 3)
    for bad in (lambda: ops.linear_attention(q, q, v, meta(4), None, None, 1.0, True),
                lambda: ops.linear_attention(q, q, v.float(), g, None, None, 1.0, True),
                lambda: ops.linear_attention(meta(2, 9, 3, 129), meta(2, 9, 3, 129), meta(2, 9, 3, 8), g, None, None, 1.0, True),
                lambda: ops.linear_attention(q, q, v, g.double(), None, None, 1.0, True),
                lambda: ops.linear_attention(q, q, v, g, meta(2, 3, 8, 16), None, 1.0, True),
                lambda: ops.linear_attention_step(q[:, 0], q[:, 0], v[:, 0], g, meta(1, 3, 16, 8).expand(2, 3, 16, 8), 1.0),
                lambda: ops.layer_norm(meta(2, 24), None, None, 1e-5, 5),
                lambda: ops.layer_norm(meta(2, 24), meta(23), None, 1e-5, 1)):
        with pytest.raises(RuntimeError):
            bad()


def test_cpu_tensors_are_refused():
    q = torch.randn(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ptb.lti.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        ptb.lpv.linear_attention(q, q, q, torch.zeros(1, 4, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        ptb.lti.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        ptb.layer_norm(q)


def test_c_entry_points_refuse():
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    s = I3(8, 8, 8)

    def fwd(dtype=0, B=1, T=4, H=1, Dk=8, Dv=8, q=p, ws=None, wsb=0, copies=0):
        return lib.ptb_linear_attention_fwd(dtype, B, T, H, Dk, Dv, q, s, p, s, p, s, p, s, None, 0, None, 1.0, copies, p, 0, None, ws, wsb,
                                            None, None)

    assert fwd(dtype=2) == 1 and fwd(dtype=9) == 1          # no complex numbers
    assert fwd(B=-1) == 1 and fwd(Dk=0) == 1 and fwd(Dk=129) == 1 and fwd(Dv=129) == 1
    assert fwd(q=None) == 1
    # a row long enough to be cut needs a workspace, and it has to be aligned
    assert fwd(T=1 << 20) == 2 and fwd(T=1 << 20, ws=256, wsb=64) == 2 and fwd(T=1 << 20, ws=257, wsb=1 << 30) == 2
    assert fwd(B=0) == 0 and fwd(H=0) == 0
    assert fwd(B=1 << 20, H=1 << 20) == 4 and fwd(dtype=5, T=0x7fffff01, ws=256, wsb=1 << 62) == 4
    assert lib.ptb_linear_attention_workspace_bytes(0, 1, 4, 1, 8, 8, 0, 0, 0) == 0
    assert lib.ptb_linear_attention_workspace_bytes(0, 1, 1 << 20, 1, 8, 8, 0, 0, 0) > 0
    assert lib.ptb_linear_attention_workspace_bytes(2, 1, 4, 1, 8, 8, 0, 0, 0) == 0
    # operands that have to be copied get their room
    some = lib.ptb_linear_attention_workspace_bytes(5, 2, 100, 3, 33, 65, 0, 0, 0)
    assert lib.ptb_linear_attention_workspace_bytes(5, 2, 100, 3, 33, 65, 0, 0, 7) >= some + 2 * 100 * 3 * (40 + 40 + 72) * 2
    assert lib.ptb_linear_attention_workspace_bytes(0, 2, 100, 3, 33, 65, 0, 0, 7) == lib.ptb_linear_attention_workspace_bytes(
        0, 2, 100, 3, 33, 65, 0, 0, 0)
    # the gradient of the decays keeps the states at the chunks' ends
    plain = lib.ptb_linear_attention_workspace_bytes(5, 1, 4096, 4, 128, 128, 1, 0, 0)
    assert lib.ptb_linear_attention_workspace_bytes(5, 1, 4096, 4, 128, 128, 1, 1, 0) >= plain + 2 * 32 * 4 * 128 * 128 * 4
    z = I2(8, 8)
    assert lib.ptb_linear_attention_step(0, 1, 1, 8, 200, p, z, p, z, p, z, p, z, 1.0, p, z, p, None) == 1
    assert lib.ptb_linear_attention_step(0, 1, 1, 8, 8, p, z, p, z, p, z, p, z, 1.0, None, z, p, None) == 1
    assert lib.ptb_layer_norm_fwd(0, 4, 1, 16385, p, 8, None, None, 0, 1e-5, 0, p, None, None, None) == 1
    assert lib.ptb_layer_norm_fwd(0, 4, 0, 8, p, 8, None, None, 0, 1e-5, 0, p, None, None, None) == 1
    assert lib.ptb_layer_norm_fwd(0, 4, 1, 8, None, 8, None, None, 0, 1e-5, 0, p, None, None, None) == 1
    assert lib.ptb_layer_norm_fwd(5, 4, 1, 8, p, 8, None, None, 0, 1e-5, 0, p, None, None, None) == 1   # only narrowing
    assert lib.ptb_layer_norm_fwd(0, 0, 1, 8, None, 8, None, None, 0, 1e-5, 0, None, None, None, None) == 0
    assert lib.ptb_layer_norm_bwd(0, 4, 1, 8, p, 8, None, 0, p, p, p, 8, p, p, p, None, 0, None, None) == 2
