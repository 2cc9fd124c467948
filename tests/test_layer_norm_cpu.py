"""Refusals of the layer norm's C entry points that need no device."""
import ctypes

from philtorch_b200 import _lib


def test_statistics_come_together():
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)

    def fwd(mean, rstd):
        return _lib.lib.ptb_layer_norm_fwd(0, 4, 1, 8, p, 8, None, None, 0, 1e-5, 0, p, mean, rstd, None)

    assert fwd(p, None) == 1 and fwd(None, p) == 1
