"""Room that the gradient of the log decays takes (no device): the states at the chunks' ends in the call's own sizes, and two sums a
token for each group of threads that forms them."""
import pytest

from philtorch_b200 import _lib

F32, F64, F16, BF16 = 0, 1, 4, 5


def bytes_of(*key):
    return _lib.lib.ptb_linear_attention_workspace_bytes(*key)


@pytest.mark.parametrize("B,T,H,Dk,Dv", [(8, 32768, 32, 16, 16), (4, 16384, 16, 128, 128), (4, 16384, 16, 20, 65), (2, 5000, 40, 100, 7),
                                         (1, 129, 1, 1, 1)])
@pytest.mark.parametrize("dtype,scalar,chunk,columns,groups", [(BF16, 4, 128, 64, 2), (F32, 4, 32, 64, 1), (F16, 4, 32, 64, 1),
                                                               (F64, 8, 32, 32, 1)])
def test_room_for_the_decays_gradient(dtype, scalar, chunk, columns, groups, B, T, H, Dk, Dv):
    without, room = bytes_of(dtype, B, T, H, Dk, Dv, 1, 0, 0), bytes_of(dtype, B, T, H, Dk, Dv, 1, 1, 0)
    chunks = -(-T // chunk)
    state = Dk * (-(-Dv // 4) * 4 if dtype == BF16 else Dv)
    states = 2 * B * H * chunks * state * scalar
    sums = 2 * groups * -(-Dk // columns) * B * H * T * 2 * scalar
    assert room - without >= states + sums
    assert room - without <= states + sums + B * H * chunks * 8 + 6 * 256      # one sum per chunk; every array starts on 256 bytes


def test_small_heads_take_less_than_their_operands():
    B, T, H, D = 8, 32768, 32, 16
    operands = 4 * B * T * H * D * 2
    assert bytes_of(BF16, B, T, H, D, D, 1, 1, 0) < operands
    assert bytes_of(F32, B, T, H, D, D, 1, 1, 0) < 2 * operands
