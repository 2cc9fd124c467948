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


def test_where_the_kernels_change_over_is_said_once():
    """Operands on any rows are copied from one length on: the library's own, for the checks of the arguments and for the room."""
    import torch
    from philtorch_b200 import attention

    last = _lib.lib.ptb_linear_attention_any_rows_tokens(BF16)
    assert all(_lib.lib.ptb_linear_attention_any_rows_tokens(d) == 2 ** 63 - 1 for d in (F32, F64, F16))
    for T in (last - 1, last, last + 1):
        copied = bytes_of(BF16, 2, T, 3, 33, 65, 0, 0, 7) > bytes_of(BF16, 2, T, 3, 33, 65, 0, 0, 0)
        assert copied == (T > last)
        odd = torch.empty(2, T, 3, 33, dtype=torch.bfloat16)
        assert attention._copies(T, odd, odd, odd) == (7 if T > last else 0)
        assert attention._copies(T, *[t.float() for t in (odd, odd, odd)]) == 0
