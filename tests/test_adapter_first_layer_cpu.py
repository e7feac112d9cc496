"""Which gradients dq_adapter_backward may be asked for."""
from diffuser_b200 import _lib

P = 0x1000


def test_the_gradients_come_in_pairs():
    def call(dx, dx_out, ddown, dup, lddx=64, M=4):
        return _lib.lib().dq_adapter_backward(P, 64, P, 64, None, P, M, 1, 64, 64, P, P, P, 16, 2, P, dx, lddx, dx_out,
                                              lddx, ddown, dup, P + 8, 1 << 30, None)
    ARG, SHAPE = 7, 1
    assert call(P, None, P, P) == ARG and call(None, P, P, P) == ARG and call(P, P, P, None) == ARG
    assert call(None, None, None, None) == ARG
    assert call(P, P, P, P, lddx=60) == SHAPE
    # the strides of operands that are not there are not looked at: on to the
    # alignment of one that is
    assert call(None, None, P + 2, P, lddx=0) == 2
    assert call(None, None, None, None, M=0) == 0
