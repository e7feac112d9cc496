"""In-place forms of the gated norm that are refused: other rows than the
operand's, one place for two results.  (Every call here is refused.)"""
import ctypes

import pytest

from diffuser_b200 import _lib

P, F, SHAPE, ARG = 0x1000, ctypes.c_float, 1, 7


@pytest.mark.parametrize("kw,status", [
    (dict(s=P, ld_s=72), SHAPE), (dict(s=2 * P, ld_s=72), SHAPE), (dict(s=2 * P, ld_y=72), SHAPE),
    (dict(s=P, ld_x=128), SHAPE), (dict(h=P, ld_h=72), SHAPE), (dict(h=2 * P, ld_y=72), SHAPE),
    (dict(s=5 * P), ARG), (dict(s=P, h=P), ARG)])
def test_results_in_the_place_of_operands(kw, status):
    a = dict(dict(x=P, ld_x=64, y=2 * P, ld_y=64, s=4 * P, ld_s=64, h=5 * P, ld_h=64), **kw)
    assert _lib.lib().dq_gated_norm(a["x"], a["ld_x"], a["y"], a["ld_y"], 4, 2, 64, None, 0, None, None, 0, None, None, 0,
                                    1, F(1.0), F(1e-6), 0, a["s"], a["ld_s"], a["h"], a["ld_h"], None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dx=P, ld_dx=72), SHAPE), (dict(dx=P, ld_ds=72), SHAPE), (dict(dy=2 * P, ld_dy=72), SHAPE),
    (dict(dy=3 * P, ld_dy=72), SHAPE), (dict(dx=4 * P, ld_dx=72), SHAPE), (dict(dx=6 * P), ARG)])
def test_gradients_in_the_place_of_operands(kw, status):
    a = dict(dict(ds=P, ld_ds=64, y=2 * P, ld_y=64, dx=5 * P, ld_dx=64, dy=6 * P, ld_dy=64), **kw)
    # (without a workspace: what is not refused before is refused for that)
    assert _lib.lib().dq_gated_norm_backward(a["ds"], a["ld_ds"], 3 * P, 64, 4 * P, 64, a["y"], a["ld_y"], 4, 2, 64, None,
                                             0, None, 0, None, None, 0, 1, F(1.0), F(1e-6), a["dx"], a["ld_dx"], a["dy"],
                                             a["ld_dy"], None, None, None, None, None, None, 0, None) == status
