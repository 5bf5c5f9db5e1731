"""Refusals of the 4-bit cache entries at the ends of their arguments (no GPU)."""
import ctypes as C

import pytest

import q3t
from test_kv4 import batch, cache


@pytest.mark.parametrize("scale, status", [(2.0 ** 127, q3t.OK), (-(2.0 ** 127), q3t.OK), (0.0, q3t.OK),
                                           (1.1 * 2.0 ** 127, q3t.INVALID_INPUT), (-3.4e38, q3t.INVALID_INPUT),
                                           (float("inf"), q3t.INVALID_INPUT), (float("nan"), q3t.INVALID_INPUT)])
def test_scales_that_32_bits_do_not_hold_in_powers_of_two_are_refused(scale, status):
    """The scores' scale is taken times log2(e)."""
    assert q3t.lib().q3t_kv4_attend(C.byref(cache()), C.byref(batch(num_tokens=0)), 16, 1 << 20, 2048, scale, 0, 1 << 20,
                                    2048, 1 << 21, 1 << 22, None) == status
