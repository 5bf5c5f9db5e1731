"""Refusals of the 4-bit cache entries at the ends of their arguments (no GPU)."""
import ctypes as C

import pytest

import q3t
from test_kv4 import batch, cache, call_append, rows


@pytest.mark.parametrize("scale, status", [(2.0 ** 127, q3t.OK), (-(2.0 ** 127), q3t.OK), (0.0, q3t.OK),
                                           (1.1 * 2.0 ** 127, q3t.INVALID_INPUT), (-3.4e38, q3t.INVALID_INPUT),
                                           (float("inf"), q3t.INVALID_INPUT), (float("nan"), q3t.INVALID_INPUT)])
def test_scales_that_32_bits_do_not_hold_in_powers_of_two_are_refused(scale, status):
    """The scores' scale is taken times log2(e)."""
    assert q3t.lib().q3t_kv4_attend(C.byref(cache()), C.byref(batch(num_tokens=0)), 16, 1 << 20, 2048, scale, 0, 1 << 20,
                                    2048, 1 << 21, 1 << 22, None) == status


ODD = (1 << 20) + 2  # a 32-bit element there would be read across its boundary


def attend_and_read(c, b):
    L = q3t.lib()
    return (L.q3t_kv4_attend(C.byref(c), C.byref(b), 16, 1 << 20, 2048, 0.1, 0, 1 << 22, 2048, 1 << 21, 1 << 22, None),
            L.q3t_kv4_read(C.byref(c), C.byref(b), 1 << 20, 1024, 1 << 20, 1024, None))


@pytest.mark.parametrize("bad", [dict(page_table=ODD), dict(q_start=ODD), dict(kv_len=ODD), dict(table_row=ODD + 1)])
def test_index_arrays_off_their_boundary_are_refused(bad):
    """Before any launch: the kernels would fault."""
    c, b = (cache(**bad), batch()) if "page_table" in bad else (cache(), batch(**bad))
    assert call_append(c, b, rows()) == q3t.INVALID_INPUT
    assert attend_and_read(c, b) == (q3t.INVALID_INPUT, q3t.INVALID_INPUT)


@pytest.mark.parametrize("bad", [dict(q_gamma=ODD), dict(k_gamma=ODD)])
def test_norm_weights_off_their_boundary_are_refused(bad):
    assert call_append(cache(), batch(), rows(**bad)) == q3t.INVALID_INPUT
