"""quantize_int8 of rows near 2^31 elements: lengths that the kernels' 32-bit counts have no room for are refused."""
import ctypes

import pytest

from cmp_ext_amd import cabi


@pytest.mark.parametrize("cols", [2**31 - 1, 2**31 - 7, 2**31 - 512])
def test_rows_too_long_are_refused(cols):
    a = cabi.QuantizeInt8Args(dtype=cabi.BF16, cols=cols, rows=1, x=0x1000, x_row=cols, codes=0x2000, codes_row=cols, scale=0x3000)
    assert cabi.lib().cmpext3_quantize_int8(ctypes.byref(a), None) == cabi.ERR_TOO_LARGE
