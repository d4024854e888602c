"""The workspace of a gated block's backward pass, without a GPU: bf16 holds dgate and dup once, f16 for dx and for the weights."""
import ctypes

import pytest

from cmp_ext_amd import cabi


def need(dtype, m, n, k, dx=0x7000, dw_gate=0x8000, dw_up=0x9000):
    a = cabi.GatedBackwardArgs(dtype=dtype, activation=cabi.ACT_SILU, M=m, N=n, K=k, grad_out=0x1000, grad_row=n, gate=0x2000, up=0x3000,
                               pre_row=n, x=0x4000, x_row=k, w_gate=0x5000, gate_row=k, w_up=0x6000, up_row=k, dx=dx, dx_row=k,
                               dw_gate=dw_gate, dgate_row=k, dw_up=dw_up, dup_row=k)
    return cabi.lib().cmpext3_gated_backward_workspace_size(ctypes.byref(a))


@pytest.mark.parametrize("m,n,k", [(4096, 14336, 4096), (4096, 4096, 4096), (1, 8, 8)])
def test_held_gradients(m, n, k):
    each = 2 * m * n  # of dgate or dup
    units = 4 * (2 * m + 4 * n)
    assert need(cabi.BF16, m, n, k) >= 2 * each
    assert need(cabi.F16, m, n, k) >= 4 * each + units
    assert need(cabi.F16, m, n, k, dx=None) >= 2 * each + units
    assert need(cabi.F16, m, n, k, dw_gate=None) >= 3 * each + units
    if m > 1:  # and no more than a tenth above it: no splits, no copies
        assert need(cabi.BF16, m, n, k) < 2.2 * each and need(cabi.F16, m, n, k) < 4.4 * each
        assert need(cabi.F16, m, n, k, dw_gate=None, dw_up=None) < 2.4 * each


def test_no_rows():
    assert need(cabi.F16, 0, 64, 64) == 0 and need(cabi.BF16, 0, 64, 64) == 0
