"""gated_linear has a backward pass only: a derivative asked for in forward mode is refused, not taken as zero."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import cmpext3


def refused(x, w, dual):
    ops = [x, w, w.clone()]
    with fwAD.dual_level():
        ops[dual] = fwAD.make_dual(ops[dual], torch.ones_like(ops[dual]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            cmpext3.gated_linear(*ops)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            cmpext3.gated_linear(*ops)
        ops[0] = ops[0].clone().requires_grad_() if dual else ops[0]
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            cmpext3.gated_linear(*ops)


@pytest.mark.parametrize("dual", [0, 1, 2])
def test_refused_before_any_other_check_of_the_device(dual):
    refused(torch.zeros(3, 16, dtype=torch.float16), torch.zeros(5, 16, dtype=torch.float16), dual)


@pytest.mark.gpu
@pytest.mark.parametrize("dual", [0, 1, 2])
def test_refused(dual):
    x, w = torch.randn(3, 16, device="cuda").half(), torch.randn(5, 16, device="cuda").half()
    refused(x, w, dual)
    with fwAD.dual_level():  # without a tangent, or with forward mode switched off, as ever
        dual = fwAD.make_dual(x, torch.ones_like(x))
        assert torch.equal(cmpext3.gated_linear(fwAD.unpack_dual(dual).primal, w, w), cmpext3.gated_linear(x, w, w))
        with fwAD._set_fwd_grad_enabled(False):
            assert torch.equal(cmpext3.gated_linear(dual, w, w), cmpext3.gated_linear(x, w, w))
