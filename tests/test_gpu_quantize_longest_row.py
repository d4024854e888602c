"""quantize_int8 of the longest row it takes, 2^31 - 513 elements: counts of 32 bits at their end."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_longest_row():
    import cmpext3

    n = 2**31 - 513
    x = torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_()
    x[n - 3] = 100.0  # the largest, behind everything else
    q, s = cmpext3.quantize_int8(x)
    assert abs(s.item() - 100 / 127) <= 100 / 127 * 2.0**-24
    for part in (slice(0, 5000), slice(n // 2, n // 2 + 5000), slice(n - 5000, n)):
        assert torch.equal(q[part].double(), torch.round(127 * x[part].double() / 100))
    with pytest.raises(RuntimeError, match="quantize_int8"):
        cmpext3.quantize_int8(torch.empty(n + 1, device="cuda", dtype=torch.bfloat16))
