"""8-bit projections whose scales are large or small: a sum times one scale may lie outside fp32 where the result does not."""
import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
KERNELS = ["", "any64x64", "rows", "small64x64,splits=1,groups=1", "small64x64,splits=2,groups=2", "tile128x128,splits=1", "tile128x128,splits=3",
           "tile256x128", "tile256x256"]
SIZES = [(1, 40, 2048), (20, 130, 2048), (60, 65, 2064), (130, 300, 2100), (300, 513, 2048)]


def codes(*shape, seed=0, low=64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(low, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def scales(n, size, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return ((torch.rand(n, generator=g, device=DEV, dtype=torch.float64) + 0.5) * size).float()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("large,small", [(1e34, 1e-36), (1e36, 1e-34)])
def test_a_large_scale_and_a_small_one(monkeypatch, kernel, m, n, k, large, small):
    """Sums of about 2e7: times 1e34 beyond 3.4e38, times both scales about 2e5 or 2e9."""
    import cmpext3

    if kernel:
        monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    x, w, u = codes(m, k, seed=1), codes(n, k, seed=2), codes(n, k, seed=3)
    for sx, sw in ((large, small), (small, large)):
        xs, ws, us = scales(m, sx, 4), scales(n, sw, 5), scales(n, sw, 6)
        for dtype in (torch.bfloat16, torch.float32):
            want = R.int8_linear(x, xs, w, ws, None, dtype)
            assert 1e4 < want[0].abs().min() and want[0].abs().max() < 1e11
            R.check(cmpext3.int8_linear(x, w, ws, x_scale=xs, dtype=dtype), want)
            R.check(cmpext3.int8_gated_linear(x, w, u, ws, us, "relu", x_scale=xs, dtype=dtype), R.int8_gated(x, xs, w, ws, u, us, "relu", dtype))


@pytest.mark.parametrize("m", [1, 30, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_inputs_at_the_end_of_the_type(m, dtype):
    """x near 3e38, quantised on the way: the weights bring the results back into range."""
    import cmpext3

    g = torch.Generator(device=DEV).manual_seed(7)
    x = (torch.rand(m, 1024, generator=g, device=DEV) * 2e38 + 1e38).to(dtype)
    w, ws = codes(200, 1024, seed=8), scales(200, 1e-7, 9)
    q, s = cmpext3.quantize_int8(x)
    y = cmpext3.int8_linear(x, w, ws)
    assert torch.isfinite(y).all()
    R.check(y, R.int8_linear(q, s, w, ws, None, dtype))
