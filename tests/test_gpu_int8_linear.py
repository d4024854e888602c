"""Projections with weights in 8-bit codes, and the codes themselves, against their definitions."""
import math

import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
DEV = "cuda"


def rand(*shape, seed=0, size=1.0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(dtype)


def rand_codes(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def scales(n, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (1, 64), (5, 127), (16, 1024), (33, 2050), (2, 14336), (3, 40000), (2, 3, 136)])
def test_quantize(dtype, shape):
    import cmpext3

    x = rand(*shape, dtype=dtype, size=3.0)
    q, s = cmpext3.quantize_int8(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.dtype == torch.float32 and s.shape == x.shape[:-1]
    want, scale = R.codes(x)
    off = (q.double() - want).abs()
    if dtype == torch.float32:
        # 127 x and its quotient are rounded: another code only next to the middle of two
        a = x.double().abs().amax(-1, keepdim=True)
        middle = ((127 * x.double() / a).abs() % 1 - 0.5).abs()
        assert (off[middle > 127 * 2.0**-22] == 0).all() and off.max() <= 1
    else:
        assert off.max() == 0
    R.check(s, (scale, R.rounded(scale, scale * 0, torch.float32)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_and_extremes(dtype):
    import cmpext3

    big = torch.finfo(dtype).max
    rows = torch.tensor([[2.0, 1.0, -1.0, 0.0], [254.0, 1.0, 3.0, -5.0], [0.0, -0.0, 0.0, 0.0], [big, -big, big / 2, 1.0],
                         [2.0**-20, 2.0**-21, -(2.0**-20), 0.0], [127.0, 0.5, 1.5, 2.5]], device=DEV).to(dtype)
    q, s = cmpext3.quantize_int8(rows)
    want, scale = R.codes(rows)
    assert torch.equal(q.double(), want)
    R.check(s, (scale, R.rounded(scale, scale * 0, torch.float32)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("cols", [5, 1032])
def test_quantize_rows_that_are_not_finite(dtype, bad, cols):
    import cmpext3

    x = rand(4, cols, dtype=dtype)
    x[1, cols - 1] = bad
    x[3, 0] = bad
    q, s = cmpext3.quantize_int8(x)
    assert torch.isnan(s).tolist() == [False, True, False, True]
    assert (q[1] == 0).all() and (q[3] == 0).all()
    assert torch.equal(q[0].double(), R.codes(x)[0][0]) or dtype == torch.float32
    y = cmpext3.int8_linear(x, rand_codes(9, cols), scales(9))
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()


def test_quantize_strides():
    import cmpext3

    x = rand(40, 300, dtype=torch.bfloat16)
    for view in (x[:, 3:200], x[::2, :256], x.t(), x[1:, 1:2], x.view(4, 10, 300)[:, 2:7, 8:264], x[:0], x[:, :0], x[5]):
        q, s = cmpext3.quantize_int8(view)
        want, scale = R.codes(view)
        assert torch.equal(q.double(), want) and q.is_contiguous()
        R.check(s, (scale, R.rounded(scale, scale * 0, torch.float32)))


SIZES = [(1, 1, 1), (1, 64, 64), (1, 4096, 4096), (2, 33, 130), (3, 7, 129), (4, 512, 1000), (16, 1024, 2048), (17, 100, 96),
         (31, 4099, 300), (33, 256, 4096), (64, 320, 1040), (65, 128, 128), (100, 129, 257), (128, 256, 512), (129, 65, 63),
         (200, 1001, 2050), (256, 256, 256), (257, 511, 640), (333, 300, 192), (512, 1024, 4096), (1000, 264, 16), (2048, 512, 768),
         (300, 2500, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int8_linear(dtype, m, n, k):
    import cmpext3

    x, w, xs, ws = rand_codes(m, k, seed=1), rand_codes(n, k, seed=2), scales(m, 3), scales(n, 4)
    bias = rand(n, seed=5, size=10.0, dtype=dtype)
    for b in (None, bias):
        y = cmpext3.int8_linear(x, w, ws, b, x_scale=xs, dtype=dtype)
        assert y.dtype == dtype and y.shape == (m, n)
        R.check(y, R.int8_linear(x, xs, w, ws, b, dtype), f"{m} x {n} x {k}")


@pytest.mark.parametrize("m,n,k", [(1, 96, 1024), (5, 512, 4096), (200, 300, 131071)])
def test_int8_largest_sums(m, n, k):
    """All codes at their ends: -128 too, which no row is quantised to, and sums near 2^31."""
    import cmpext3

    x = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    one = torch.ones(max(m, n), device=DEV)
    y = cmpext3.int8_linear(x, w, one[:n], x_scale=one[:m], dtype=torch.float32)
    R.check(y, R.int8_linear(x, one[:m], w, one[:n], None, torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 128, 512), (1, 4096, 4096), (1, 9000, 16384), (3, 70, 512), (4, 520, 4096), (16, 100, 1024), (8, 33, 2048),
                                   (17, 64, 512), (16, 300, 136), (77, 500, 1001), (300, 520, 2048), (5, 40, 15), (40, 1000, 100)])
def test_int8_linear_quantises_its_input(dtype, m, n, k):
    import cmpext3

    x, w, ws = rand(m, k, dtype=dtype), rand_codes(n, k, seed=2), scales(n, 4)
    y = cmpext3.int8_linear(x, w, ws)
    q, s = cmpext3.quantize_int8(x)
    assert y.dtype == dtype
    assert torch.equal(y, cmpext3.int8_linear(q, w, ws, x_scale=s, dtype=dtype))
    R.check(y, R.int8_linear(q, s, w, ws, None, dtype))
    y32 = cmpext3.int8_linear(x, w, ws, dtype=torch.float32)
    R.check(y32, R.int8_linear(q, s, w, ws, None, torch.float32))
    z = cmpext3.int8_gated_linear(x, w, w.flip(0), ws * 0.1, ws, "gelu")
    assert torch.equal(z, cmpext3.int8_gated_linear(q, w, w.flip(0), ws * 0.1, ws, "gelu", x_scale=s, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_int8_linear_of_few_rows_that_are_not_finite(dtype):
    import cmpext3

    x = rand(6, 1024, dtype=dtype)
    x[1, 1000], x[4, 0] = math.nan, math.inf
    w, ws = rand_codes(50, 1024, seed=2), scales(50, 4)
    y = cmpext3.int8_linear(x, w, ws)
    assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all()
    x[1, 1000], x[4, 0] = 0, 0
    z = cmpext3.int8_linear(x, w, ws)
    assert torch.equal(y[[0, 2, 3, 5]], z[[0, 2, 3, 5]])
    big = torch.zeros(2, 512, dtype=dtype, device=DEV)
    big[0, 0], big[0, 1] = torch.finfo(dtype).max, torch.finfo(dtype).max / 2
    q, s = cmpext3.quantize_int8(big)
    assert torch.equal(cmpext3.int8_linear(big, w[:, :512], ws), cmpext3.int8_linear(q, w[:, :512], ws, x_scale=s, dtype=dtype))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4096, 512), (4, 100, 1024), (16, 257, 160), (40, 96, 2049), (64, 640, 256), (100, 130, 72),
                                   (128, 128, 128), (300, 500, 1000), (600, 1030, 320)])
def test_int8_gated(act, dtype, m, n, k):
    import cmpext3

    x, wg, wu = rand_codes(m, k, seed=1), rand_codes(n, k, seed=2), rand_codes(n, k, seed=6)
    # gates of a few units, where activations bend
    xs, gs, us = scales(m, 3), scales(n, 4) * (0.3 / math.sqrt(k)), scales(n, 7)
    y = cmpext3.int8_gated_linear(x, wg, wu, gs, us, act, x_scale=xs, dtype=dtype)
    assert y.dtype == dtype and y.shape == (m, n)
    # results in 32 bits keep the hardware's 2^x and reciprocal, which act_error counts
    R.check(y, R.int8_gated(x, xs, wg, gs, wu, us, act, dtype), act)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_int8_strides_and_shapes(m):
    import cmpext3

    n, k = 70, 256
    big = rand_codes(m, 2, k + 48, seed=1)
    w = rand_codes(2 * n, k + 32, seed=2)
    xs, ws = scales(m, 3), scales(n, 4)
    for x in (big[:, 0, :k], big[:, 1, 16 : k + 16], big[:, 0, 3 : k + 3], big[:, 0].t()[:k].contiguous().t()):
        for wv in (w[::2, :k], w[:n, 16 : k + 16], w[n:, 5 : k + 5], w[:n, :k].t().contiguous().t()):
            R.check(cmpext3.int8_linear(x, wv, ws, x_scale=xs), R.int8_linear(x, xs, wv, ws, None, torch.bfloat16))
    x3 = rand_codes(2, m, k, seed=8)
    y = cmpext3.int8_linear(x3, w[:n, :k], ws, x_scale=scales(2 * m, 9).view(2, m))
    assert y.shape == (2, m, n)
    R.check(y.view(-1, n), R.int8_linear(x3.view(-1, k), scales(2 * m, 9), w[:n, :k], ws, None, torch.bfloat16))
    y1 = cmpext3.int8_linear(x3[0, 0], w[:n, :k], ws, x_scale=xs[0])
    assert y1.shape == (n,)


def test_int8_empty():
    import cmpext3

    w, ws = rand_codes(5, 32), scales(5)
    assert cmpext3.int8_linear(rand(0, 32), w, ws).shape == (0, 5)
    assert cmpext3.int8_linear(rand(3, 32), w[:0], ws[:0]).shape == (3, 0)
    bias = rand(5, seed=1)
    y = cmpext3.int8_linear(rand(3, 0), rand_codes(5, 0), ws, bias)
    assert torch.equal(y, bias.expand(3, 5))
    assert (cmpext3.int8_linear(rand(70, 0), rand_codes(5, 0), ws) == 0).all()
    assert (cmpext3.int8_gated_linear(rand(3, 0), rand_codes(5, 0), rand_codes(5, 0), ws, ws) == 0).all()


def test_int8_rows_stay_apart():
    """Rows of scale NaN or infinity, and a weight row of scale NaN, change nothing beside them."""
    import cmpext3

    for m in (3, 70, 300):
        x, w, xs, ws = rand_codes(m, 128, seed=1), rand_codes(40, 128, seed=2), scales(m, 3), scales(40, 4)
        xs[1], xs[2], ws[7] = math.nan, math.inf, math.nan
        y = cmpext3.int8_linear(x, w, ws, x_scale=xs, dtype=torch.float32)
        assert torch.isnan(y[1]).all() and torch.isnan(y[:, 7]).all()
        keep = [i for i in range(m) if i not in (1, 2)]
        cols = [i for i in range(40) if i != 7]
        R.check(y[keep][:, cols], R.int8_linear(x[keep], xs[keep], w[cols], ws[cols], None, torch.float32))


@pytest.mark.parametrize("m", [2, 48, 400])
def test_int8_graph(m):
    import cmpext3

    x = rand(m, 512, dtype=torch.bfloat16)
    w, wu, ws = rand_codes(384, 512, seed=2), rand_codes(384, 512, seed=3), scales(384, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cmpext3.int8_linear(x, w, ws)
        cmpext3.int8_gated_linear(x, w, wu, ws * 0.1, ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cmpext3.int8_linear(x, w, ws)
        z = cmpext3.int8_gated_linear(x, w, wu, ws * 0.1, ws)
    for seed in range(4):
        x.copy_(rand(m, 512, seed=seed, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        a, b = y.clone(), z.clone()
        assert torch.equal(a, cmpext3.int8_linear(x, w, ws))
        assert torch.equal(b, cmpext3.int8_gated_linear(x, w, wu, ws * 0.1, ws))
