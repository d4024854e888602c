"""Feed-forward operators on tensors of more than 2^31 elements and bytes past 4 GiB: offsets of 64 bits."""
import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ends(n, many=300):
    """Some first, middle and last indices."""
    return torch.cat([torch.arange(many), torch.arange(n // 2, n // 2 + many), torch.arange(n - many, n)]).to(DEV)


def test_results_past_32_bits():
    import cmpext3

    m, n, k = 70001, 40008, 64  # 2.8e9 results
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randint(-127, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    xs, ws = torch.rand(m, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    y = cmpext3.int8_linear(x, w, ws, x_scale=xs)
    rows = ends(m, 100)
    R.check(y[rows], R.int8_linear(x[rows], xs[rows], w, ws, None, torch.bfloat16))
    del y
    y = cmpext3.int8_gated_linear(x, w, w.flip(0), ws * 0.001, ws, x_scale=xs)
    R.check(y[rows], R.int8_gated(x[rows], xs[rows], w, ws * 0.001, w.flip(0), ws, "silu", torch.bfloat16))


def test_codes_past_32_bits():
    import cmpext3

    rows, cols = 140000, 16384  # 2.3e9 elements
    x = torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16).normal_()
    q, s = cmpext3.quantize_int8(x)
    at = ends(rows)
    want, scale = R.codes(x[at])
    assert torch.equal(q[at].double(), want)
    R.check(s[at], (scale, R.rounded(scale, scale * 0, torch.float32)))


@pytest.mark.parametrize("k", [8192, 8191])
def test_gradients_of_a_long_batch(k):
    """x of 4.9 GB: rows and steps of k past 4 GiB from its start."""
    import cmpext3

    m, n = 300000, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(m, k, generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_()
    wg, wu = ((torch.randn(n, k, generator=g, device=DEV) * k**-0.5).to(torch.bfloat16).requires_grad_() for _ in range(2))
    grad = torch.zeros(m, n, device=DEV, dtype=torch.bfloat16)
    rows = ends(m)  # the others add nothing to the weights' gradients
    grad[rows] = torch.randn(len(rows), n, generator=g, device=DEV).to(torch.bfloat16)
    y = cmpext3.gated_linear(x, wg, wu)
    R.check(y.detach()[rows], R.gated(x.detach()[rows], wg.detach(), wu.detach(), "silu"))
    got = torch.autograd.grad(y, (x, wg, wu), grad)
    want = R.gated_backward(x.detach()[rows], wg.detach(), wu.detach(), grad[rows], "silu")
    R.check(got[0][rows], want[0])
    R.check(got[1], want[1])
    R.check(got[2], want[2])
    assert (got[0][1000:2000] == 0).all()
