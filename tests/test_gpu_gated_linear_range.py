"""Gradients of a gated block in fp16 whose intermediate products lie outside fp16's range: dgate and dup above 65504
or below 2^-24, where the gradients that follow from them do not.

Bounds as in projection_ref, but for how dgate and dup are held: times a power of two that puts the largest of a row
(of both, for dx) or of a column (of one, for its weight) at 2^14 or more, so that an element is off by 2^-11 of itself or,
where that makes it subnormal, by 2^-25 of the unit: 2^-39 of the largest."""
import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
KERNELS = ["", "any64x64", "small64x64,splits=1,groups=1", "small64x64,splits=1,groups=2", "small64x64,splits=2,groups=2", "tile128x128,splits=1",
           "tile128x128,splits=3", "tile256x256"]
SIZES = [(1, 1, 1), (5, 40, 72), (70, 264, 136), (300, 257, 640), (129, 1100, 33)]


def rand(*shape, seed=0, size=1.0, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(dtype)


def held(d, e, largest):
    """The bound of an element known up to e, after it is held in fp16 beside others of up to `largest`."""
    return e + R.UNIT[torch.float16] * (d.abs() + e) + 2.0**-39 * largest


def backward(x, wg, wu, grad, name):
    """projection_ref.gated_backward with dgate and dup held as above."""
    t = torch.float16
    g, eg = R.products(x, wg)
    u, eu = R.products(x, wu)
    value, slope, bend = R.act(name, g)
    ea = R.act_error(name, g, value, eg)
    es = bend * eg + (1 + g.abs().clamp(max=40)) ** 2 * 2.0**-21
    if name == "relu":
        es = es + (g.abs() <= eg).double()
    d = grad.double()
    dg, du = d * u * slope, d * value
    edg = d.abs() * ((u.abs() + eu) * es + eu * slope.abs()) + 3 * R.F32 * dg.abs()
    edu = d.abs() * ea + 2 * R.F32 * du.abs()
    mg, mu = dg.abs() + edg, du.abs() + edu
    row = torch.maximum(mg, mu).amax(1, keepdim=True)

    def sums(pairs):
        y = sum(a @ b for a, _, b in pairs)
        k = sum(a.shape[1] for a, _, _ in pairs)
        tol = sum(e @ b.abs() + (a.abs() + e) @ b.abs() * (k * 2 * R.F32) for a, e, b in pairs)
        return y, R.rounded(y, tol, t)

    xd, wgd, wud = x.double(), wg.double(), wu.double()
    return (sums([(dg, held(dg, edg, row), wgd), (du, held(du, edu, row), wud)]),
            sums([(dg.t(), held(dg, edg, mg.amax(0, keepdim=True)).t(), xd)]),
            sums([(du.t(), held(du, edu, mu.amax(0, keepdim=True)).t(), xd)]))


def compare(x, wg, wu, grad, act):
    """The gradients, held to the definition; returns the definition's."""
    import cmpext3

    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(cmpext3.gated_linear(*leaves, act), leaves, grad)
    want = backward(x, wg, wu, grad, act)
    for name, a, b in zip(("dx", "dw_gate", "dw_up"), got, want):
        assert torch.isfinite(b[0]).all() and b[0].abs().max() < 65000, "the definition leaves fp16"
        R.check(a, b, name)
    return want


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_beyond_the_type(monkeypatch, kernel, m, n, k):
    """up is about 1000 and the gradient 300, so that dgate is 1e5 and more, infinite in fp16; w_gate and x are small, so
    that no gradient is."""
    if kernel:
        monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    size = 0.03 / m**0.5
    x, wu = rand(m, k, size=size), rand(n, k, seed=1, size=min(1000 / (size * k**0.5), 6000.0))
    wg = rand(n, k, seed=2, size=0.007 / n**0.5)
    grad = rand(m, n, seed=3, size=300.0)
    compare(x, wg, wu, grad, "silu")


@pytest.mark.parametrize("m,n,k", [(20000, 24, 16), (8200, 600, 24), (3, 5000, 40), (1, 4104, 8), (1030, 513, 24)])
def test_blocks_of_rows_and_columns(m, n, k):
    """Where the search for the largest values has many blocks of rows, of several rounds, or of columns, the last ones partly filled."""
    x, wu = rand(m, k, size=0.001), rand(n, k, seed=1, size=6000.0)
    wg, grad = rand(n, k, seed=2, size=0.001), rand(m, n, seed=3, size=1.0)
    grad[m - 1] *= 30
    grad[:, n - 1] *= 30
    grad[m // 2, n // 2] = 60000.0
    compare(x, wg, wu, grad, "silu")


@pytest.mark.parametrize("act", ACTS)
def test_each_activation_beyond_the_type(act):
    x, wu = rand(64, 64, size=0.005), rand(96, 64, seed=1, size=6000.0)
    compare(x, rand(96, 64, seed=2, size=0.001), wu, rand(64, 96, seed=3, size=1000.0), act)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", SIZES[1:])
def test_products_below_the_type(monkeypatch, kernel, m, n, k):
    """dgate and dup of about 1e-8, fp16's last digit and below, between rows of x of some hundreds (for dw), and between weights
    of some hundreds (for dx)."""
    if kernel:
        monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    grad = rand(m, n, seed=3, size=2e-5)
    x, w = rand(m, k, size=500.0), rand(2 * n, k, seed=1, size=2e-6 / k**0.5)
    want = compare(x, w[:n], w[n:], grad, "gelu")
    assert all(want[i][0].abs().max() > 1e-5 for i in (1, 2))  # where fp16 has digits
    x, w = rand(m, k, size=2e-6 / k**0.5), rand(2 * n, k, seed=1, size=500.0)
    assert compare(x, w[:n], w[n:], grad, "gelu")[0][0].abs().max() > 1e-5


def test_rows_and_channels_stay_apart():
    """One token with a gradient of 1e5 and more in one channel: the other tokens' dx and the other channels' dw keep their digits, and a
    token of infinite gradients leaves other tokens' dx alone."""
    import cmpext3

    m, n, k = 70, 130, 64
    x, wg = rand(m, k, size=0.01), rand(n, k, seed=1, size=1e-4)
    wu, grad = rand(n, k, seed=2, size=1.0), rand(m, n, seed=3, size=0.01)
    wu[7] *= 200.0
    grad[5, 7] = 60000.0
    compare(x, wg, wu, grad, "silu")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    bad = grad.clone()
    bad[9, 100] = torch.inf
    got = torch.autograd.grad(cmpext3.gated_linear(*leaves), leaves, bad)
    want = torch.autograd.grad(cmpext3.gated_linear(*leaves), leaves, grad)
    rows, channels = [i for i in range(m) if i != 9], [i for i in range(n) if i != 100]
    assert torch.equal(got[0][rows], want[0][rows]) and not torch.isfinite(got[0][9]).any()
    assert all(torch.equal(a[channels], b[channels]) for a, b in zip(got[1:], want[1:]))


def test_tokens_of_no_gradient():
    """Rows and channels of zeros (padding, relu below 0) have gradients of zero beside others of any size."""
    import cmpext3

    x, wg, wu = rand(33, 64), rand(40, 64, seed=1, size=0.1), rand(40, 64, seed=2, size=0.1)
    grad = rand(33, 40, seed=3, size=1e-5)
    grad[::2] = 0
    grad[:, 3] = 0
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(cmpext3.gated_linear(*leaves, "relu"), leaves, grad)
    for a, b in zip(got, backward(x, wg, wu, grad, "relu")):
        R.check(a, b)
    assert (got[0][::2] == 0).all() and (got[1][3] == 0).all() and (got[2][3] == 0).all()


@pytest.mark.parametrize("asked", [(0,), (1,), (2,), (1, 2), (0, 2)])
def test_some_gradients_only(asked):
    import cmpext3

    x, wu = rand(64, 64, size=0.005), rand(96, 64, seed=1, size=6000.0)
    wg, grad = rand(96, 64, seed=2, size=0.001), rand(64, 96, seed=3, size=1000.0)
    leaves = [t.clone().requires_grad_(i in asked) for i, t in enumerate((x, wg, wu))]
    want = backward(x, wg, wu, grad, "silu")
    for i, a in zip(asked, torch.autograd.grad(cmpext3.gated_linear(*leaves), [leaves[i] for i in asked], grad)):
        R.check(a, want[i])


@pytest.mark.parametrize("m", [8, 300])
def test_graph(m):
    """Captured and replayed with gradients of other sizes: units are found anew."""
    import cmpext3

    x, wg, wu = (t.requires_grad_() for t in (rand(m, 192), rand(264, 192, seed=1, size=0.07), rand(264, 192, seed=2, size=0.07)))
    grad = rand(m, 264, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(cmpext3.gated_linear(x, wg, wu), (x, wg, wu), grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(cmpext3.gated_linear(x, wg, wu), (x, wg, wu), grad)
    for seed in range(4):
        grad.copy_(rand(m, 264, seed=seed + 50, size=100.0 ** (seed - 2)))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in grads]
        want = torch.autograd.grad(cmpext3.gated_linear(x, wg, wu), (x, wg, wu), grad)
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
