"""The gated block's first half and its gradients, against the definition, autograd in 64 bits and differences."""
import math

import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
DEV = "cuda"


def rand(*shape, seed=0, size=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(dtype)


def operands(m, n, k, dtype, seed=0):
    size = max(k, 1) ** -0.5
    return rand(m, k, seed=seed, dtype=dtype), rand(n, k, seed=seed + 1, size=size, dtype=dtype), rand(n, k, seed=seed + 2, size=size, dtype=dtype)


SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 1024), (2, 33, 65), (4, 300, 512), (16, 1024, 256), (17, 100, 48), (31, 515, 300), (33, 128, 1024),
         (64, 200, 520), (65, 128, 64), (77, 273, 101), (128, 128, 128), (129, 130, 72), (200, 500, 1001), (256, 256, 256), (300, 257, 640),
         (513, 384, 200), (1000, 136, 24), (600, 1500, 320)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward(dtype, act, m, n, k):
    import cmpext3

    x, wg, wu = operands(m, n, k, dtype)
    y = cmpext3.gated_linear(x, wg, wu, act)
    assert y.dtype == dtype and y.shape == (m, n) and not y.requires_grad
    R.check(y, R.gated(x, wg, wu, act), f"{m} x {n} x {k}")


GRAD_SIZES = [(1, 1, 1), (1, 64, 64), (3, 33, 65), (16, 128, 256), (40, 100, 48), (64, 256, 128), (100, 273, 101), (130, 128, 72), (256, 256, 256),
              (300, 257, 640), (513, 384, 200), (31, 515, 300), (700, 640, 520)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", GRAD_SIZES)
def test_backward(dtype, act, m, n, k):
    import cmpext3

    x, wg, wu = (t.requires_grad_() for t in operands(m, n, k, dtype, seed=10))
    grad = rand(m, n, seed=20, dtype=dtype)
    y = cmpext3.gated_linear(x, wg, wu, act)
    with torch.no_grad():
        assert torch.equal(y, cmpext3.gated_linear(x, wg, wu, act))  # the same with and without what is kept
    got = torch.autograd.grad(y, (x, wg, wu), grad)
    want = R.gated_backward(x.detach(), wg.detach(), wu.detach(), grad, act)
    for name, a, b, t in zip(("dx", "dw_gate", "dw_up"), got, want, (x, wg, wu)):
        assert a.dtype == dtype and a.shape == t.shape
        R.check(a, b, f"{name} {m} x {n} x {k}")


@pytest.mark.parametrize("act", ACTS)
def test_formula_against_autograd_and_differences(act):
    """The formula that the kernels are held to, against autograd in 64 bits and central differences."""
    torch.manual_seed(0)
    x, wg, wu = (t.double().requires_grad_() for t in (torch.randn(9, 7), torch.randn(5, 7), torch.randn(5, 7)))
    grad = torch.randn(9, 5).double()

    def loss(x, wg, wu):
        return (R.act(act, x @ wg.t())[0] * (x @ wu.t()) * grad).sum()

    auto = torch.autograd.grad(loss(x, wg, wu), (x, wg, wu))
    xd, gd, ud = x.detach(), wg.detach(), wu.detach()
    g, u = xd @ gd.t(), xd @ ud.t()
    value, slope, _ = R.act(act, g)
    dg, du = grad * u * slope, grad * value
    formula = (dg @ gd + du @ ud, dg.t() @ xd, du.t() @ xd)
    for a, b in zip(auto, formula):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-12)
    h = 1e-5
    for i in range(3):
        v = torch.randn_like((xd, gd, ud)[i])
        plus, minus = [xd, gd, ud], [xd, gd, ud]
        plus[i], minus[i] = plus[i] + h * v, minus[i] - h * v
        assert abs(((loss(*plus) - loss(*minus)) / (2 * h) - (formula[i] * v).sum()).item()) < 1e-6 * (1 + (formula[i] * v).sum().abs().item())


@pytest.mark.parametrize("act", [a for a in ACTS if a != "relu"])  # which has no third derivative at 0
def test_gradient_against_differences_of_the_result(act):
    """Directional differences of the operator's own result: a step of 2^-4 along v, where rounding (2^-11 of
    each result) and the third derivative (below 2, times h^2 / 6) both stay below 2 % of the sizes summed."""
    import cmpext3

    x, wg, wu = operands(64, 96, 128, torch.float16, seed=3)
    grad = rand(64, 96, seed=4, dtype=torch.float16)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(cmpext3.gated_linear(*leaves, act), leaves, grad)
    for i in range(3):
        v = torch.randn_like(leaves[i].float()) * (1.0 if i == 0 else 128**-0.5)
        h = 2.0**-4
        a, b = [x, wg, wu], [x, wg, wu]
        a[i], b[i] = (a[i].float() + h * v).half(), (b[i].float() - h * v).half()
        step = (a[i].double() - b[i].double())  # as it was rounded
        diff = ((cmpext3.gated_linear(*a, act).double() - cmpext3.gated_linear(*b, act).double()) * grad.double()).sum().item()
        along = (got[i].double() * step).sum().item()
        size = (got[i].double() * step).norm().item() * 3 + 1
        assert abs(diff - along) < 0.1 * size, (i, diff, along, size)


def test_some_gradients_only():
    import cmpext3

    x, wg, wu = operands(40, 72, 56, torch.bfloat16)
    grad = rand(40, 72, seed=9)
    want = R.gated_backward(x, wg, wu, grad, "silu")
    for asked in [(0,), (1,), (2,), (0, 2), (1, 2)]:
        leaves = [t.clone().requires_grad_(i in asked) for i, t in enumerate((x, wg, wu))]
        y = cmpext3.gated_linear(*leaves)
        got = torch.autograd.grad(y, [leaves[i] for i in asked], grad)
        for i, a in zip(asked, got):
            R.check(a, want[i])
    with pytest.raises(RuntimeError):  # once only
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
        (d,) = torch.autograd.grad(cmpext3.gated_linear(*leaves), leaves[:1], grad, create_graph=True)
        torch.autograd.grad(d.sum(), leaves[1:2])


def test_shared_and_expanded_inputs():
    """One tensor as both weights, one row for a whole batch, a sum's gradient (stride 0), halves of one weight."""
    import cmpext3

    x, wg, wu = operands(48, 64, 80, torch.bfloat16)
    w = wg.clone().requires_grad_()
    grad = rand(48, 64, seed=7)
    cmpext3.gated_linear(x, w, w).backward(grad)
    _, (a, ta), (b, tb) = R.gated_backward(x, wg, wg, grad, "silu")
    R.check(w.grad, (a + b, R.rounded(a + b, ta + tb, torch.bfloat16)))

    row = x[:1].clone().requires_grad_()
    cmpext3.gated_linear(row.expand(48, 80), wg, wu).sum().backward()
    (d, t), _, _ = R.gated_backward(x[:1].expand(48, 80), wg, wu, torch.ones(48, 64, device=DEV), "silu")
    d, t = d.sum(0, keepdim=True), t.sum(0, keepdim=True)
    assert row.grad.shape == (1, 80)
    R.check(row.grad, (d, R.rounded(d, t + 48 * R.UNIT[torch.bfloat16] * d.abs(), torch.bfloat16)))

    both = torch.cat([wg, wu]).requires_grad_()
    x3 = x.view(4, 12, 80)
    y = cmpext3.gated_linear(x3, both[:64], both[64:])
    assert y.shape == (4, 12, 64)
    y.backward(grad.view(4, 12, 64))
    _, (a, ta), (b, tb) = R.gated_backward(x, wg, wu, grad, "silu")
    R.check(both.grad, (torch.cat([a, b]), torch.cat([ta, tb])))


@pytest.mark.parametrize("m", [3, 60, 200])
def test_strides(m):
    import cmpext3

    n, k = 70, 128
    xs, ws = rand(m, 2, k + 24, seed=1), rand(2 * n, k + 24, seed=2, size=0.1)
    grad = rand(n, m, seed=3).t()
    for x in (xs[:, 0, :k], xs[:, 1, 8 : k + 8], xs[:, 0, 3 : k + 3], xs[:, 0, :k].t().contiguous().t()):
        for wg, wu in ((ws[:n, :k], ws[n:, :k]), (ws[::2, 8 : k + 8], ws[1::2, 1 : k + 1]), (ws[:n, :k].t().contiguous().t(), ws[n:, 2 : k + 2])):
            R.check(cmpext3.gated_linear(x, wg, wu, "gelu"), R.gated(x, wg, wu, "gelu"))
            leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
            got = torch.autograd.grad(cmpext3.gated_linear(*leaves, "gelu"), leaves, grad)
            for a, b in zip(got, R.gated_backward(x, wg, wu, grad, "gelu")):
                R.check(a, b)


def test_empty():
    import cmpext3

    for m, n, k in [(0, 8, 16), (5, 0, 16), (5, 8, 0), (0, 0, 0), (200, 8, 0)]:
        leaves = [t.requires_grad_() for t in operands(m, n, k, torch.float16)]
        y = cmpext3.gated_linear(*leaves)
        assert y.shape == (m, n) and (y == 0).all()
        for d, t in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
            assert d.shape == t.shape and (d == 0).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [4, 130])
def test_values_that_are_not_numbers_stay_in_their_row(act, m):
    import cmpext3

    x, wg, wu = operands(m, 72, 64, torch.bfloat16, seed=5)
    clean = cmpext3.gated_linear(x, wg, wu, act)
    x[1, 5], x[2, 63] = math.nan, math.inf
    y = cmpext3.gated_linear(x, wg, wu, act)
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("act", ACTS)
def test_large_gates(act):
    """Gates far out: the activation is 0 or the gate itself, its derivative 0 or 1, none of them NaN."""
    import cmpext3

    g = torch.tensor([-3e38, -1e30, -1e15, -1000.0, -100.0, -64.0, 64.0, 100.0, 1000.0, 1e15, 1e30], device=DEV).to(torch.bfloat16)
    x = g[:, None].clone().requires_grad_()
    one = torch.ones(1, 1, device=DEV, dtype=torch.bfloat16)
    small = torch.full((1, 1), 2.0**-100, device=DEV, dtype=torch.bfloat16)
    wg, wu = one.clone().requires_grad_(), small.clone().requires_grad_()
    y = cmpext3.gated_linear(x, wg, wu, act)
    pos = g > 0
    u = (g.double() * 2.0**-100).to(torch.bfloat16)
    want = torch.where(pos, g.double() * u.double(), torch.zeros_like(u).double())
    R.check(y[:, 0], (want, R.rounded(want, want.abs() * 2.0**-7 + 1e-24, torch.bfloat16)))
    dx, dwg, dwu = torch.autograd.grad(y, (x, wg, wu), torch.full_like(y, 2.0**-30))
    assert torch.isfinite(dx).all() and not torch.isnan(dwg).any() and not torch.isnan(dwu).any()
    assert (dx[~pos] == 0).all() or act != "relu"


def test_other_stream_and_threads():
    import threading

    import cmpext3

    x, wg, wu = operands(300, 257, 200, torch.float16)
    want = cmpext3.gated_linear(x, wg, wu)
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(3):
                got[i] = cmpext3.gated_linear(x, wg, wu)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("m", [8, 300])
def test_graph_with_backward(m):
    import cmpext3

    x, wg, wu = (t.requires_grad_() for t in operands(m, 264, 192, torch.bfloat16))
    grad = rand(m, 264, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(cmpext3.gated_linear(x, wg, wu), (x, wg, wu), grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cmpext3.gated_linear(x, wg, wu)
        grads = torch.autograd.grad(y, (x, wg, wu), grad)
    for seed in range(4):
        with torch.no_grad():
            x.copy_(rand(m, 192, seed=seed))
            grad.copy_(rand(m, 264, seed=seed + 50))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.detach().clone() for t in (y, *grads)]
        again = cmpext3.gated_linear(x, wg, wu)
        want = [again, *torch.autograd.grad(again, (x, wg, wu), grad)]
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_results_do_not_change_from_run_to_run():
    import cmpext3

    for m, n, k in [(16, 1024, 512), (512, 1024, 640)]:
        leaves = [t.requires_grad_() for t in operands(m, n, k, torch.bfloat16)]
        grad = rand(m, n, seed=8)
        runs = []
        for _ in range(3):
            y = cmpext3.gated_linear(*leaves)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, grad)])
        assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
