"""Every kernel of the feed-forward operators on sizes that are not its own: chosen by CMPEXT3_PROJECTION_CONFIG, over
edges of tiles, steps and splits; the C ABI's own forms; calls that must be refused."""
import ctypes
import math

import pytest
import torch

from cmp_ext_amd import cabi
from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
KERNELS = ["any64x64", "rows", "small64x64,splits=1,groups=1", "small64x64,splits=1,groups=2", "small64x64,splits=2,groups=2", "small64x64,splits=3,groups=1",
           "tile128x128,splits=1", "tile128x128,splits=3", "tile256x128", "tile256x256"]
SIZES = [(1, 17, 64), (60, 65, 1032), (64, 32, 128), (65, 33, 129), (127, 250, 513), (129, 257, 640), (255, 130, 1999), (300, 70, 2048), (257, 513, 72)]


def rand(*shape, seed=0, size=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(dtype)


def rand_codes(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def scales(n, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_projections(monkeypatch, kernel, m, n, k):
    import cmpext3

    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    x, w, u, xs, ws = rand_codes(m, k, seed=1), rand_codes(n, k, seed=2), rand_codes(n, k, seed=3), scales(m, 3), scales(n, 4)
    for dtype in (torch.bfloat16, torch.float32):
        bias = rand(n, seed=5, dtype=dtype)
        R.check(cmpext3.int8_linear(x, w, ws, bias, x_scale=xs, dtype=dtype), R.int8_linear(x, xs, w, ws, bias, dtype))
        gs = ws * (0.3 / math.sqrt(k))
        R.check(cmpext3.int8_gated_linear(x, w, u, gs, ws, "gelu", x_scale=xs, dtype=dtype), R.int8_gated(x, xs, w, gs, u, ws, "gelu", dtype))
    for dtype in (torch.float16, torch.bfloat16):
        x16, wg, wu = rand(m, k, seed=1, dtype=dtype), rand(n, k, seed=2, size=k**-0.5, dtype=dtype), rand(n, k, seed=3, size=k**-0.5, dtype=dtype)
        R.check(cmpext3.gated_linear(x16, wg, wu), R.gated(x16, wg, wu, "silu"))


@pytest.mark.parametrize("kernel", [k for k in KERNELS if k != "rows"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gradients(monkeypatch, kernel, m, n, k):
    import cmpext3

    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    for dtype in (torch.float16, torch.bfloat16):
        leaves = [t.requires_grad_() for t in (rand(m, k, seed=1, dtype=dtype), rand(n, k, seed=2, size=k**-0.5, dtype=dtype),
                                               rand(n, k, seed=3, size=k**-0.5, dtype=dtype))]
        grad = rand(m, n, seed=4, dtype=dtype)
        got = torch.autograd.grad(cmpext3.gated_linear(*leaves, "gelu_tanh"), leaves, grad)
        for a, b in zip(got, R.gated_backward(*[t.detach() for t in leaves], grad, "gelu_tanh")):
            R.check(a, b)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nothing_outside_is_read_into_results_or_written(monkeypatch, kernel):
    """Operands and results inside larger tensors whose other elements are NaN, and stay as they are."""
    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    lib = cabi.lib()
    for m, n, k in [(5, 40, 72), (70, 33, 100), (130, 129, 65), (260, 70, 136)]:
        big = [torch.full((r + 2, c + 24), math.nan, device=DEV, dtype=torch.bfloat16) for r, c in ((m, k), (n, k), (n, k), (m, n))]
        x, wg, wu, out = (b[1 : 1 + r, 8 : 8 + c] for b, (r, c) in zip(big, ((m, k), (n, k), (n, k), (m, n))))
        x.copy_(rand(m, k)), wg.copy_(rand(n, k, seed=1, size=k**-0.5)), wu.copy_(rand(n, k, seed=2, size=k**-0.5))
        pre = torch.full((2, m + 1, n + 5), math.nan, device=DEV)
        a = cabi.ProjectionArgs(dtype=cabi.BF16, x_dtype=cabi.BF16, out_dtype=cabi.BF16, activation=cabi.ACT_SILU, M=m, N=n, K=k, x=x.data_ptr(),
                                x_row=k + 24, w_gate=wg.data_ptr(), gate_row=k + 24, w_up=wu.data_ptr(), up_row=k + 24, out=out.data_ptr(),
                                out_row=n + 24, gate_out=pre[0].data_ptr(), up_out=pre[1].data_ptr(), pre_row=n + 5)
        need = lib.cmpext3_projection_workspace_size(ctypes.byref(a))
        ws = torch.empty(max(need, 16), device=DEV, dtype=torch.uint8)
        assert lib.cmpext3_projection(ctypes.byref(a), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        R.check(out, R.gated(x, wg, wu, "silu"))
        for i, w in enumerate((wg, wu)):
            y, tol = R.products(x, w)
            R.check(pre[i, :m, :n], (y, R.rounded(y, tol, torch.float32)))
        assert torch.isnan(pre[:, m:]).all() and torch.isnan(pre[:, :, n:]).all()
        inside = torch.zeros_like(big[3], dtype=torch.bool)
        inside[1 : 1 + m, 8 : 8 + n] = True
        assert torch.isnan(big[3][~inside]).all()


def test_workspace_shared_by_two_captured_calls():
    """Two calls in one graph, one after the other, and two graphs replayed in turn: each has its own results."""
    import cmpext3

    x, w, ws = rand(100, 1000, dtype=torch.float16), rand_codes(300, 1000, seed=1), scales(300, 2)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cmpext3.int8_linear(x, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    for s in (1.0, 2.0):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((cmpext3.int8_linear(x * s, w, ws), cmpext3.int8_linear(x * -s, w, ws)))
        graphs.append(g)
    for i in (0, 1, 1, 0):
        x.copy_(rand(100, 1000, seed=10 + i, dtype=torch.float16))
        for g, s, (a, b) in zip(graphs, (1.0, 2.0), outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, cmpext3.int8_linear(x * s, w, ws)) and torch.equal(b, cmpext3.int8_linear(x * -s, w, ws))


def test_capture_is_refused_while_an_eager_graph_holds_a_leaf():
    import cmpext3

    x, wg, wu = rand(16, 64), rand(32, 64, seed=1).requires_grad_(), rand(32, 64, seed=2).requires_grad_()
    held = cmpext3.gated_linear(x, wg, wu)  # its graph lives on
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="made on another stream"):
        with torch.cuda.graph(graph):
            cmpext3.gated_linear(x, wg, wu)
    torch.cuda.synchronize()
    grads = torch.autograd.grad(held, (wg, wu), torch.ones_like(held))  # as before
    for a, b in zip(grads, R.gated_backward(x, wg.detach(), wu.detach(), torch.ones_like(held), "silu")[1:]):
        R.check(a, b)
    del held, grads
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cmpext3.gated_linear(x, wg, wu)
    graph.replay()
    torch.cuda.synchronize()
    R.check(y.detach(), R.gated(x, wg.detach(), wu.detach(), "silu"))


def refuses(match, fn, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def test_refusals():
    import cmpext3

    x, w, s = rand(4, 32), rand_codes(6, 32), scales(6)
    wh = rand(6, 32)
    f, g, h = cmpext3.int8_linear, cmpext3.int8_gated_linear, cmpext3.gated_linear
    refuses("weights must be 2-D", f, x, w[0], s)
    refuses("shape mismatch", f, x[:, :31], w, s)
    refuses("int8 codes", f, x, wh, s)
    refuses("unsupported input dtype", f, x.double(), w, s)
    refuses("an int8 input needs x_scale", f, w, w, s)
    refuses("only an int8 input has x_scale", f, x, w, s, x_scale=scales(4))
    refuses("x_scale must have 6", f, w, w, s, x_scale=scales(4))
    refuses("must be float32", f, x, w, s.double())
    refuses("must have 6 elements", f, x, w, scales(5))
    refuses("unsupported output dtype", f, x, w, s, dtype=torch.float64)
    refuses("bias must have 6", f, x, w, s, rand(5))
    refuses("output's dtype", f, x, w, s, rand(6, dtype=torch.float32))
    refuses("must be on a GPU", f, x, w.cpu(), s)
    refuses("must be on a GPU", f, x, w, s.cpu())
    refuses("32-bit sums", f, torch.zeros(1, 131072, device=DEV), torch.zeros(2, 131072, device=DEV, dtype=torch.int8), scales(2))
    refuses("weight shape mismatch", g, x, w, w[:5], s, s)
    refuses("weight dtype mismatch", g, x, w, wh, s, s)
    refuses("unknown activation", g, x, w, w, s, s, "swish")
    refuses("unknown activation", h, x, wh, wh, "")
    refuses("unsupported dtype", h, x.float(), wh.float(), wh.float())
    refuses("dtype mismatch", h, x.half(), wh, wh)
    refuses("weight dtype mismatch", h, x, wh, wh.half())
    refuses("weight shape mismatch", h, x, wh, wh[:3])
    refuses("unsupported dtype", cmpext3.quantize_int8, w)


def test_gradients_have_no_gradient():
    import cmpext3

    x, wg, wu = (t.requires_grad_() for t in (rand(8, 16), rand(8, 16, seed=1), rand(8, 16, seed=2)))
    y = cmpext3.gated_linear(x, wg, wu)
    (d,) = torch.autograd.grad(y.float().square().sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once only"):
        d.sum().backward()


@pytest.mark.parametrize("kernel", ["tile128x128,splits=1", "small64x64"])
def test_odd_rows_while_memory_is_mapped(monkeypatch, kernel):
    """Rows that are shifted into place, beside allocations that come and go: every call gives the same bits."""
    import cmpext3

    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=" + kernel)
    x, w, u = rand_codes(300, 1000, seed=1), rand_codes(500, 1000, seed=2), rand_codes(500, 1000, seed=3)
    xs, ws = scales(300, 3), scales(500, 4)
    want = None
    for i in range(150):
        t = torch.empty(1 << (20 + i % 5), device=DEV)
        t.fill_(1.0)
        noise = torch.empty(170000, device=DEV, dtype=torch.float64).normal_()
        del t, noise
        if i % 25 == 0:
            torch.cuda.empty_cache()
        y = cmpext3.int8_gated_linear(x, w, u, ws * 0.01, ws, x_scale=xs, dtype=torch.float32)
        if want is None:
            want = y.clone()
            R.check(y, R.int8_gated(x, xs, w, ws * 0.01, u, ws, "silu", torch.float32))
        assert torch.equal(y, want), i
