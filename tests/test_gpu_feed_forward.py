"""The feed-forward operators together, as the example has them: a block's training step against autograd in 64
bits, the served block step by step against its definition, captured and replayed, and the example's own run."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXAMPLE = os.path.join(ROOT, "examples", "feed_forward.py")
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("feed_forward", EXAMPLE)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("tokens,width,inner", [(7, 48, 72), (130, 264, 520), (300, 101, 75)])
def test_gradients_of_a_block(example, dtype, act, tokens, width, inner):
    block = example.FeedForward(width, inner, act, dtype, "cuda", seed=1)
    x = torch.randn(tokens, width, device="cuda").to(dtype).requires_grad_()
    grad = torch.randn(tokens, width, device="cuda").to(dtype)
    y = block.forward(x)
    got = torch.autograd.grad(y, (x, block.w_in, block.w_down), grad)
    # the gradient that reaches the operator is torch's product, rounded: taken as it is
    d = torch.matmul(grad, block.w_down.detach())
    wg, wu = block.w_in.detach()[:inner], block.w_in.detach()[inner:]
    want = R.gated_backward(x.detach(), wg, wu, d, act)
    R.check(got[0], want[0], "dx")
    R.check(got[1][:inner], want[1], "dw_gate")
    R.check(got[1][inner:], want[2], "dw_up")
    h, th = R.gated(x.detach(), wg, wu, act)
    dw = grad.double().t() @ h
    tol = grad.double().abs().t() @ (th + h.abs() * tokens * 2.0**-23)
    R.check(got[2], (dw, R.rounded(dw, tol, dtype)), "dw_down")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 5, 40, 200])
@pytest.mark.parametrize("width,inner", [(512, 1024), (100, 333)])
def test_served_block(example, dtype, tokens, width, inner):
    block = example.FeedForward(width, inner, "silu", dtype, "cuda", seed=2)
    served = example.ServedFeedForward(block)
    w = torch.cat([served.gate, served.up])
    want, scale = R.codes(block.w_in.detach())
    assert torch.equal(w.double(), want)
    x = torch.randn(tokens, width, device="cuda").to(dtype)
    import cmpext3

    h = cmpext3.int8_gated_linear(x, served.gate, served.up, served.gate_scale, served.up_scale)
    q, s = R.codes(x)
    s32 = s.float()
    R.check(h, R.int8_gated(q, s32, served.gate, served.gate_scale, served.up, served.up_scale, "silu", dtype))
    q, s = R.codes(h)
    y = served.forward(x)
    R.check(y, R.int8_linear(q, s.float(), served.w_down, served.down_scale, None, dtype))
    # and near the block in 16 bits: codes are off by half a step of 1 / 127 of their row's largest value
    z = block.forward(x).float()
    assert ((y.float() - z).norm() / z.norm()).item() < 0.05


@pytest.mark.parametrize("tokens", [1, 60, 300])
def test_served_block_captured(example, tokens):
    block = example.FeedForward(512, 1024, "gelu_tanh", torch.bfloat16, "cuda", seed=3)
    served = example.ServedFeedForward(block)
    x = torch.randn(tokens, 512, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        served.forward(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = served.forward(x)
    for seed in range(4):
        x.copy_(torch.randn(tokens, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, served.forward(x))


@pytest.mark.parametrize("rate", [2.0**-12, 0.125])  # the larger one leaves the numbers: bits are compared, NaN among them
def test_captured_training_step(example, rate):
    """A whole step, weights updated in place, against the same steps run eagerly."""
    def same(a, b):
        return torch.equal(a.detach().view(torch.int16), b.detach().view(torch.int16))

    def make():
        return example.FeedForward(256, 512, "silu", torch.bfloat16, "cuda", seed=4)

    x = torch.randn(96, 256, device="cuda").to(torch.bfloat16)
    target = torch.randn(96, 256, device="cuda")
    block, eager = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        example.train_step(make(), x, target, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.forward(x)
        grads = torch.autograd.grad(y, (block.w_in, block.w_down), y)
        with torch.no_grad():
            block.w_in -= rate * grads[0]
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        z = eager.forward(x)
        want = torch.autograd.grad(z, (eager.w_in, eager.w_down), z)
        assert same(grads[0], want[0])
        with torch.no_grad():
            eager.w_in -= rate * want[0]
        assert same(block.w_in, eager.w_in)
        assert rate > 0.1 or torch.isfinite(block.w_in).all()


def test_example_runs():
    for args in (["--steps", "2", "--tokens", "64"], ["--dtype", "fp16", "--act", "gelu", "--steps", "1", "--tokens", "33", "--width", "200", "--inner", "300"]):
        out = subprocess.run([sys.executable, EXAMPLE, *args], capture_output=True, text=True, timeout=110)
        assert out.returncode == 0, out.stdout + out.stderr
        assert "relative difference" in out.stdout
