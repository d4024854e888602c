"""Capturing gated_linear whose inputs are views or results of leaves: an eager graph that still holds such a leaf is seen."""
import pytest
import torch

from tests import projection_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(torch.bfloat16)


def captured(fn):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_refused_while_an_eager_graph_holds_the_leaf():
    """Only the forward call is captured, so that nothing reaches a backward pass where it is not refused."""
    import cmpext3

    x, both = rand(16, 64), rand(64, 64, seed=1, size=0.1).requires_grad_()
    hold = cmpext3.gated_linear(x, both[:32], both[32:])  # its graph lives on
    with pytest.raises(RuntimeError, match="made on another stream"):
        captured(lambda: cmpext3.gated_linear(x, both[:32], both[32:]))
    halves = both[:32], both[32:]  # views made before the capture
    with pytest.raises(RuntimeError, match="made on another stream"):
        captured(lambda: cmpext3.gated_linear(x, *halves))
    leaf = rand(16, 64, seed=2).requires_grad_()
    hidden = leaf * 2  # a result instead of a view, two steps from its leaf
    with pytest.raises(RuntimeError, match="made on another stream"):
        captured(lambda: cmpext3.gated_linear(hidden.relu(), both.detach()[:32], both.detach()[32:]))
    torch.cuda.synchronize()
    (d,) = torch.autograd.grad(hold, both, torch.ones_like(hold))  # as before
    want = R.gated_backward(x, both.detach()[:32], both.detach()[32:], torch.ones_like(hold), "silu")
    R.check(d[:32], want[1])
    R.check(d[32:], want[2])


@pytest.mark.parametrize("tokens", [8, 200])
def test_captured_with_its_backward_pass(tokens):
    """Views of one weight and a result as x, all made inside the capture, no eager graph alive: replays give the eager gradients."""
    import cmpext3

    leaf, both, grad = rand(tokens, 64, seed=2).requires_grad_(), rand(144, 64, seed=1, size=0.1).requires_grad_(), rand(tokens, 72, seed=3)

    def step():
        y = cmpext3.gated_linear(leaf * 2, both[:72], both[72:])
        return [y.detach(), *torch.autograd.grad(y, (leaf, both), grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, got = captured(step)
    for seed in range(4):
        with torch.no_grad():
            leaf.copy_(rand(tokens, 64, seed=seed + 10))
            grad.copy_(rand(tokens, 72, seed=seed + 20))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
