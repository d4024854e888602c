"""The gradients of gated_linear where a wrong slope cannot hide: along themselves, and at gates far out."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def rand(*shape, seed=0, size=1.0, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(dtype)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])  # relu has no third derivative at 0
def test_differences_along_the_gradient(act, which):
    """A step of 2^-4 each way along the gradient itself, of 1 (x) or 128^-1/2 (weights) in the mean square: the difference of
    the results' sum is the integral of the gradient along the step, by Simpson's rule on either half.

    The gradient in the middle alone would be off by a second derivative along the step, which is much here: the elements that
    move most are those with the largest gradients (5.3 % for w_gate, from the definition in 64 bits on these numbers).  One
    Simpson's rule over both halves leaves 1.6 %, a rule for each a sixteenth of that, 0.1 %.  The results' rounding, 2^-11 of about 1,
    independent in 2 * 6144 results, is 0.05 of a sum of some 700.  Asked for: 2 %."""
    import cmpext3

    x, w = rand(64, 128, seed=3), rand(192, 128, seed=4, size=128**-0.5)
    grad = rand(64, 96, seed=5)
    operands = [x, w[:96], w[96:]]

    def gradient(at):
        leaves = [t.clone().requires_grad_() for t in at]
        return torch.autograd.grad(cmpext3.gated_linear(*leaves, act), leaves, grad)[which].double()

    got = gradient(operands)
    v = got / got.square().mean().sqrt() * (1.0 if which == 0 else 128**-0.5)
    at = [list(operands) for _ in range(5)]
    for i in range(5):
        at[i][which] = (operands[which].double() + (i - 2) * 2.0**-5 * v).half()
    step = at[4][which].double() - at[0][which].double()  # as it was rounded
    diff = ((cmpext3.gated_linear(*at[4], act).double() - cmpext3.gated_linear(*at[0], act).double()) * grad.double()).sum().item()
    along = (sum(c / 12 * gradient(p) for c, p in zip((1, 4, 2, 4, 1), at)) * step).sum().item()
    assert along > 300 and abs(diff - along) < 0.02 * along, (diff, along)


@pytest.mark.parametrize("dtype,gates", [(torch.bfloat16, [64.0, 100.0, 1000.0, 1e6]), (torch.float16, [64.0, 100.0, 200.0])])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_slopes_far_out(act, dtype, gates):
    """One product of K = 1, exact: from |g| = 64 on the activation is g with slope 1, or 0 with slope 0, to 2^-70 at least
    (64 e^-64 for silu, less for the others)."""
    import cmpext3

    for g in [s * a for a in gates for s in (1.0, -1.0)]:
        x = torch.full((1, 1), g, device=DEV, dtype=dtype).requires_grad_()
        g = x.item()
        wg, wu = (torch.full((1, 1), s, device=DEV, dtype=dtype).requires_grad_() for s in (1.0, 2.0**-10))
        y = cmpext3.gated_linear(x, wg, wu, act)
        got = [t.item() for t in torch.autograd.grad(y, (x, wg, wu), torch.ones_like(y))]
        up, on = g * 2.0**-10, float(g > 0)
        # dgate = up slope, dup = act: held in 16 bits, then the products, rounded once more
        for a, b in zip(got, (on * (up * 1.0 + g * 2.0**-10), on * up * g, on * g * g)):
            assert abs(a - b) <= 2.1 * HALF_STEP[dtype] * abs(b) + 2.0**-25, (g, got)
