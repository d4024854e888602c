"""The operators of a feed-forward block, as cases that can be timed and checked:

  int8        a projection with weights in 8-bit integers: activations quantised for each token, the product in
              integers, scales for each token and channel, a bias
  gated       act(x Wg^T) * (x Wu^T): both projections of a gated block, its activation and the product
  train       the same with its backward pass: gradients of the input and of both weights
  int8_gated  the gated block's first half with weights in 8-bit integers

`run` computes a case from elementary torch operations in 32 bits, or, where `own` is true, through the
framework's operators.  Sizes go from a single token, all latency, to prompts and training batches that are bound
by the matrix cores; tokens, channels and inner sizes are odd or ragged in some.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
MOST = 127.0           # the largest code
LEAST_AMAX = 2.0**-100  # rows smaller than this share its scale
GRAD_SIZE = 0.1        # of the gradients that come back to a block


def _int8(dtype, tokens, inner, channels, bias):
    return {"op": "int8", "dtype": dtype, "tokens": tokens, "inner": inner, "channels": channels, "bias": bias}


def _gated(op, dtype, tokens, inner, channels, act):
    return {"op": op, "dtype": dtype, "tokens": tokens, "inner": inner, "channels": channels, "act": act}


def listed():
    return [
        # generation of one sequence, an attention layer's projection: a call that is all latency
        dict(_int8("bf16", 1, 4096, 4096, False), name="int8_decode1"),
        # generation for 16 sequences: bound by reading the weights
        dict(_int8("bf16", 16, 8192, 8192, False), name="int8_decode16"),
        # a short prompt, every size ragged, with a bias
        dict(_int8("fp16", 333, 2050, 1001, True), name="int8_ragged"),
        # a prompt of 4096 tokens through a block's second projection: bound by the matrix cores
        dict(_int8("bf16", 4096, 14336, 4096, False), name="int8_prompt"),
        # generation for 16 sequences
        dict(_gated("gated", "bf16", 16, 4096, 14336, "silu"), name="gated_decode16"),
        # a few requests' tokens, odd inner size (rows of no whole 16 bytes), another activation
        dict(_gated("gated", "fp16", 77, 1001, 2731, "gelu"), name="gated_odd"),
        # a prompt of 4096 tokens
        dict(_gated("gated", "bf16", 4096, 4096, 14336, "silu"), name="gated_prompt"),
        # a training step of a small model
        dict(_gated("train", "fp16", 500, 1024, 2816, "gelu_tanh"), name="train_small"),
        # a training step of a large one, the largest case
        dict(_gated("train", "bf16", 4096, 4096, 14336, "silu"), name="train_large"),
        # generation for a few sequences
        dict(_gated("int8_gated", "bf16", 4, 4096, 14336, "silu"), name="int8_gated_decode4"),
        # a batch of verified draft tokens, odd sizes
        dict(_gated("int8_gated", "fp16", 100, 1000, 4099, "gelu_tanh"), name="int8_gated_ragged"),
        # a prompt of 2048 tokens
        dict(_gated("int8_gated", "bf16", 2048, 4096, 11008, "silu"), name="int8_gated_prompt"),
    ]


def _size(rng, lo, hi):
    """A whole number from lo to hi, uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    """A size of a layer: mostly a multiple of 64 or 8, sometimes any number."""
    n = _size(rng, lo, hi)
    unit = rng.choice([64, 64, 64, 8, 8, 1])
    return max(1, n // unit) * unit


def draw(rng):
    while True:
        op = rng.choice(["int8", "int8", "gated", "gated", "train", "int8_gated"])
        dtype = rng.choice(["fp16", "bf16"])
        tokens = _size(rng, 1, 64) if rng.random() < 0.4 and op != "train" else _size(rng, 16, 8192)
        inner, channels = _width(rng, 64, 16384), _width(rng, 64, 16384)
        if op == "int8":
            case = _int8(dtype, tokens, inner, channels, rng.random() < 0.3)
        else:
            case = _gated(op, dtype, tokens, inner, channels, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]))
        most = work(listed()[8])
        got = work(case)
        if got["flops"] <= most["flops"] and got["bytes"] <= most["bytes"]:
            return case


def _normal(gen, shape, size):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * size


def _weight_codes(gen, channels, inner):
    """A weight in codes with a scale for each of its rows, as a program keeps it."""
    w = _normal(gen, (channels, inner), inner**-0.5)
    scale = w.abs().amax(-1).clamp(min=LEAST_AMAX) / MOST
    return torch.round(w / scale[:, None]).to(torch.int8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    t, k, n = case["tokens"], case["inner"], case["channels"]
    x = _normal(gen, (t, k), 1.0)
    x[:, :: max(1, k // 8)] *= 8  # a few channels are large, as activations have them
    state = {"case": case, "x": x.to(dtype)}
    if case["op"] == "int8":
        state["w"], state["w_scale"] = _weight_codes(gen, n, k)
        state["bias"] = _normal(gen, (n,), 1.0).to(dtype) if case["bias"] else None
    elif case["op"] == "int8_gated":
        for name in ("gate", "up"):
            state[name], state[name + "_scale"] = _weight_codes(gen, n, k)
    else:
        both = _normal(gen, (2, n, k), k**-0.5).to(dtype)
        state["gate"], state["up"] = both[0], both[1]
        if case["op"] == "train":
            state["grad"] = _normal(gen, (t, n), GRAD_SIZE).to(dtype)
    return state


def _act(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        below = 0.5 * torch.erfc(g * -math.sqrt(0.5))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-c * (g + 0.044715 * g * g * g)))
        return g * s, s + g * s * (1 - s) * c * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).to(g.dtype)


def _codes(x):
    """Rows as whole numbers up to 127 and their scales, in 32 bits."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True).clamp(min=LEAST_AMAX)
    return torch.round(MOST * x / amax), amax / MOST


def _run_plain(s):
    op, x = s["case"]["op"], s["x"]
    if op in ("int8", "int8_gated"):
        codes, scale = _codes(x)
        if op == "int8":
            y = torch.matmul(codes, s["w"].float().t()) * scale * s["w_scale"]
            return (y if s["bias"] is None else y + s["bias"].float()).to(x.dtype)
        g, u = (torch.matmul(codes, s[w].float().t()) * scale * s[w + "_scale"] for w in ("gate", "up"))
        return (_act(s["case"]["act"], g)[0] * u).to(x.dtype)
    xf, wg, wu = x.float(), s["gate"].float(), s["up"].float()
    g, u = torch.matmul(xf, wg.t()), torch.matmul(xf, wu.t())
    a, slope = _act(s["case"]["act"], g)
    h = (a * u).to(x.dtype)
    if op == "gated":
        return h
    grad = s["grad"].float()
    dg, du = grad * u * slope, grad * a
    dx = torch.matmul(dg, wg) + torch.matmul(du, wu)
    return h, dx.to(x.dtype), torch.matmul(dg.t(), xf).to(x.dtype), torch.matmul(du.t(), xf).to(x.dtype)


def _run_own(s):
    import cmpext3

    case, x = s["case"], s["x"]
    if case["op"] == "int8":
        return cmpext3.int8_linear(x, s["w"], s["w_scale"], s["bias"])
    if case["op"] == "int8_gated":
        return cmpext3.int8_gated_linear(x, s["gate"], s["up"], s["gate_scale"], s["up_scale"], activation=case["act"])
    if case["op"] == "gated":
        return cmpext3.gated_linear(x, s["gate"], s["up"], activation=case["act"])
    leaves = [t.detach().requires_grad_() for t in (x, s["gate"], s["up"])]
    h = cmpext3.gated_linear(*leaves, activation=case["act"])
    return (h.detach(), *torch.autograd.grad(h, leaves, s["grad"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    t, k, n = case["tokens"], case["inner"], case["channels"]
    if case["op"] == "int8":
        # activations, codes and scales of the weight, the bias, results
        return {"bytes": 2 * t * k + n * k + 4 * n + (2 * n if case["bias"] else 0) + 2 * t * n, "flops": 2 * t * k * n}
    if case["op"] == "int8_gated":
        return {"bytes": 2 * t * k + 2 * n * k + 8 * n + 2 * t * n, "flops": 4 * t * k * n}
    if case["op"] == "gated":
        return {"bytes": 2 * t * k + 4 * n * k + 2 * t * n, "flops": 4 * t * k * n}
    # the input, both weights and the gradient in; the result and the gradients of the input and both weights out
    return {"bytes": 4 * t * k + 8 * n * k + 4 * t * n, "flops": 12 * t * k * n}


def _exact_act(name, g):
    """Values and derivatives from the definitions, by the error function and tanh of 64 bits."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.special.erf(g / 2**0.5))
        return g * cdf, cdf + g * torch.exp(-(g**2) / 2) / (2 * math.pi) ** 0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        th = torch.tanh(c * (g + 0.044715 * g**3))
        return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th**2) * c * (1 + 0.134145 * g**2)
    return torch.where(g > 0, g, torch.zeros_like(g)), torch.where(g > 0, torch.ones_like(g), torch.zeros_like(g))


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"].startswith("int8"):
        # 127 times a 16-bit value over its row's largest is never so near to the middle of two codes, but on it
        # (half the largest is), that 32 and 64 bits could round it apart
        most = x.abs().max(dim=1, keepdim=True).values.clamp(min=LEAST_AMAX)
        held = torch.round(127 * x / most) * (most / 127)

        def product(name):
            return torch.nn.functional.linear(held, s[name].double() * s[name + "_scale"].double()[:, None])

        if case["op"] == "int8":
            y = product("w")
            return y if s["bias"] is None else y + s["bias"].double()
        return _exact_act(case["act"], product("gate"))[0] * product("up")
    wg, wu = s["gate"].double(), s["up"].double()
    g, u = x @ wg.T, x @ wu.T
    value, slope = _exact_act(case["act"], g)
    if case["op"] == "gated":
        return value * u
    grad = s["grad"].double()
    to_gate, to_up = grad * u * slope, grad * value
    return value * u, to_gate @ wg + to_up @ wu, to_gate.T @ x, to_up.T @ x
