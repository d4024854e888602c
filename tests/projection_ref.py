"""Plain 64-bit forms of the feed-forward operators and what their kernels may be off.

  codes     round(127 x / a), a = max(max |x|, 2^-100) of the row, scale a / 127
  gated     act(x Wg^T) * (x Wu^T)
  backward  dg = grad u act'(g), du = grad act(g); dx = dg Wg + du Wu; dWg = dg^T x; dWu = du^T x

Bounds count roundings.  A sum of K products in fp32 is off by at most K 2^-23 times the sum of
their sizes (one rounding a term, truncated at worst).
"""
import math

import torch

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a spacing, relative
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}  # half the least spacing
F32 = 2.0**-24


def codes(x):
    """(codes, scales) as float64, whatever device x is on; rows that are not finite: 0 and NaN."""
    d = x.double()
    a = d.abs().amax(-1, keepdim=True) if x.shape[-1] else d.new_zeros((*x.shape[:-1], 1))
    fine = torch.isfinite(a)
    a = torch.where(fine, a, torch.ones_like(a)).clamp(min=2.0**-100)
    q = torch.round(127 * d / a)
    q = torch.where(fine, q, torch.zeros_like(q))
    scale = torch.where(fine, a / 127, torch.full_like(a, math.nan))
    return q, scale.squeeze(-1)


def act(name, g):
    """Value, derivative, and a bound of the second derivative's size (relu: none)."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g), 0.5
    if name == "gelu":
        below = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * below, below + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 0.8
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (g + 0.044715 * g**3))
        slope = 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 3 * 0.044715 * g * g)
        return 0.5 * g * (1 + th), slope, 0.9
    return g.clamp(min=0), (g > 0).double(), 0.0


def act_error(name, g, value, e):
    """How far act may be off where g is off by e: its slope is at most 1.13, and its own arithmetic
    (a few roundings; those of the exponent count |g| to |g|^3 times) is relative to the value."""
    b = g.abs().clamp(max=40)
    return 1.13 * e + value.abs() * (1 + b + b * b + 0.1 * b**3) * 2.0**-21


def rounded(y, tol, dtype):
    return tol + UNIT[dtype] * (y.abs() + tol) + TINY[dtype]


def products(x, w):
    """x w^T in 64 bits and the bound of its sum in fp32."""
    x, w = x.double(), w.double()
    return x @ w.t(), (x.abs() @ w.abs().t()) * x.shape[-1] * 2 * F32


def gated(x, wg, wu, name):
    """(result, bound) for 16-bit inputs [M, K], [N, K]."""
    g, eg = products(x, wg)
    u, eu = products(x, wu)
    a = act(name, g)[0]
    ea = act_error(name, g, a, eg)
    y = a * u
    tol = ea * u.abs() + a.abs() * eu + ea * eu + F32 * y.abs()
    return y, rounded(y, tol, x.dtype)


def gated_backward(x, wg, wu, grad, name):
    """((dx, bound), (dWg, bound), (dWu, bound)): dg and du are held in the inputs' type."""
    t = x.dtype
    g, eg = products(x, wg)
    u, eu = products(x, wu)
    value, slope, bend = act(name, g)
    ea = act_error(name, g, value, eg)
    es = bend * eg + (1 + g.abs().clamp(max=40)) ** 2 * 2.0**-21
    if name == "relu":
        es = es + (g.abs() <= eg).double()  # on which side of 0 it falls is open
    d = grad.double()
    dg, du = d * u * slope, d * value
    edg = d.abs() * ((u.abs() + eu) * es + eu * slope.abs()) + 3 * F32 * dg.abs()
    edu = d.abs() * ea + 2 * F32 * du.abs()
    edg, edu = rounded(dg, edg, t), rounded(du, edu, t)

    def sums(pairs):
        y = sum(a @ b for a, _, b in pairs)
        k = sum(a.shape[1] for a, _, _ in pairs)
        tol = sum(e @ b.abs() + (a.abs() + e) @ b.abs() * (k * 2 * F32) for a, e, b in pairs)
        return y, rounded(y, tol, t)

    xd, wgd, wud = x.double(), wg.double(), wu.double()
    return sums([(dg, edg, wgd), (du, edu, wud)]), sums([(dg.t(), edg.t(), xd)]), sums([(du.t(), edu.t(), xd)])


def int8_product(xq, xs, wq, ws):
    """(value, bound) before the last rounding: integer sums are exact, then they become a float and
    are multiplied twice."""
    y = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    return y, y.abs() * 3.01 * F32


def int8_linear(xq, xs, wq, ws, bias, dtype):
    y, tol = int8_product(xq, xs, wq, ws)
    if bias is not None:
        y = y + bias.double()
        tol = tol + (y.abs() + tol) * F32
    return y, rounded(y, tol, dtype)


def int8_gated(xq, xs, wg, gs, wu, us, name, dtype):
    g, eg = int8_product(xq, xs, wg, gs)
    u, eu = int8_product(xq, xs, wu, us)
    a = act(name, g)[0]
    ea = act_error(name, g, a, eg)
    y = a * u
    return y, rounded(y, ea * u.abs() + a.abs() * eu + ea * eu + F32 * y.abs(), dtype)


def check(out, want, what=""):
    """Every element within its bound; NaN where NaN is expected and nowhere else."""
    y, tol = want
    out = out.double()
    y, tol = y.to(out.device).reshape(out.shape), tol.to(out.device).reshape(out.shape)
    nan = torch.isnan(y)
    assert torch.equal(torch.isnan(out), nan), f"{what}: NaN at other places"
    off = torch.where(nan | (out == y), torch.zeros_like(y), (out - y).abs())
    tol = torch.where(nan, torch.ones_like(tol), tol)
    worst = (off / tol).max().item() if out.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound at {int((off / tol).argmax())} of {tuple(out.shape)}"
    return worst
