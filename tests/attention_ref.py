"""Plain 64-bit forms of the attention operators and what their kernels may be off.

Everything here runs on the CPU in float64, from the definitions:
  rotation   y = x / sqrt(mean(x^2) + eps) * w, pairs turned by cos and sin
  codes      e4m3(x * (448 / a)), a = max(max |x|, 2^-100) over the finite elements, scale a / 448
  attention  softmax(scale q k^T) v over the keys a query sees, zeros where it sees none
"""
import math

import torch

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24, torch.float64: 0.0}  # half a spacing at 1
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150, torch.float64: 0.0}  # half the least spacing


def rope(x, weight, cos, sin, positions, eps, interleaved):
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    half = c.shape[-1]
    out = y.clone()
    a = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    b = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    # what one element can be off: the fp32 steps of its pair (the sum of squares: one rounding
    # per element in the worst order, halved by the square root; root, quotient, two products;
    # then two products and a sum), and the last rounding
    size = y.abs()
    size[..., a] = y[..., a].abs() + y[..., b].abs()
    size[..., b] = size[..., a].clone()
    steps = (x.shape[-1] / 2 + 6 if weight is not None else 0) + 3
    tol = size * steps * 2.0**-24
    return out, tol + UNIT[x.dtype] * (out.abs() + tol) + TINY[x.dtype]


def quantise(x):
    """(codes, scales) of rows, with the two divisions and the product in float32 as defined."""
    f = x.float()
    f = torch.where(torch.isfinite(f), f, torch.full_like(f, math.nan))
    a = f.abs().nan_to_num(0.0).amax(-1, keepdim=True).clamp(min=2.0**-100)
    y = f * (torch.tensor(448.0) / a)
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), (a / 448.0).squeeze(-1)


def dequantise(codes, scales):
    return codes.double() * scales.double()[..., None]


def attention(q, k, v, scale, causal):
    """One sequence: q [n, heads, dim], k and v [m, kv_heads, dim] (float64 accepted for what a
    cache holds).  Returns the outputs and how far the kernels may be off each of them."""
    dtype = q.dtype
    n, heads, dim = q.shape
    m, kv_heads = k.shape[:2]
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    tol = torch.zeros_like(out)
    if n == 0 or m == 0:
        return out, tol
    g = heads // kv_heads
    qd = q.double().permute(1, 0, 2)
    kd = k.double().permute(1, 0, 2).repeat_interleave(g, 0)
    vd = v.double().permute(1, 0, 2).repeat_interleave(g, 0)
    seen = torch.ones(n, m, dtype=torch.bool)
    if causal:
        seen = torch.arange(m)[None] <= torch.arange(n)[:, None] + (m - n)
    s = torch.einsum("hnd,hmd->hnm", qd, kd) * scale
    size = torch.einsum("hnd,hmd->hnm", qd.abs(), kd.abs()) * scale
    s = s.masked_fill(~seen, -math.inf)
    some = seen.any(-1)[None, :, None]
    top = torch.where(some, s.amax(-1, keepdim=True), torch.zeros((), dtype=torch.float64))
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    w = torch.where(some, w / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(w))
    # a key's value where no weight is: not even NaN takes part
    vz = torch.where(seen.any(0)[None, :, None], vd, torch.zeros_like(vd))
    o = torch.einsum("hnm,hmd->hnd", w, vz)
    ov = torch.einsum("hnm,hmd->hnd", w, vz.abs())
    # scores: dim + 4 roundings of their products' sizes, the exponent's own error and that of its
    # argument (both scores, the maximum's too), in the weights and in their sum
    worst = (size * seen).amax(-1, keepdim=True)
    e = 2 * (2 * worst * (dim + 4) * 2.0**-24 + 2.0**-21) + (m + 4) * 2.0**-24
    e = torch.expm1(e)
    u = UNIT[dtype]
    # weights are rounded once (and, in 16 bits, to no less than half the least spacing, against
    # a largest weight of at least 1 in the kernel's units); the result once
    small = TINY[dtype] * m * vz.abs().amax((1, 2), keepdim=True) if m else 0.0
    t = ov * (u + 2.0**-24 * 4 + e) * (1 + u) + small + u * o.abs() + TINY[dtype]
    return o.permute(1, 0, 2), t.permute(1, 0, 2)


def starts(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def check(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    off = (got - want).abs() - tol
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))  # infinities and NaN
    bad = ~((off <= 0) | same)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
        f"{got[bad][0].item()} for {want[bad][0].item()} (may be off {tol[bad][0].item():.3g})"
