"""cmpext3.rope_table against its formulas, term by term in Python floats."""
import math

import pytest
import torch

import cmpext3


def check(cos, sin, freq, size=1.0):
    assert cos.dtype == sin.dtype == torch.float32 and cos.shape == sin.shape
    for p in (0, 1, 7, cos.shape[0] - 1):
        for i, f in enumerate(freq):
            # one rounding of a product of at most p * f, in float64, then of the result to fp32
            tol = 2.0**-24 + p * f * 2.0**-50
            assert abs(float(cos[p, i]) - size * math.cos(p * f)) <= size * tol
            assert abs(float(sin[p, i]) - size * math.sin(p * f)) <= size * tol


@pytest.mark.parametrize("dim", [2, 20, 64, 128])
def test_plain_and_linear(dim):
    freq = [10000.0 ** (-2 * i / dim) for i in range(dim // 2)]
    check(*cmpext3.rope_table(500, dim), freq)
    check(*cmpext3.rope_table(500, dim, 500000.0), [500000.0 ** (-2 * i / dim) for i in range(dim // 2)])
    check(*cmpext3.rope_table(500, dim, scaling="linear", factor=4.0), [f / 4 for f in freq])


def test_ntk():
    dim, factor = 64, 8.0
    cos, sin = cmpext3.rope_table(300, dim, scaling="ntk", factor=factor)
    base = 10000.0 * factor ** (dim / (dim - 2))
    freq = [base ** (-2 * i / dim) for i in range(dim // 2)]
    check(cos, sin, freq)
    assert freq[0] == 1.0 and math.isclose(freq[-1], 10000.0 ** (-2 * 31 / 64) / factor, rel_tol=1e-12)


def test_yarn():
    dim, factor, original = 128, 16.0, 4096
    plain = [10000.0 ** (-2 * i / dim) for i in range(dim // 2)]
    freq = []
    for f in plain:
        kept = min(1.0, max(0.0, (original * f / (2 * math.pi) - 1) / (32 - 1)))
        freq.append(f * kept + f / factor * (1 - kept))
    assert freq[0] == plain[0] and freq[-1] == plain[-1] / factor
    check(*cmpext3.rope_table(300, dim, scaling="yarn", factor=factor, original_positions=original), freq,
          0.1 * math.log(factor) + 1)
    check(*cmpext3.rope_table(300, dim, scaling="yarn", factor=factor, original_positions=original, attention_factor=1.0), freq)


def test_empty_and_refusals():
    assert cmpext3.rope_table(0, 64)[0].shape == (0, 32)
    assert cmpext3.rope_table(5, 0)[0].shape == (5, 0)
    for args, kw in (((-1, 64), {}), ((5, 63), {}), ((5, -2), {}), ((5, 64, 0.0), {}), ((5, 64, math.inf), {}),
                     ((5, 64), dict(factor=2.0)), ((5, 64), dict(scaling="linear", factor=0.5)), ((5, 64), dict(scaling="other")),
                     ((5, 64), dict(scaling="yarn", factor=2.0)),
                     ((5, 64), dict(scaling="yarn", factor=2.0, original_positions=64, beta_fast=1.0, beta_slow=2.0))):
        with pytest.raises(ValueError):
            cmpext3.rope_table(*args, **kw)
