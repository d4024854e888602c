"""The example's attention layer (projections, norms and rotation, cache, attention) against the same
layer in 64 bits: a packed prompt, a chunk for some sequences, then single tokens."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

from tests import attention_ref as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXAMPLE = os.path.join(ROOT, "examples", "attention_layer.py")


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("attention_layer", EXAMPLE)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(layer, x):
    """A whole sequence through the layer in float64 (the tables as they are)."""
    h, hk, d = layer.heads, layer.kv_heads, layer.dim
    qkv = (x.double() @ layer.w_qkv.cpu().double().t()).unflatten(-1, (h + 2 * hk, d))
    pos = torch.arange(len(x))
    cos, sin = layer.cos.cpu(), layer.sin.cpu()
    q = R.rope(qkv[:, :h], layer.q_norm.cpu(), cos, sin, pos, 1e-6, False)[0] if len(x) else qkv[:, :h]
    k = R.rope(qkv[:, h : h + hk], layer.k_norm.cpu(), cos, sin, pos, 1e-6, False)[0]
    v = qkv[:, h + hk :]
    k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
    s = torch.einsum("nhd,mhd->hnm", q, k) * d**-0.5
    s = s.masked_fill(torch.ones(len(x), len(x), dtype=torch.bool).triu(1), float("-inf"))
    o = torch.einsum("hnm,mhd->nhd", s.softmax(-1), v)
    return o.flatten(1) @ layer.w_out.cpu().double().t()


# Relative 2-norm of the difference: each of the seven roundings to 16 bits on the way (qkv, q and k,
# weights, o, result, with the keys' and values' counted apart) is off by half a spacing at most, the
# norms keep q and k at size one, so scores (of size one) move by no more than a rounding of q and of k,
# and so do the weights; 8-bit codes are off by 2^-4 at most, 2^-5.8 as a root mean square over their
# range, in k (through the scores) and in v.
@pytest.mark.parametrize("dtype,held,most", [(torch.float16, None, 10 * 2.0**-11), (torch.bfloat16, None, 10 * 2.0**-8),
                                             (torch.bfloat16, torch.float8_e4m3fn, 10 * 2.0**-8 + 2 * 2.0**-4)])
def test_layer(example, dtype, held, most):
    width, heads, kv_heads, dim, page = 128, 8, 2, 64, 16
    layer = example.AttentionLayer(width, heads, kv_heads, dim, dtype, "cuda", max_positions=512)
    lens = [90, 1, 33]
    cache = example.PagedCache(40, page, kv_heads, dim, held or dtype, len(lens), "cuda")
    total = [n + 25 for n in lens]
    g = torch.Generator().manual_seed(1)
    xs = [torch.randn(n, width, generator=g).to(dtype) for n in total]
    want = [plain(layer, x) for x in xs]
    at = [0] * len(lens)
    for new in [lens, [20, 0, 17]] + [[1, 1, 1]] * 5:
        y = layer.forward(torch.cat([x[a : a + n] for x, a, n in zip(xs, at, new)]).cuda(), list(new), cache).cpu().double()
        ref = torch.cat([w[a : a + n] for w, a, n in zip(want, at, new)])
        off = ((y - ref).norm() / ref.norm()).item()
        assert off <= most, (new, off)
        at = [a + n for a, n in zip(at, new)]
    assert cache.lens == at


def test_script(example):
    r = subprocess.run([sys.executable, EXAMPLE, "--cache", "fp8", "--prompts", "300", "17", "--steps", "3", "--width", "256"],
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "relative difference" in r.stdout
