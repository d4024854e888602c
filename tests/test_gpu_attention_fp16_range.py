"""Weights of the second product in fp16, whose normal numbers end at 2^-14: one key far above the
rest must not push the others' weights out of that range (an attention sink: a key that all queries
look at, whose value is small)."""
import math

import pytest
import torch

from tests import attention_ref as R
from tests.test_gpu_attention_edges import run

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def bound(q, k, v, scale, held, least):
    """softmax(scale q k^T) v of one sequence whose last rows are the queries, and how far it may be off
    if weights are held to a factor of 1 +- `held`, or to `least` of the largest one."""
    n, heads, dim = q.shape
    m, kv_heads = k.shape[:2]
    g = heads // kv_heads
    qd, kd, vd = (x.double().transpose(0, 1) for x in (q, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)))
    seen = torch.arange(m)[None] <= torch.arange(n)[:, None] + (m - n)
    kt = kd.transpose(1, 2).contiguous()
    s = (qd @ kt * scale).masked_fill(~seen, -math.inf)
    size = ((qd.abs() @ kt.abs()) * scale * seen).amax(-1, keepdim=True)
    top = torch.exp(s - s.amax(-1, keepdim=True))
    total = top.sum(-1, keepdim=True)
    o, ov = top @ vd / total, top @ vd.abs() / total
    # dim + 4 roundings of a score's products, of the maximum's as well; the exponential's own and its argument's;
    # the sums over the keys; the numerator's and the denominator's
    e = torch.expm1(2 * (2 * size * (dim + 4) * 2.0**-24 + 2.0**-21) + (m + 4) * 2.0**-24)
    u = R.UNIT[q.dtype]
    tol = ov * (held + e) * (1 + u) + least * m * vd.abs().amax((1, 2), keepdim=True) / total + u * o.abs() + R.TINY[q.dtype]
    return o.transpose(0, 1), tol.transpose(0, 1)


# The tile kernel: a weight of 11 bits, and the largest one at 2^10 at least, so that half the least spacing,
# 2^-25, is 2^-35 of it.  The few-rows kernel: two parts of 11 bits, the largest weight at 2^15.
TILE, FEW = (2.0**-11, 2.0**-35), (2.0**-21, 2.0**-40)
WAYS = [  # as in test_gpu_attention_edges: whole tiles, two groups of waves, splits; few rows whole and in splits; chunks
    (False, [200, 70], [200, 70], 4, 2, 128, TILE), (False, [1000], [1000], 8, 2, 128, TILE), (False, [2361], [2361], 8, 2, 64, TILE),
    (False, [130], [700], 4, 1, 256, TILE), (True, [1, 1], [600, 100], 4, 1, 128, FEW), (True, [1, 1], [3000, 500], 8, 2, 128, FEW),
    (True, [4, 9], [3000, 500], 4, 2, 64, FEW), (True, [1], [2000], 4, 2, 256, FEW), (True, [64], [3000], 8, 2, 128, TILE),
    (True, [300, 40], [9000, 400], 4, 2, 64, TILE)]


@pytest.mark.parametrize("paged,new,lens,heads,kv_heads,dim,held", WAYS)
@pytest.mark.parametrize("above", [0, 8, 12, 16, 18])
@pytest.mark.parametrize("at_end", [False, True])
def test_a_key_far_above_the_rest(paged, new, lens, heads, kv_heads, dim, held, above, at_end):
    """Its score is `above` (natural units) over the others', its value zero; the values are large enough
    that the result itself is a normal number."""
    ck, cq = R.starts(lens), R.starts(new)
    inputs = {}

    def change(q, k, v):
        v *= 256
        q[..., 0] = 4
        k[..., 0] = 0
        # seen by every query of its sequence
        at = [int(ck[i]) + (lens[i] - new[i] if at_end else 0) for i in range(len(lens))]
        k[at] = 0
        k[at, :, 0] = above * dim**0.5 / 4
        v[at] = 0
        inputs.update(q=q.clone(), k=k.clone(), v=v.clone())

    got = run(F16, F16, new, lens, heads, kv_heads, dim, change, paged)[0]
    for i in range(len(lens)):
        a, b, c, d = cq[i], cq[i + 1], ck[i], ck[i + 1]
        R.check(got[a:b], *bound(inputs["q"][a:b], inputs["k"][c:d], inputs["v"][c:d], dim**-0.5, *held), f"sequence {i}")
