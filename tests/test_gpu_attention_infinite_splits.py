"""Infinite values at the keys of one split, the others' sums finite: joined, they stay infinite."""
import math

import pytest
import torch

from tests import attention_ref as R
from tests.test_gpu_attention_edges import run

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("paged,new,lens,heads,kv_heads,dim", [
    (False, [2361], [2361], 8, 2, 64), (False, [130], [5000], 4, 1, 256), (False, [9, 20], [5003, 700], 4, 2, 128), (True, [64], [3000], 8, 2, 128),
    (True, [300, 40], [9000, 400], 4, 2, 64), (True, [4, 9], [3000, 500], 4, 2, 64), (True, [5], [20000], 4, 2, 128)])
def test_infinite_values_in_the_last_split(dtype, paged, new, lens, heads, kv_heads, dim):
    """At the last two tokens, in two elements: seen by the last queries alone."""
    cq, ck, group = R.starts(new), R.starts(lens), heads // kv_heads
    at = [int(x) for x in ck[1:]]
    kept = {}

    def change(q, k, v):
        kept.update(q=q.clone(), k=k.clone())
        kept["v"] = v.clone()
        for n in at:
            kept["v"][n - 1, 0, 3] = kept["v"][n - 2, 1 % kv_heads, 5] = 0
            v[n - 1, 0, 3] = math.inf
            v[n - 2, 1 % kv_heads, 5] = -math.inf

    got = run(dtype, dtype, new, lens, heads, kv_heads, dim, change, paged)[0]
    for i in range(len(new)):
        a, b, c, d = cq[i], cq[i + 1], ck[i], ck[i + 1]
        want, tol = R.attention(kept["q"][a:b], kept["k"][c:d], kept["v"][c:d], dim**-0.5, True)
        want[-1:, :group, 3] = math.inf
        last = 1 % kv_heads
        want[-2:, last * group : (last + 1) * group, 5] = -math.inf
        R.check(got[a:b], want, tol, f"sequence {i}")
