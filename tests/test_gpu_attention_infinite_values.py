"""Values of infinity and NaN that rows of few queries see, over pages: they reach the rows that see them,
in their elements, as in a packed prompt (test_gpu_attention.test_infinite_values_that_are_seen)."""
import math

import pytest
import torch

from tests import attention_ref as R
from tests.test_gpu_attention_edges import run
from tests.test_gpu_attention_scales import inputs, run as run_scales

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("held", ["same", "codes"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens,heads,kv_heads,dim", [([1, 1], [150, 90], 4, 2, 64), ([1, 1], [3000, 500], 8, 2, 128), ([4, 9], [3000, 500], 4, 2, 64),
                                                         ([1, 3], [100, 2000], 4, 2, 256), ([70, 40], [200, 100], 4, 2, 64)])
def test_infinite_values_that_are_seen(dtype, held, causal, new, lens, heads, kv_heads, dim):
    """The same elements of the same rows as by the definition; codes hold NaN for all of them."""
    first, second = 0, lens[0]  # the first tokens of the two sequences
    kept = {}

    def change(q, k, v):
        v[first + 40, 0, 3] = math.inf
        v[first + 41, 0, 5] = -math.inf
        v[first + 42, 1, 7] = math.nan
        v[first + 10, 1, 9], v[first + 60, 1, 9] = math.inf, -math.inf  # both: NaN
        v[second + 20, 1, 0], v[second + 22, 1, 0] = math.inf, math.inf
        v[second + lens[1] - 1, 0, 1] = math.inf  # the last token: with `causal` the last query alone sees it
        if held == "codes":
            v[:] = torch.where(v.isfinite(), v, torch.full_like(v, math.nan))
        kept.update(q=q.clone(), k=k.clone(), v=v.clone())

    got = run(dtype, dtype if held == "same" else F8, new, lens, heads, kv_heads, dim, change, True, causal=causal)[0]
    q, k, v = kept["q"], kept["k"], kept["v"]
    if held == "codes":
        k, v = (R.dequantise(*R.quantise(x)) for x in (k, v))
    cq, ck, group = R.starts(new), R.starts(lens), heads // kv_heads
    for i in range(2):
        x = v[ck[i] : ck[i + 1]].double()
        want, tol = R.attention(q[cq[i] : cq[i + 1]], k[ck[i] : ck[i + 1]], x.nan_to_num(0.0, 0.0, 0.0), dim**-0.5, causal)
        # each value that is not finite, to the rows that see it
        for t, h, e in (~x.isfinite()).nonzero().tolist():
            rows = slice(max(0, t - (lens[i] - new[i])), None) if causal else slice(None)
            want[rows, h * group : (h + 1) * group, e] += x[t, h, e]
        assert not want.isfinite().all()
        R.check(got[cq[i] : cq[i + 1]], want, tol, f"sequence {i}")


@pytest.mark.parametrize("new,keys,heads,kv_heads,dim", [(1, 150, 4, 2, 128), (1, 300, 4, 2, 64), (6, 150, 4, 2, 128), (12, 150, 4, 2, 64), (5, 3000, 4, 2, 64),
                                                         (3, 100, 2, 1, 256), (100, 150, 4, 2, 64), (64, 3000, 8, 2, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [3, 47])
def test_a_scale_that_is_seen_by_all(new, keys, heads, kv_heads, dim, dtype, value, at):
    """Of one value: infinities of its codes' signs, NaN where the code is zero."""
    q, codes, scales = inputs(dtype, new, keys, heads, kv_heads, dim)
    k, v = (R.dequantise(c, s).flatten(0, 1)[:keys] for c, s in zip(codes, scales))
    want, tol = R.attention(q, k, v, dim**-0.5, True)
    scales[1].flatten(0, 1)[at, 0] = value
    want[:, : heads // kv_heads] = codes[1].flatten(0, 1)[at, 0].double() * value
    R.check(run_scales(q, codes, scales, keys), want, tol)
