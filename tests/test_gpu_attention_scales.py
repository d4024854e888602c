"""Scales of 8-bit keys and values that are no finite numbers: they take no part in rows that do not see
their token, and make the others what code * scale makes of them."""
import math

import pytest
import torch

import cmpext3
from tests import attention_ref as R

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# new tokens, keys, heads, kv heads, dim.  Few rows: whole, 32 rows, splits, heads of 256; tiles: two groups of
# waves, splits, one group, heads of 256
WAYS = [(6, 150, 4, 2, 128), (12, 150, 4, 2, 64), (5, 3000, 4, 2, 64), (3, 100, 2, 1, 256), (100, 150, 4, 2, 64), (64, 3000, 8, 2, 128),
        (300, 9000, 4, 2, 64), (400, 500, 64, 32, 64), (90, 200, 2, 1, 256)]


def inputs(dtype, new, keys, heads, kv_heads, dim):
    page = 32
    pages = -(-keys // page)
    g = torch.Generator().manual_seed(keys)
    q = torch.randn(new, heads, dim, generator=g).to(dtype)
    held = [R.quantise(torch.randn(pages, page, kv_heads, dim, generator=g).to(dtype)) for _ in range(2)]
    return q, [c for c, _ in held], [s for _, s in held]


def run(q, codes, scales, keys):
    table = torch.arange(codes[0].shape[0], dtype=torch.int32)[None].cuda()
    n, cu = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([keys], [0, len(q)]))
    return cmpext3.paged_attention(q.cuda(), *(c.cuda() for c in codes), table, n, cu, k_scale=scales[0].cuda(), v_scale=scales[1].cuda()).cpu()


@pytest.mark.parametrize("new,keys,heads,kv_heads,dim", WAYS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_scales_of_later_tokens_take_no_part(new, keys, heads, kv_heads, dim, dtype, value, which):
    q, codes, scales = inputs(dtype, new, keys, heads, kv_heads, dim)
    k, v = (R.dequantise(c, s).flatten(0, 1)[:keys] for c, s in zip(codes, scales))
    want, tol = R.attention(q, k, v, dim**-0.5, True)
    for name in which:
        scales["kv".index(name)].flatten(0, 1)[keys - 2 : keys] = value  # the last two queries' tokens
    got = run(q, codes, scales, keys)
    R.check(got[: new - 2], want[: new - 2], tol[: new - 2], "rows before the tokens")
    if which != "k":
        assert not got[new - 2 :].isfinite().any()
    elif math.isnan(value):
        assert got[new - 2 :].isnan().all()


@pytest.mark.parametrize("new,keys,heads,kv_heads,dim", WAYS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_values_scale_at_its_own_token(new, keys, heads, kv_heads, dim, dtype, value):
    """Rows that see the token get infinities of the codes' signs, NaN where the code is zero; one kv head
    of one token only, the others stay what they are."""
    q, codes, scales = inputs(dtype, new, keys, heads, kv_heads, dim)
    k, v = (R.dequantise(c, s).flatten(0, 1)[:keys] for c, s in zip(codes, scales))
    want, tol = R.attention(q, k, v, dim**-0.5, True)
    at, group = keys - 3, heads // kv_heads
    scales[1].flatten(0, 1)[at, 0] = value
    got = run(q, codes, scales, keys)
    sees = torch.zeros(new, heads, 1, dtype=torch.bool)
    sees[new - 3 :, :group] = True
    want = torch.where(sees, codes[1].flatten(0, 1)[at, 0].double() * value, want)
    R.check(got, want, tol)
