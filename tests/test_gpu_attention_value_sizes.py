"""fp16 queries over 8-bit codes whose values are small or large, or differ in size from token to token:
within the bound of values of size one (attention_ref.attention), all of it relative to the values."""
import pytest
import torch

from tests import attention_ref as R
from tests.test_gpu_attention_edges import run

pytestmark = pytest.mark.gpu
F16, F8 = torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


FEW = [  # new tokens, lengths, heads, kv heads, dim: whole keys with four waves and eight, splits, 32 rows, heads of 256
    ([1, 1], [100, 1], 4, 1, 128), ([1, 1], [300, 250], 4, 2, 64), ([1, 1], [3000, 500], 8, 2, 128), ([4, 9], [3000, 500], 4, 2, 64),
    ([1], [2000], 4, 2, 256)]
TILE = [  # chunks: one group of waves, two, splits, heads of 256
    ([300, 90], [700, 500], 64, 16, 64), ([64], [3000], 8, 2, 128), ([300, 40], [9000, 400], 4, 2, 64), ([90, 30], [200, 64], 2, 1, 256),
    ([70, 1, 40], [150, 65, 40], 4, 2, 128)]
WAYS = FEW + TILE


def sizes(kind, tokens):
    """What the tokens' values are multiplied by."""
    if kind == "mixed":  # powers of two from 1 down to 2^-12, in any order
        return 2.0 ** -torch.randint(0, 13, (tokens,), generator=torch.Generator().manual_seed(tokens)).double()
    if kind == "rising":
        return torch.logspace(-4, 0, tokens, dtype=torch.float64)
    if kind == "falling":
        return torch.logspace(0, -4, tokens, dtype=torch.float64)
    return torch.full((tokens,), float(kind), dtype=torch.float64)


@pytest.mark.parametrize("new,lens,heads,kv_heads,dim", WAYS)
@pytest.mark.parametrize("kind", [1, 0.03, 1e-3, 1e-4, 12000, "mixed", "rising", "falling"])
@pytest.mark.parametrize("causal", [True, False])
def test_values_of_any_size(new, lens, heads, kv_heads, dim, kind, causal):
    def change(q, k, v):
        v[:] = (v.double() * sizes(kind, v.shape[0])[:, None, None]).clamp(-65504, 65504).to(v.dtype)

    got, want, tol = run(F16, F8, new, lens, heads, kv_heads, dim, change, True, causal=causal)
    assert want.abs().max() > 0
    R.check(got, want, tol)
