"""cmpext3.kv_cache_read with starts that fall, are negative or lie past the rows: every element is that of
a token of some sequence that holds the row, or zero."""
import pytest
import torch

import cmpext3

pytestmark = pytest.mark.gpu
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn

STARTS = [
    [0, 100, 200, 5, 300],           # row 10: the count of starts at or before it names the sequence from 100 on
    [40, 20, 30, 10, 50, 0, 60],
    [-50, -7, 3, -20, 90, 64],
    [0, 1 << 30, 64, 64, 1 << 30],
    [2**31 - 1, -(2**31), 2**31 - 1, 0, 128],
    [300, 200, 100, 0],
    [0] * 70 + [90, 50] + [10] * 60 + [128],  # more than one look at 64 starts
]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("starts", STARTS, ids=range(len(STARTS)))
@pytest.mark.parametrize("page", [4, 12])
@pytest.mark.parametrize("held,dim", [(BF16, 64), (F8, 64), (F8, 24)])
def test_starts_that_fall_stay_inside(starts, page, held, dim):
    """The table and the cache are the middles of larger tensors: what lies around them would show."""
    heads, pages, cols, total, batch = 2, 9, 7, 128, len(starts) - 1
    g = torch.Generator().manual_seed(page)
    around = torch.zeros(3 * batch, cols, dtype=torch.int32) + pages - 1  # a page of nobody's table
    around[batch : 2 * batch] = torch.randint(0, pages - 1, (batch, cols), generator=g)
    table = around[batch : 2 * batch]
    value = torch.arange(1, pages * page + 1).view(pages, page) % 120 + 1.0  # of a token, in all its elements
    value[pages - 1] = 127
    x = value[:, :, None, None].expand(pages, page, heads, dim)
    wide = torch.full((3 * pages, page, heads, dim), 125.0)
    wide[pages : 2 * pages] = x
    cache = wide.to(held).cuda()[pages : 2 * pages]
    scale = torch.ones(3 * pages, page, heads, device="cuda")[pages : 2 * pages] if held == F8 else None
    print(f"kv_cache_read starts {starts[:7]} page {page} {held} dim {dim}", flush=True)
    got = cmpext3.kv_cache_read(cache, cache, around.cuda()[batch : 2 * batch], torch.tensor(starts, dtype=torch.int32, device="cuda"), total,
                                dtype=BF16, k_scale=scale, v_scale=scale)
    held_value = cache[..., 0, 0].float().cpu()
    for out in got:
        out = out.float().cpu()
        for t in range(total):
            may = {0.0}
            for b in range(batch):
                if starts[b] <= t < starts[b + 1] and t - starts[b] < cols * page:
                    key = t - starts[b]
                    may.add(float(held_value[table[b, key // page], key % page]))
            assert set(out[t].unique().tolist()) <= may, t
