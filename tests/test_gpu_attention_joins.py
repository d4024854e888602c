"""Splits joined by a second launch outside graph capture (more row tiles than a stream has counters), tables
much wider than the lengths, and starts that fall."""
import math

import pytest
import torch

import cmpext3
from tests import attention_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def pages_of(held, pages, page, heads, dim):
    """(codes or elements, scales or None, what they stand for) of keys and values."""
    got = []
    for name in range(2):
        x = rand((pages, page, heads, dim), BF16, 70 + name)
        if held == F8:
            c, s = R.quantise(x)
            got.append((c, s, R.dequantise(c, s)))
        else:
            got.append((x, None, x))
    return got


def call(q, held, table, lens, cu):
    (k, ks, _), (v, vs, _) = held
    return cmpext3.paged_attention(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                   cu_seqlens_q=None if cu is None else cu.cuda(), **({} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda()))).cpu()


@pytest.mark.parametrize("held", [BF16, F8])
def test_more_row_tiles_than_counters(held):
    """600 sequences and 8 kv heads share a few pages; 4096 counters."""
    batch, heads, dim, page, pages, cols = 600, 8, 64, 64, 40, 48
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, cols * page + 1, (batch,), generator=g).tolist()
    table = torch.randint(0, pages, (batch, cols), generator=g).int()
    caches, q = pages_of(held, pages, page, heads, dim), rand((batch, heads, dim), BF16, 7)
    print(f"600 single tokens over {held}", flush=True)
    got = call(q, caches, table, lens, None)
    for i in range(0, batch, 7):
        k, v = (x[2][table[i].long()].flatten(0, 1)[: lens[i]] for x in caches)
        R.check(got[i : i + 1], *R.attention(q[i : i + 1], k, v, dim**-0.5, True), f"sequence {i} of {lens[i]}")


@pytest.mark.parametrize("held", [BF16, F8])
@pytest.mark.parametrize("cols", [70, 1024, 20000])
@pytest.mark.parametrize("new", [[1, 1, 1], [1] * 40, [5, 1, 9], [70, 130, 3], [300, 1, 64, 1, 1, 1, 1]])
def test_tables_wider_than_the_lengths(held, cols, new):
    """A table of one width for all lengths, as a captured graph has it; what lies past them names no page."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    lens = [(97 * i + 300) % 1100 + n for i, n in enumerate(new)]
    need = [-(-n // page) for n in lens]
    first = R.starts(need)
    table = torch.full((len(new), cols), -(1 << 30), dtype=torch.int32)
    for i in range(len(new)):
        table[i, : need[i]] = torch.arange(first[i], first[i + 1])
    caches, cq = pages_of(held, int(first[-1]), page, kv_heads, dim), R.starts(new)
    q = rand((sum(new), heads, dim), BF16, 9)
    print(f"table of {cols} columns, new {new[:5]}", flush=True)
    got = call(q, caches, table, lens, None if max(new) == 1 else cq)
    for i in range(len(new)):
        k, v = (x[2][first[i] : first[i + 1]].flatten(0, 1)[: lens[i]] for x in caches)
        R.check(got[cq[i] : cq[i + 1]], *R.attention(q[cq[i] : cq[i + 1]], k, v, dim**-0.5, True), f"sequence {i}")


@pytest.mark.parametrize("cu", [[0, 100, 64], [-5, 30, 64], [50, 10, 64], [64, 64, 1 << 30], [40, 20, 30, 10, 64], [2**31 - 1, -(2**31), 64]])
def test_starts_that_fall_give_numbers(cu):
    """No row from outside the tensors: those around them hold NaN."""
    wide = torch.full((3 * 64, 2, 64), math.nan, dtype=F16, device="cuda")
    wide[64:128] = rand((64, 2, 64), F16, 1).cuda()
    x, t = wide[64:128], torch.tensor(cu, dtype=torch.int32, device="cuda")
    for causal in (True, False):
        print(f"attention starts {cu} causal {causal}", flush=True)
        got = cmpext3.attention(x.clone(), x, x, t, t, causal=causal)
        fixed = torch.tensor([0, 30, 64] + [64] * (len(cu) - 3), dtype=torch.int32, device="cuda")
        assert cmpext3.attention(x.clone(), x, x, fixed, t, causal=causal).isfinite().all()
        assert got.shape == x.shape
