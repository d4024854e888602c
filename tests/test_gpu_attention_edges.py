"""Attention where a row's scores are no numbers, or where rows belong to no sequence: against the
definition in 64 bits, over all ways the keys are shared among waves, groups of waves and splits."""
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


def run(dtype, held, new, lens, heads, kv_heads, dim, change, paged, causal=True):
    """The output, and what it should be, of sequences of lens[i] keys whose last new[i] are queries."""
    q, k, v = (rand((n, h, dim), dtype, i) for i, (n, h) in enumerate(((sum(new), heads), (sum(lens), kv_heads), (sum(lens), kv_heads))))
    change(q, k, v)
    cq, ck = R.starts(new), R.starts(lens)
    print(f"{dtype} {held} new {new} lens {lens} heads {heads}/{kv_heads} dim {dim}", flush=True)
    if not paged:
        got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), cq.cuda(), ck.cuda(), causal=causal)
    else:
        page = 16
        need = [-(-n // page) for n in lens]
        first = R.starts(need)
        table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        caches, scales = [], []
        for x in (k, v):
            c = torch.full((int(first[-1]) * page, kv_heads, dim), math.nan, dtype=dtype)
            for i, n in enumerate(lens):
                table[i, : need[i]] = torch.arange(first[i], first[i + 1])
                c[first[i] * page : first[i] * page + n] = x[ck[i] : ck[i + 1]]
            c = c.unflatten(0, (-1, page))
            if held == F8:
                c, s = R.quantise(c)
                scales.append(s.cuda())
            caches.append(c.cuda())
        got = cmpext3.paged_attention(q.cuda(), *caches, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                      cu_seqlens_q=None if all(n == 1 for n in new) else cq.cuda(), causal=causal,
                                      **(dict(k_scale=scales[0], v_scale=scales[1]) if scales else {}))
        if held == F8:
            k, v = (R.dequantise(*R.quantise(x)) for x in (k, v))
    want = [R.attention(q[cq[i] : cq[i + 1]], k[ck[i] : ck[i + 1]], v[ck[i] : ck[i + 1]], dim**-0.5, causal) for i in range(len(new))]
    return got.cpu(), torch.cat([w for w, _ in want]), torch.cat([t for _, t in want])


# whole tiles; two groups of waves; splits; few rows in one range of keys and in splits; chunks
WAYS = [
    (False, [200, 70], [200, 70], 4, 2, 128), (False, [1000], [1000], 8, 2, 128), (False, [2361], [2361], 8, 2, 64),
    (False, [130], [700], 4, 1, 256), (True, [1, 1], [40, 1], 4, 1, 128), (True, [1, 1], [3000, 500], 8, 2, 128),
    (True, [4, 9], [3000, 500], 4, 2, 64), (True, [1], [2000], 4, 2, 256), (True, [64], [3000], 8, 2, 128), (True, [300, 40], [9000, 400], 4, 2, 64),
]


@pytest.mark.parametrize("paged,new,lens,heads,kv_heads,dim", WAYS)
@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (F16, F8)])
def test_a_query_of_nan_gives_nan(paged, new, lens, heads, kv_heads, dim, dtype, held):
    """All scores of such a row are NaN: so is the row, and no other one."""
    rows = sorted({0, sum(new) // 2, sum(new) - 1})

    def change(q, k, v):
        q[rows, 1] = math.nan

    got, want, tol = run(dtype, held, new, lens, heads, kv_heads, dim, change, paged)
    assert want[rows, 1].isnan().all()
    R.check(got, want, tol)


@pytest.mark.parametrize("paged,new,lens,heads,kv_heads,dim", WAYS)
@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (F16, F8)])
def test_scores_of_minus_infinity(paged, new, lens, heads, kv_heads, dim, dtype, held):
    """A row whose every visible score is -inf has no largest one: 0 / 0, not the zeros of a row
    that sees no key."""
    row = sum(new) - 1

    def change(q, k, v):
        k[..., 0] = -1 - k[..., 0].abs()
        q[row, 0] = 0
        q[row, 0, 0] = math.inf

    got, want, tol = run(dtype, held, new, lens, heads, kv_heads, dim, change, paged)
    assert want[row, 0].isnan().all()
    R.check(got, want, tol)


def test_one_key_of_minus_infinity_among_others():
    """Its weight is zero."""
    def change(q, k, v):
        q[..., 0] = q[..., 0].abs() + 0.25
        k[3, :, 0] = -math.inf

    got, want, _ = run(BF16, BF16, [150], [150], 2, 1, 64, change, False, causal=False)
    assert not got.isnan().any() and not want.isnan().any()
    without = lambda x: torch.cat([x[:3], x[4:]])  # noqa: E731
    q, k, v = rand((150, 2, 64), BF16, 0), rand((150, 1, 64), BF16, 1), rand((150, 1, 64), BF16, 2)
    change(q, k, v)
    R.check(got, *R.attention(q, without(k), without(v), 64**-0.5, False))


@pytest.mark.parametrize("paged,new,lens,before,after", [
    (False, [200, 0, 70], [200, 0, 70], 0, 9), (False, [5], [5], 3, 300), (False, [1000], [1000], 130, 1), (False, [2361], [2361], 1, 129),
    (True, [64, 3], [3000, 3], 0, 40), (True, [4, 1], [700, 100], 7, 5), (True, [300, 200], [9000, 400], 64, 200)])
def test_rows_of_no_sequence_are_zeros(paged, new, lens, before, after):
    """Rows before the first sequence and past the last one, as in a batch filled up to a fixed size."""
    heads, kv_heads, dim = 4, 2, 64
    total = before + sum(new) + after
    q = rand((total, heads, dim), BF16, 4)
    q[:before] = math.nan
    q[total - after :] = math.nan
    cq, ck = R.starts(new) + before, R.starts(lens)
    k, v = rand((sum(lens), kv_heads, dim), BF16, 5), rand((sum(lens), kv_heads, dim), BF16, 6)
    junk = torch.full((8, total, heads, dim), math.nan, dtype=BF16, device="cuda")  # memory the output may take
    del junk
    if paged:
        page = 4
        assert all(n % page == 0 for n in lens if n != 3)
        need = [-(-n // page) for n in lens]
        table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        first = R.starts(need)
        caches = []
        for x in (k, v):
            c = torch.zeros(int(first[-1]) * page, kv_heads, dim, dtype=BF16)
            for i, n in enumerate(lens):
                table[i, : need[i]] = torch.arange(first[i], first[i + 1])
                c[first[i] * page : first[i] * page + n] = x[ck[i] : ck[i + 1]]
            caches.append(c.unflatten(0, (-1, page)).cuda())
        got = cmpext3.paged_attention(q.cuda(), *caches, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), cu_seqlens_q=cq.cuda())
    else:
        got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), cq.cuda(), ck.cuda())
    got = got.cpu()
    assert not got[:before].any() and not got[total - after :].any()
    for i in range(len(new)):
        a, b, c, d = cq[i], cq[i + 1], ck[i], ck[i + 1]
        R.check(got[a:b], *R.attention(q[a:b], k[c:d], v[c:d], dim**-0.5, True), f"sequence {i}")


def test_no_sequence_at_all():
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.ones(5, 4, 64, dtype=F16, device="cuda")
    k = torch.ones(7, 2, 64, dtype=F16, device="cuda")
    assert not cmpext3.attention(q, k, k, none, none).any()
    cache = torch.ones(2, 16, 2, 64, dtype=F16, device="cuda")
    table = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    assert not cmpext3.paged_attention(q, cache, cache, table, none[:0], cu_seqlens_q=none).any()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("count,most,longest,held", [(6, 700, 1500, BF16), (20, 200, 600, BF16), (62, 120, 300, F8), (63, 120, 300, BF16)])
def test_many_tiles_of_uneven_sequences(causal, count, most, longest, held):
    """Enough row tiles that those with most keys go first (up to 62 sequences): every row once, with
    sequences of no token, of no key and of fewer keys than queries among them."""
    heads, dim, page = 64, 8, 16
    g = torch.Generator().manual_seed(count)
    new = torch.randint(40, most, (count,), generator=g).tolist()
    lens = [n + int(e) for n, e in zip(new, torch.randint(0, longest, (count,), generator=g))]
    new[1] = 0
    lens[2] = 0
    lens[3] = new[3] // 2
    need = [-(-n // page) for n in lens]
    first = R.starts(need)
    table = torch.full((count, max(need)), -1, dtype=torch.int32)
    for i in range(count):
        table[i, : need[i]] = torch.arange(first[i], first[i + 1])
    caches, plain, scales = [], [], []
    for name in range(2):
        x = rand((int(first[-1]) * page, heads, dim), BF16, 30 + name)
        if held == F8:
            c, s = R.quantise(x)
            plain.append(R.dequantise(c, s))
            scales.append(s.unflatten(0, (-1, page)).cuda())
            x = c
        else:
            plain.append(x)
        caches.append(x.unflatten(0, (-1, page)).cuda())
    cq = R.starts(new) + 5
    q = rand((int(cq[-1]) + 9, heads, dim), BF16, 29)
    junk = torch.full((4, *q.shape), math.nan, dtype=BF16, device="cuda")
    del junk
    print(f"new {new} lens {lens}", flush=True)
    got = cmpext3.paged_attention(q.cuda(), *caches, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), cu_seqlens_q=cq.cuda(),
                                  causal=causal, **(dict(k_scale=scales[0], v_scale=scales[1]) if scales else {})).cpu()
    assert not got[:5].any() and not got[cq[-1] :].any()
    for i in range(count):
        a, b, c = cq[i], cq[i + 1], first[i] * page
        R.check(got[a:b], *R.attention(q[a:b], plain[0][c : c + lens[i]], plain[1][c : c + lens[i]], dim**-0.5, causal), f"sequence {i}")


@pytest.mark.parametrize("dim", [24, 64, 128])
@pytest.mark.parametrize("dtype,held", [(BF16, F8), (F16, F8), (F16, F16)])
@pytest.mark.parametrize("new,lens", [([1, 1], [129, 250]), ([1] * 4, [512, 31, 257, 500]), ([1] * 9, [400, 1, 256, 130, 33, 512, 64, 255, 7]),
                                      ([1] * 32, [1000 - 31 * i for i in range(32)]), ([2, 3, 1, 1, 2], [300, 200, 77, 1, 129])])
def test_short_keys_stay_whole(dim, dtype, held, new, lens):
    """Few rows over keys that no split is worth: four waves, or eight for 8 bits, each with its share."""
    heads, kv_heads = (8, 4) if len(new) == 32 else (4, 2)
    got, want, tol = run(dtype, held, new, lens, heads, kv_heads, dim, lambda q, k, v: None, True)
    R.check(got, want, tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("held", [BF16, F8])
@pytest.mark.parametrize("new,lens,heads,kv_heads,dim", [
    ([300, 1, 200, 0, 3], [5000, 300, 4200, 7, 1], 8, 8, 64), ([200], [4500], 16, 8, 128), ([90, 300], [1500, 700], 2, 1, 256),
    ([70, 65, 129], [4200, 0, 60], 16, 16, 64)])
def test_splits_that_follow_from_the_lengths(causal, held, new, lens, heads, kv_heads, dim):
    got, want, tol = run(BF16, held, new, lens, heads, kv_heads, dim, lambda q, k, v: None, True, causal=causal)
    R.check(got, want, tol)


def test_splits_found_on_the_device_in_a_graph():
    """Joined by a second launch, which finds the same splits: the same result, with the lengths of each replay."""
    heads, kv_heads, dim, page, pages = 8, 8, 64, 64, 200
    q, k, v = (rand(s, BF16, i).cuda() for i, s in enumerate(((400, heads, dim), (pages, page, kv_heads, dim), (pages, page, kv_heads, dim))))
    table = torch.arange(160, dtype=torch.int32).view(2, 80).cuda()
    cu, lens = torch.tensor([0, 300, 400], dtype=torch.int32).cuda(), torch.tensor([5000, 4100], dtype=torch.int32).cuda()
    call = lambda: cmpext3.paged_attention(q, k, v, table, lens, cu_seqlens_q=cu)  # noqa: E731
    eager = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in (5000, 700, 4999, 5000):
        lens[0] = n
        want = call()
        torch.cuda.synchronize()
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
    assert torch.equal(want, eager)
