"""Attention over a paged cache (cmpext3.paged_attention) against its definition in 64 bits: one
token for each sequence and chunks, 16 bits and 8, pages of any size, splits of the keys."""
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


def paged(dtype, held, new, lens, heads, kv_heads, dim, page, causal=True, scale=None, seed=0, wide=0, head_major=False,
          uniform=None, spoil=False):
    """new: queries of each sequence; lens: its keys.  Pages nobody names hold NaN, and with
    `spoil` so do the places of the last page past the length."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(need + [1]) + wide), -1, dtype=torch.int32)
    shape = (pages, kv_heads, page, dim) if head_major else (pages, page, kv_heads, dim)
    caches, scales, plain = [], [], []
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    for name in range(2):
        x = rand((pages, page, kv_heads, dim), dtype, seed + 10 + name)
        if spoil:
            for i, n in enumerate(lens):
                if n % page:
                    x[table[i, n // page], n % page :] = float("nan")
        x[order[at:].long()] = float("nan")
        if held == F8:
            codes, s = R.quantise(x)
            plain.append(R.dequantise(codes, s))
            x = codes
            s = s.transpose(1, 2).contiguous().cuda().transpose(1, 2) if head_major else s.cuda()
            scales.append(s)
        else:
            plain.append(x)
            scales.append(None)
        x = x.cuda()
        caches.append(x.transpose(1, 2).contiguous().transpose(1, 2) if head_major else x)
    q = rand((sum(new), heads, dim), dtype, seed + 1)
    cu = R.starts(new)
    one = uniform if uniform is not None else all(n == 1 for n in new)
    print(f"paged_attention {dtype} {held} new {new[:6]} lens {lens[:6]} heads {heads}/{kv_heads} dim {dim} page {page}", flush=True)
    got = cmpext3.paged_attention(q.cuda(), *caches, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                                  cu_seqlens_q=None if one else cu.cuda(), k_scale=scales[0], v_scale=scales[1], causal=causal,
                                  scale=scale).cpu()
    for i, n in enumerate(lens):
        k, v = (x[table[i, : need[i]].long()].flatten(0, 1)[:n] for x in plain)
        want, tol = R.attention(q[cu[i] : cu[i + 1]], k, v, scale or dim**-0.5, causal)
        R.check(got[cu[i] : cu[i + 1]], want, tol, f"sequence {i} of {n}")
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [8, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 9], [70, 130, 3]])
def test_head_sizes(dtype, quantised, dim, new):
    paged(dtype, F8 if quantised else dtype, new, [100, 33, 260], 4, 2, dim, 16, seed=dim)


@pytest.mark.parametrize("page", [1, 7, 16, 24, 32, 48, 64, 100, 256])
@pytest.mark.parametrize("held", [BF16, F8])
def test_page_sizes(page, held):
    paged(BF16, held, [1, 1, 1], [200, 1, 131], 4, 2, 64, page, spoil=True)
    paged(BF16, held, [90, 1, 40], [200, 1, 131], 4, 2, 128, page, spoil=True)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (8, 8), (40, 8), (32, 1), (24, 2), (64, 1)])
@pytest.mark.parametrize("held", [F16, F8])
def test_groups(heads, kv_heads, held):
    paged(F16, held, [1, 1, 1], [70, 5, 300], heads, kv_heads, 128, 32, seed=heads)
    paged(F16, held, [3, 6, 2], [70, 6, 300], heads, kv_heads, 64, 32, seed=heads)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_lengths(n):
    paged(BF16, BF16, [1, 1], [n, max(1, n - 1)], 4, 1, 128, 16, seed=n, spoil=True)
    paged(F16, F8, [min(n, 40), 1], [n, n], 4, 1, 64, 16, seed=n, spoil=True)


@pytest.mark.parametrize("held", [BF16, F8])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_sequences_are_split(held, dim):
    paged(BF16, held, [1, 1, 1], [5000, 17, 2049], 8, 2, dim, 64, seed=1, spoil=True)
    paged(BF16, held, [40, 3, 70], [5000, 17, 2049], 8, 2, dim, 64, seed=2, spoil=True)


@pytest.mark.parametrize("held", [BF16, F8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens", [([64], [3000]), ([70, 1, 33, 9, 50], [700, 1, 1500, 40, 64]), ([100] * 6, [100, 1900, 130, 64, 65, 700]),
                                      ([40], [9000]), ([300, 200], [9000, 400])])
def test_chunks_share_their_keys(held, dim, new, lens):
    """Chunks over few row tiles: groups of waves and splits of a tile's keys, joined in both ways."""
    paged(BF16, held, new, lens, 4, 2, dim, 64, seed=sum(lens), spoil=True)
    paged(BF16, held, new, lens, 4, 2, dim, 64, seed=sum(lens), spoil=True, causal=False)


def test_a_long_cache_past_32_bits():
    """Chunks and single tokens over pages whose elements lie past 2^32 bytes, both kinds of cache."""
    page, heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * heads * dim * 2)
    k = torch.empty(pages, page, heads, dim, dtype=F16, device="cuda")
    k8, v8 = (torch.empty(2 * pages, page, heads, dim, dtype=F8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(2 * pages, page, heads, device="cuda") for _ in range(2))
    x, y = rand((2 * page, heads, dim), F16, 3), rand((2 * page, heads, dim), F16, 4)
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32)
    table8 = torch.tensor([[2 * pages - 2, 2 * pages - 1]], dtype=torch.int32)
    slots = (table[0].long()[:, None] * page + torch.arange(page)).flatten().cuda()
    slots8 = (table8[0].long()[:, None] * page + torch.arange(page)).flatten().cuda()
    cmpext3.kv_cache_write(x.cuda(), x.cuda(), k, k, slots)
    cmpext3.kv_cache_write(x.cuda(), y.cuda(), k8, v8, slots8, ks, vs)
    n = torch.tensor([2 * page - 3], dtype=torch.int32, device="cuda")
    for new in (1, 90):
        q = rand((new, heads, dim), F16, new)
        cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        got = cmpext3.paged_attention(q.cuda(), k, k, table.cuda(), n, cu)
        R.check(got, *R.attention(q, x[:-3], x[:-3], dim**-0.5, True))
        got = cmpext3.paged_attention(q.cuda(), k8, v8, table8.cuda(), n, cu, k_scale=ks, v_scale=vs)
        R.check(got, *R.attention(q, R.dequantise(*R.quantise(x))[:-3], R.dequantise(*R.quantise(y))[:-3], dim**-0.5, True))


def test_empty_sequences():
    got = paged(BF16, BF16, [1, 1, 1], [0, 5, 0], 4, 2, 64, 16)
    assert not got[0].any() and not got[2].any() and got[1].any()
    paged(F16, F8, [0, 4, 0, 3, 0], [0, 9, 7, 3, 0], 4, 2, 64, 16)
    # more queries than keys: the first ones see none
    assert not paged(BF16, F8, [50, 9], [3, 2], 4, 2, 128, 16)[:47].any()
    cache = torch.zeros(2, 4, 2, 64, dtype=F16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    none = cmpext3.paged_attention(torch.zeros(0, 4, 64, dtype=F16, device="cuda"), cache, cache, torch.zeros(0, 3, **i32), torch.zeros(0, **i32))
    assert none.shape == (0, 4, 64)
    assert not cmpext3.paged_attention(torch.ones(2, 4, 64, dtype=F16, device="cuda"), cache, cache, torch.zeros(2, 0, **i32),
                                       torch.zeros(2, **i32)).any()


@pytest.mark.parametrize("held", [F16, F8])
def test_layouts_and_tables(held):
    paged(F16, held, [1, 1], [90, 40], 4, 2, 128, 32, wide=40, head_major=True)   # a table wider than the lengths
    paged(F16, held, [30, 9], [90, 40], 4, 2, 128, 32, wide=3, head_major=True)
    paged(F16, held, [9, 9], [90, 40], 4, 2, 64, 32, causal=False)
    paged(F16, held, [1, 1], [90, 40], 4, 2, 64, 32, scale=0.7, uniform=False)
    paged(F16, held, [1, 1], [900, 400], 4, 2, 64, 32, scale=3.0)


def test_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(1, 200, (130,), generator=g).tolist()
    paged(BF16, F8, [1] * 130, lens, 4, 1, 64, 16, uniform=False)
    paged(BF16, BF16, [min(n, 1 + i % 7) for i, n in enumerate(lens)], lens, 4, 1, 64, 16)


@pytest.mark.parametrize("new", [6, 100])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_later_tokens_take_no_part(new, dim, value):
    """Keys and values that are not finite at the places of later new tokens."""
    page, n = 32, 150
    cache = rand((5, page, 2, dim), BF16, 1)
    q = rand((new, 4, dim), BF16, 2)
    table, i32 = torch.arange(5, dtype=torch.int32)[None], dict(dtype=torch.int32, device="cuda")
    run = lambda c: cmpext3.paged_attention(q.cuda(), c.cuda(), c.cuda(), table.cuda(), torch.tensor([n], **i32), torch.tensor([0, new], **i32)).cpu()  # noqa: E731
    clean = run(cache)
    spoilt = cache.clone()
    spoilt.flatten(0, 1)[n - 3 : n] = value
    assert torch.equal(run(spoilt)[: new - 3], clean[: new - 3])
    assert not run(spoilt)[new - 3 :].isfinite().all()


def test_bad_tables_stay_inside():
    """Page numbers outside the cache, and lengths past the table: nothing outside is read."""
    cache = rand((3, 8, 2, 64), F16, 1).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1 << 30], [-1, 2]], **i32)
    for rows in (1, 40):
        q = rand((2 * rows, 4, 64), F16, 2).cuda()
        got = cmpext3.paged_attention(q, cache, cache, table, torch.tensor([1 << 30, 16], **i32), torch.tensor([0, rows, 2 * rows], **i32))
        assert got.isfinite().all()
        got = cmpext3.paged_attention(q, cache, cache, table, torch.tensor([-7, 16], **i32), torch.tensor([0, rows, 2 * rows], **i32))
        assert not got[:rows].any()


def test_graph_replays_match_eager():
    """The whole path (write, attend) in a captured graph, with new lengths between the replays."""
    i32 = dict(dtype=torch.int32, device="cuda")
    kc, vc = (torch.zeros(40, 64, 2, 128, dtype=F8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(40, 64, 2, device="cuda") for _ in range(2))
    table = torch.arange(40, **i32).view(2, 20)
    k, v = (rand((2, 2, 128), BF16, s).cuda() for s in (1, 2))
    q = rand((2, 8, 128), BF16, 3).cuda()
    lens, slots = torch.tensor([1, 1], **i32), torch.tensor([0, 20 * 64], device="cuda")

    def step():
        cmpext3.kv_cache_write(k, v, kc, vc, slots, ks, vs)
        return cmpext3.paged_attention(q, kc, vc, table, lens, k_scale=ks, v_scale=vs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for t, s in ((k, 20), (v, 30), (q, 40)):
            t.copy_(rand(t.shape, BF16, s + i))
        lens.fill_(2 + 300 * i)
        slots.copy_(torch.tensor([1 + 300 * i, 20 * 64 + 1 + 300 * i]))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
