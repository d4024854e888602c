"""Attention over whole prompts (cmpext3.attention) against its definition in 64 bits on the CPU,
each element within what the kernels' roundings allow (attention_ref.attention)."""
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


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def packed(dtype, lens_q, lens_k, heads, kv_heads, dim, causal, scale=None, seed=0, change=None):
    q = rand((sum(lens_q), heads, dim), dtype, seed)
    k = rand((sum(lens_k), kv_heads, dim), dtype, seed + 1)
    v = rand((sum(lens_k), kv_heads, dim), dtype, seed + 2)
    if change:
        change(q, k, v)
    cq, ck = R.starts(lens_q), R.starts(lens_k)
    print(f"attention {dtype} q{lens_q} k{lens_k} heads {heads}/{kv_heads} dim {dim} causal {causal}", flush=True)
    got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), cq.cuda(), ck.cuda(), causal=causal, scale=scale).cpu()
    for i in range(len(lens_q)):
        a, b, c, d = cq[i], cq[i + 1], ck[i], ck[i + 1]
        want, tol = R.attention(q[a:b], k[c:d], v[c:d], scale or dim**-0.5, causal)
        R.check(got[a:b], want, tol, f"sequence {i}")
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_head_sizes(dtype, dim, causal):
    packed(dtype, [1, 77, 130, 64], [1, 77, 130, 64], 4, 2, dim, causal, seed=dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (4, 1), (10, 2), (7, 1), (40, 8), (64, 1)])
def test_groups(heads, kv_heads):
    packed(BF16, [33, 5, 129], [33, 5, 129], heads, kv_heads, 64, True, seed=heads)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500])
def test_lengths(n):
    packed(F16, [n], [n], 2, 2, 128, True, seed=n)
    packed(BF16, [n, 3, n], [n, 3, n], 4, 2, 64, True, seed=n)


@pytest.mark.parametrize("causal", [True, False])
def test_more_keys_than_queries_and_fewer(causal):
    """Queries end where the keys end; queries before the first key see none and get zeros."""
    got = packed(BF16, [5, 100, 64, 7, 3], [70, 300, 1, 0, 2], 4, 2, 128, causal, seed=3)
    at = R.starts([5, 100, 64, 7, 3])
    if causal:
        assert not got[at[2] : at[2] + 63].any()          # 64 queries, one key
        assert not got[at[4] : at[4] + 1].any()           # 3 queries, two keys
    assert not got[at[3] : at[4]].any()                   # no keys at all


def test_empty_sequences():
    packed(F16, [0, 17, 0, 0, 200, 0], [0, 17, 9, 0, 200, 0], 2, 1, 64, True)
    q = torch.zeros(0, 4, 64, dtype=F16, device="cuda")
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert cmpext3.attention(q, q[:, :2], q[:, :2], none, none).shape == (0, 4, 64)
    assert cmpext3.attention(q[None][:0], q[None][:0], q[None][:0]).shape == (0, 0, 4, 64)
    k = torch.zeros(5, 0, 2, 64, dtype=F16, device="cuda")
    assert not cmpext3.attention(torch.ones(5, 3, 4, 64, dtype=F16, device="cuda"), k, k).any()


def test_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 40, (150,), generator=g).tolist()
    packed(BF16, lens, lens, 2, 1, 64, True)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strided_operands(dtype):
    """Parts of one qkv product, [batch, heads, tokens, dim] memory, and rows that need a copy."""
    b, n, h, hk, d = 2, 90, 6, 2, 64
    qkv = rand((b, n, (h + 2 * hk) * d), dtype, 5).cuda()
    q, k, v = (x.unflatten(-1, (-1, d)) for x in qkv.split([h * d, hk * d, hk * d], -1))
    want = [R.attention(q[i].cpu(), k[i].cpu(), v[i].cpu(), d**-0.5, True) for i in range(b)]

    def same(got):
        for i in range(b):
            R.check(got[i], *want[i])

    same(cmpext3.attention(q, k, v))
    same(cmpext3.attention(*(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))))
    odd = torch.empty(b, n, h, d + 1, dtype=dtype, device="cuda")[..., 1:]  # misaligned heads
    same(cmpext3.attention(odd.copy_(q), k, v))
    same(cmpext3.attention(q, k.transpose(2, 3).contiguous().transpose(2, 3), v))
    flat = [x.flatten(0, 1) for x in (q, k, v)]
    cu = R.starts([n] * b).cuda()
    assert torch.equal(cmpext3.attention(*flat, cu, cu).view(b, n, h, d), cmpext3.attention(q, k, v))
    # one head of keys and values for all batch entries
    one = cmpext3.attention(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1), causal=False)
    R.check(one[1], *R.attention(q[1].cpu(), k[0].cpu(), v[0].cpu(), d**-0.5, False))


@pytest.mark.parametrize("causal", [True, False])
def test_long_keys_are_split(causal):
    """One short stretch of queries over many keys: ranges of the keys are joined."""
    q, k, v = rand((2, 9, 4, 128), BF16, 1), rand((2, 5003, 2, 128), BF16, 2), rand((2, 5003, 2, 128), BF16, 3)
    got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), causal=causal).cpu()
    for i in range(2):
        R.check(got[i], *R.attention(q[i], k[i], v[i], 128**-0.5, causal))


@pytest.mark.parametrize("n", [511, 512, 700, 1100, 2100])
@pytest.mark.parametrize("dim", [64, 128])
def test_few_tiles_share_their_keys(n, dim):
    """Prompts with fewer row tiles than CUs: two groups of waves, and splits, over a tile's keys."""
    packed(BF16, [n], [n], 2, 1, dim, True, seed=n)
    packed(F16, [n, 5, 0, n - 300], [n, 70, 9, n], 2, 2, dim, False, seed=n)
    def spoil(q, k, v):
        k[n - 65 : n - 60] = float("nan")
        v[n - 65 : n - 60] = float("inf")
    q, k, v = (rand((n, 2, dim), BF16, s) for s in (1, 2, 3))
    one = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    clean = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), one, one).cpu()
    spoil(q, k, v)
    got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), one, one).cpu()
    assert torch.equal(got[: n - 65], clean[: n - 65]) and not got[n - 60 :].isfinite().any()


def test_large_scores():
    """Scores of some thousands, growing along the keys (the running maximum keeps moving), and a
    maximum that the first keys hold."""
    def grow(q, k, v):
        k *= torch.linspace(0, 40, k.shape[0]).to(k.dtype)[:, None, None]

    def fall(q, k, v):
        k *= torch.linspace(40, 0, k.shape[0]).to(k.dtype)[:, None, None]

    for change in (grow, fall):
        packed(F16, [300], [300], 2, 2, 64, False, scale=1.0, change=change)
        packed(BF16, [300], [300], 2, 2, 128, True, scale=1.0, change=change)
    packed(BF16, [50], [50], 2, 2, 64, True, scale=1e-30)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_a_row_does_not_see_takes_no_part(dtype, value, dim):
    """NaN and infinities in keys and values of later tokens and of other sequences."""
    lens = [70, 50, 90]
    def spoil(q, k, v):
        k[40:70] = value       # the first sequence's rows from 40 on see them
        v[40:70] = value
        k[130:133] = value     # the third one's
        v[130:133] = value

    q, k, v = (rand((210, 2, dim), dtype, s) for s in (1, 2, 3))
    clean = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), R.starts(lens).cuda(), R.starts(lens).cuda()).cpu()
    spoil(q, k, v)
    got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda(), R.starts(lens).cuda(), R.starts(lens).cuda()).cpu()
    for a, b in ((0, 40), (70, 120), (120, 130)):
        R.check(got[a:b], clean[a:b].double(), torch.zeros(b - a, 2, dim, dtype=torch.float64), f"rows {a}..{b}")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinite_values_that_are_seen(dtype):
    """Values of infinity and NaN at a key reach exactly the rows that see it, in their elements."""
    q, k, v = (rand((100, 2, 64), dtype, s) for s in (1, 2, 3))
    v[50, 0, 3] = float("inf")
    v[60, 0, 5] = float("-inf")
    v[70, 1, 7] = float("nan")
    got = cmpext3.attention(q.cuda(), k.cuda(), v.cuda()).cpu().float()
    fine = torch.ones(100, 2, 64, dtype=torch.bool)
    assert (got[50:, 0, 3] == float("inf")).all() and (got[60:, 0, 5] == float("-inf")).all()
    assert got[70:, 1, 7].isnan().all()
    fine[50:, 0, 3] = fine[60:, 0, 5] = fine[70:, 1, 7] = False
    assert got[fine].isfinite().all()


def test_other_streams_and_repeats():
    q, k, v = (rand((1, 700, 4, 128), BF16, s).cuda() for s in (1, 2, 3))
    want = cmpext3.attention(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [cmpext3.attention(q, k, v) for _ in range(3)]
    side.synchronize()
    for x in got:
        assert torch.equal(x, want)


def test_bad_starts_stay_inside():
    """Starts that are out of order or past the rows name no rows outside the tensors."""
    q = rand((64, 2, 64), F16, 1).cuda()
    for cu in ([0, 100, 64], [-5, 30, 64], [50, 10, 64], [64, 64, 1 << 30]):
        t = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = cmpext3.attention(q, q, q, t, t)
        torch.cuda.synchronize()
        assert out.shape == q.shape
