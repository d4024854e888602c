"""Paged caches of keys and values (cmpext3.kv_cache_write / kv_cache_read): which bytes land
where, and codes and scales bit for bit as defined."""
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


def rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def make(pages, page, heads, dim, held, head_major=False):
    shape = (pages, heads, page, dim) if head_major else (pages, page, heads, dim)
    def one(s, dtype):
        t = torch.full(s, 1.0, dtype=torch.float32).to(dtype).cuda()
        return t.transpose(1, 2) if head_major else t
    caches = [one(shape, held) for _ in range(2)]
    scales = [one(shape[:3], torch.float32) for _ in range(2)] if held == F8 else [None, None]
    return caches, scales


def held_rows(cache, scale, slots):
    """What a cache holds at the slots, in 64 bits."""
    x = cache.cpu().float().flatten(0, 1)[slots].double()
    return x if scale is None else x * scale.cpu().flatten(0, 1)[slots].double()[..., None]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [8, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("head_major", [False, True])
def test_write_and_read(dtype, quantised, dim, head_major):
    held = F8 if quantised else dtype
    pages, page, heads = 13, 12, 3
    (kc, vc), (ks, vs) = make(pages, page, heads, dim, held, head_major)
    lens = [30, 1, 0, 25, 40]
    g = torch.Generator().manual_seed(dim)
    order = torch.randperm(pages, generator=g).int()
    table, at = torch.full((5, 5), -1, dtype=torch.int32), 0
    for i, n in enumerate(lens):
        need = -(-n // page)
        table[i, :need] = order[at : at + need]
        at += need
    seq = torch.repeat_interleave(torch.arange(5), torch.tensor(lens))
    place = torch.cat([torch.arange(n) for n in lens])
    slots = table[seq, place // page].long() * page + place % page
    k, v = rand((sum(lens), heads, dim), dtype, 1, 3.0), rand((sum(lens), heads, dim), dtype, 2, 0.01)
    mix = torch.randperm(sum(lens), generator=g)  # in any order
    cmpext3.kv_cache_write(k[mix].cuda(), v[mix].cuda(), kc, vc, slots[mix].cuda(), ks, vs)
    got = cmpext3.kv_cache_read(kc, vc, table.cuda(), R.starts(lens).cuda(), sum(lens), dtype=dtype, k_scale=ks, v_scale=vs)
    for x, cache, scale, back in ((k, kc, ks, got[0]), (v, vc, vs, got[1])):
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[slots] = False
        assert (cache.cpu().float().flatten(0, 1)[rest] == 1).all()  # nothing else was written
        if quantised:
            codes, scales = R.quantise(x)
            assert torch.equal(cache.cpu().view(torch.uint8).flatten(0, 1)[slots], codes.view(torch.uint8))
            assert torch.equal(scale.cpu().flatten(0, 1)[slots], scales)
            assert torch.equal(back.cpu(), (codes.float() * scales[..., None]).to(dtype))
            # within half a step of what was written
            off = (R.dequantise(codes, scales) - x.double()).abs()
            step = torch.maximum(x.double().abs() * 2.0**-4, scales.double()[..., None] * 2.0**-10)
            assert (off <= step * (1 + 2.0**-20)).all()
        else:
            assert torch.equal(back.cpu(), x)


@pytest.mark.parametrize("held", [F16, F8])
def test_slots_outside_are_left_out(held):
    (kc, vc), (ks, vs) = make(2, 4, 2, 64, held)
    k = rand((5, 2, 64), F16, 1)
    slots = torch.tensor([-1, 8, 1 << 40, 7, -(1 << 62)])
    cmpext3.kv_cache_write(k.cuda(), k.cuda(), kc, vc, slots.cuda(), ks, vs)
    for c, s in ((kc, ks), (vc, vs)):
        assert (c.cpu().float().flatten(0, 1)[:7] == 1).all()
        want = k[3].double() if s is None else R.dequantise(*R.quantise(k[3]))
        assert torch.equal(held_rows(c, s, torch.tensor([7]))[0], want)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_values_at_the_edges(dtype):
    """Zeros, the largest and smallest numbers, ties between codes; infinities and NaN by themselves."""
    most = torch.finfo(dtype).max
    x = torch.zeros(8, 1, 64, dtype=torch.float64)
    x[1] = most
    x[2, 0, 0], x[2, 0, 1:] = most, torch.linspace(-most, most, 63, dtype=torch.float64)
    x[3] = torch.finfo(dtype).tiny
    x[4] = torch.arange(-31.5, 32.5) * 14  # halfway between codes
    x[5] = torch.linspace(-2, 2, 64)
    x[6] = torch.linspace(-2, 2, 64)
    x[7, 0, 0] = 2.0**-14 if dtype == F16 else 1e-38
    x = x.to(dtype)
    x[5, 0, 3], x[5, 0, 9], x[6, 0, 0] = float("inf"), float("nan"), float("-inf")
    (kc, vc), (ks, vs) = make(1, 8, 1, 64, F8)
    cmpext3.kv_cache_write(x.cuda(), x.cuda(), kc, vc, torch.arange(8).cuda(), ks, vs)
    codes, scales = R.quantise(x)
    nan = codes.float().isnan()
    assert torch.equal(kc.cpu()[0].float().isnan(), nan) and int(nan.sum()) == 3
    assert torch.equal(kc.cpu()[0].float()[~nan], codes.float()[~nan])
    assert torch.equal(ks.cpu()[0], scales) and scales.isfinite().all()
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), R.starts([8]).cuda()
    back = cmpext3.kv_cache_read(kc, vc, table, cu, 8, dtype=dtype, k_scale=ks, v_scale=vs)[0].cpu()
    assert torch.equal(back.isnan(), nan) and back[~nan].isfinite().all()


@pytest.mark.parametrize("held", [BF16, F8])
def test_reading_stays_inside(held):
    """Rows of no sequence, lengths past the table and pages that are none read as zeros."""
    (kc, vc), (ks, vs) = make(3, 4, 2, 64, held)
    table = torch.tensor([[0, 7], [-3, 1]], dtype=torch.int32)
    cu = torch.tensor([2, 12, 18], dtype=torch.int32)  # 10 tokens in a table of 8, 6 tokens; total 20
    k, v = cmpext3.kv_cache_read(kc, vc, table.cuda(), cu.cuda(), 20, dtype=BF16, k_scale=ks, v_scale=vs)
    want = torch.zeros(20)
    want[2:6] = 1
    want[16:18] = 1
    for x in (k, v):
        assert torch.equal(x.cpu().float(), want[:, None, None].expand(20, 2, 64))
    assert cmpext3.kv_cache_read(kc, vc, table.cuda(), cu.cuda(), 0, dtype=BF16, k_scale=ks, v_scale=vs)[0].shape == (0, 2, 64)


def test_inputs_with_strides():
    (kc, vc), (ks, vs) = make(4, 8, 2, 64, F8)
    rows = rand((10, 2, 2, 64), BF16, 1).cuda()
    odd = torch.empty(10, 2, 65, dtype=BF16, device="cuda")[..., 1:]
    odd.copy_(rows[:, 0])
    slots = torch.arange(20, 30, device="cuda")
    cmpext3.kv_cache_write(rows[:, 0], rows[:, 1], kc, vc, slots, ks, vs)
    first = kc.view(torch.uint8).clone()
    cmpext3.kv_cache_write(odd, rows[:, 1].transpose(1, 2).contiguous().transpose(1, 2), kc, vc, slots, ks, vs)
    assert torch.equal(first, kc.view(torch.uint8))
    codes, scales = R.quantise(rows[:, 1].cpu())
    assert torch.equal(vc.cpu().view(torch.uint8).flatten(0, 1)[20:30], codes.view(torch.uint8))
    assert torch.equal(vs.cpu().flatten(0, 1)[20:30], scales)
    cmpext3.kv_cache_write(rows[:0, 0], rows[:0, 1], kc, vc, slots[:0], ks, vs)


def test_a_cache_past_32_bits():
    """Pages whose elements lie past 2^32 bytes."""
    page, heads, dim = 64, 8, 128
    pages = (5 << 30) // (page * heads * dim * 2)
    kc = torch.empty(pages, page, heads, dim, dtype=F16, device="cuda")
    k = rand((3, heads, dim), F16, 1)
    slots = torch.tensor([pages * page - 1, 5, pages * page - page])
    cmpext3.kv_cache_write(k.cuda(), k.cuda(), kc, kc, slots.cuda())
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    back = cmpext3.kv_cache_read(kc, kc, table, R.starts([page]).cuda(), page)[0].cpu()
    assert torch.equal(back[0], k[2]) and torch.equal(back[-1], k[0])
    q = rand((1, heads, dim), F16, 2)
    kc[pages - 1] = rand((page, heads, dim), F16, 3).cuda()
    got = cmpext3.paged_attention(q.cuda(), kc, kc, table, torch.tensor([page], dtype=torch.int32, device="cuda"))
    x = kc[pages - 1].cpu()
    R.check(got, *R.attention(q, x, x, dim**-0.5, True))
