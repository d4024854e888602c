"""Norms of queries and keys with the position rotation (cmpext3.qk_norm_rope, cmpext3.rope_table)
against the definition in 64 bits."""
import pytest
import torch

import cmpext3
from tests import attention_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def table(rows, rotary, seed):
    angle = torch.rand(rows, rotary // 2, generator=torch.Generator().manual_seed(seed)) * 6.3
    return angle.cos(), angle.sin()


def run(q, k, cos, sin, pos, wq, wk, eps, interleaved):
    dev = [None if x is None else x if x.is_cuda else x.cuda() for x in (q, k, cos, sin, pos, wq, wk)]
    got = cmpext3.qk_norm_rope(*dev, eps=eps, interleaved=interleaved)
    for y, x, w, name in ((got[0], q, wq, "q"), (got[1], k, wk, "k")):
        want, tol = R.rope(x.cpu(), w, cos, sin, pos, eps, interleaved)
        assert y.dtype == x.dtype and y.is_contiguous()
        R.check(y, want, tol, name)
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 32), (256, 256), (80, 80), (96, 32), (512, 64), (1024, 1024),
                                        (16, 16), (128, 0), (63, 20), (40, 40), (1, 0), (130, 66), (1000, 500)])
def test_head_sizes(dtype, interleaved, dim, rotary):
    cos, sin = table(50, rotary, 1)
    pos = torch.randint(0, 50, (7,), generator=torch.Generator().manual_seed(2))
    for norm in (True, False):
        w = [rand((dim,), dtype, 3 + i) if norm else None for i in range(2)]
        run(rand((7, 3, dim), dtype, 5), rand((7, 2, dim), dtype, 6), cos, sin, pos, *w, 1e-6, interleaved)


@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (513, 5, 1), (3, 0, 4), (3, 4, 0), (0, 4, 2)])
def test_counts(tokens, heads, kv_heads):
    cos, sin = table(9, 64, 1)
    pos = torch.arange(tokens) % 9
    run(rand((tokens, heads, 64), BF16, 1), rand((tokens, kv_heads, 64), BF16, 2), cos, sin, pos, rand((64,), BF16, 3),
        rand((64,), BF16, 4), 1e-5, False)


def test_one_weight_only():
    cos, sin = table(9, 64, 1)
    pos = torch.arange(5)
    q, k, w = rand((5, 4, 64), F16, 1), rand((5, 2, 64), F16, 2), rand((64,), F16, 3)
    run(q, k, cos, sin, pos, w, None, 1e-6, False)
    run(q, k, cos, sin, pos, None, w, 1e-6, True)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides(dtype):
    """Parts of a qkv product, transposed memory, and rows at odd addresses."""
    cos, sin = table(40, 64, 1)
    pos = torch.arange(20)
    rows = rand((20, 8 * 64), dtype, 1).cuda()
    q, k = rows[:, : 4 * 64].view(20, 4, 64), rows[:, 4 * 64 : 6 * 64].view(20, 2, 64)
    w = [rand((64,), dtype, 3), rand((64,), dtype, 4)]
    want = run(q, k, cos, sin, pos, *w, 1e-6, False)
    odd = torch.empty(20, 6, 65, dtype=dtype, device="cuda")[..., 1:]
    odd[:, :4], odd[:, 4:] = q, k
    run(odd[:, :4], odd[:, 4:], cos, sin, pos, *w, 1e-6, False)
    run(q.transpose(0, 1).contiguous().transpose(0, 1), k, cos, sin, pos, *w, 1e-6, True)
    run(q.transpose(1, 2).contiguous().transpose(1, 2), k.expand(20, 2, 64), cos, sin, pos, *w, 1e-6, False)
    assert not torch.equal(want[0], q)


def test_sizes_of_values():
    """Rows of zeros (eps alone), of the smallest and of large numbers, and infinities and NaN by themselves."""
    cos, sin = table(9, 64, 1)
    q = rand((9, 4, 64), BF16, 1)
    q[0] = 0
    q[1] *= 1e-20
    q[2] *= 1e15
    run(q, q[:, :1].clone(), cos, sin, torch.arange(9), rand((64,), BF16, 2), rand((64,), BF16, 3), 1e-6, False)
    q[4, 2, 5], q[5, 1, 6] = float("nan"), float("inf")
    got = cmpext3.qk_norm_rope(q.cuda(), q[:, :1].cuda(), cos.cuda(), sin.cuda(), torch.arange(9).cuda(),
                               torch.ones(64, dtype=BF16, device="cuda"))[0].cpu()
    spoilt = torch.zeros(9, 4, dtype=torch.bool)
    spoilt[4, 2] = spoilt[5, 1] = True
    assert got[~spoilt].isfinite().all() and not got[4, 2].isfinite().any()


@pytest.mark.parametrize("dim,rotary", [(64, 32), (60, 20)])
def test_positions_outside_the_table(dim, rotary):
    cos, sin = table(8, rotary, 1)
    pos = torch.tensor([0, 8, -1, 1 << 40, 7])
    q = rand((5, 2, dim), F16, 1)
    got = cmpext3.qk_norm_rope(q.cuda(), q.cuda(), cos.cuda(), sin.cuda(), pos.cuda())[0].cpu()
    assert got[[0, 4]].isfinite().all()
    assert got[[1, 2, 3]][..., :rotary].isnan().all()
    assert torch.equal(got[..., rotary:], q[..., rotary:])
