"""The attention operators without a GPU: what the Python surface and the C ABI refuse before any
launch, the plans of the kernels, and the rotation tables."""
import ctypes
import os
import re

import pytest
import torch

import cmpext3
from cmp_ext_amd import cabi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cmpext3_attention.h")
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
I32, I64 = torch.int32, torch.int64


def test_exports_match_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(cmpext3_\w+)\s*\(", text))
    assert declared == set(cabi.ATTENTION_SIGNATURES)
    for name in declared:
        assert hasattr(cabi.lib(), name)


def test_structures_match_the_header():
    """Field by field: names, order and types of the ctypes structures."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "cmpext3_kv_cache": cabi.KvCache}
    for cls, name in ((cabi.QkNormRopeArgs, "cmpext3_qk_norm_rope_args"), (cabi.KvCache, "cmpext3_kv_cache"),
                      (cabi.AttentionArgs, "cmpext3_attention_args")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        want = []
        for line in body.split(";"):
            m = re.match(r"\s*(const )?(\w+)(\*?)\s+(.*)", line.strip(), re.S)
            if not m:
                continue
            for field in m.group(4).split(","):
                pointer = m.group(3) or field.strip().startswith("*")
                want.append((field.strip().lstrip("*"), ctypes.c_void_p if pointer else kinds[m.group(2)]))
        assert [tuple(f) for f in cls._fields_] == want


# ---------------------------------------------------------------- Python surface
def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def refuses(match, fn, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def test_qk_norm_rope_refusals():
    f = cmpext3.qk_norm_rope
    q, k, c, p = z(4, 8, 64), z(4, 2, 64), z(16, 32, dtype=torch.float32), z(4, dtype=I64)
    refuses("on a GPU", f, q, k, c, c, p)
    refuses(r"\[tokens, heads, dim\]", f, q[0], k, c, c, p)
    refuses("dtype mismatch", f, q, k.float(), c, c, p)
    refuses("unsupported dtype", f, q.double(), k.double(), c, c, p)
    refuses("shape mismatch", f, q, z(3, 2, 64), c, c, p)
    refuses("shape mismatch", f, q, z(4, 2, 32), c, c, p)
    refuses("float32", f, q, k, c.half(), c.half(), p)
    refuses("float32", f, q, k, c, c[:, :3], p)
    refuses("turn", f, q, k, z(16, 33, dtype=torch.float32), z(16, 33, dtype=torch.float32), p)
    refuses("head size", f, z(4, 1, 1025), z(4, 1, 1025), c, c, p)
    refuses("eps", f, q, k, c, c, p, eps=-1.0)
    refuses("eps", f, q, k, c, c, p, eps=float("nan"))


def test_kv_cache_refusals():
    w, r = cmpext3.kv_cache_write, cmpext3.kv_cache_read
    k, c, s = z(4, 2, 64), z(3, 16, 2, 64), z(4, dtype=I64)
    c8, sc = z(3, 16, 2, 64, dtype=torch.float32).to(F8), z(3, 16, 2, dtype=torch.float32)
    refuses("on a GPU", w, k, k, c, c, s)
    refuses("caches must be", w, k, k, c[0], c[0], s)
    refuses("cache shape mismatch", w, k, k, c, c[:2], s)
    refuses("cache dtype mismatch", w, k, k, c, c.bfloat16(), s)
    refuses("unsupported cache dtype", w, k, k, c.float(), c.float(), s)
    refuses("needs k_scale", w, k, k, c8, c8, s)
    refuses("needs k_scale", w, k, k, c8, c8, s, sc)
    refuses("only a float8", w, k, k, c, c, s, sc, sc)
    refuses("scales must be", w, k, k, c8, c8, s, sc[:, :3], sc)
    refuses("scales must be", w, k, k, c8, c8, s, sc.half(), sc.half())
    refuses("multiple of 8", w, z(4, 2, 60), z(4, 2, 60), z(3, 16, 2, 60), z(3, 16, 2, 60), s)
    refuses("multiple of 8", w, k, k, z(3, 16, 2, 264), z(3, 16, 2, 264), s)
    odd = z(3, 16, 2, 65)[..., 1:]
    refuses("unit stride|multiples of 8", w, k, k, odd, odd, s)
    refuses("like the cache", w, z(4, 3, 64), z(4, 3, 64), c, c, s)
    refuses("like the cache", w, k, k[:3], c, c, s)
    refuses("float16 or bfloat16", w, k.float(), k.float(), c8, c8, s, sc, sc)
    refuses("dtype mismatch with the cache", w, k.bfloat16(), k.bfloat16(), c, c, s)
    t, cu = z(1, 2, dtype=I32), z(2, dtype=I32)
    refuses("on a GPU", r, c, c, t, cu, 4)
    refuses("dtype must be", r, c8, c8, t, cu, 4, k_scale=sc, v_scale=sc)
    refuses("dtype mismatch", r, c, c, t, cu, 4, dtype=BF16)
    refuses("total", r, c, c, t, cu, -1)


def test_attention_refusals():
    f = cmpext3.attention
    q, k = z(1, 5, 4, 64), z(1, 5, 2, 64)
    refuses("on a GPU", f, q, k, k)
    refuses("q, k and v must be", f, q, k[0], k[0])
    refuses("q, k and v must be", f, q[0, 0], k[0, 0], k[0, 0])
    refuses("shape mismatch", f, q, k, k[:, :3])
    refuses("head size mismatch", f, q, z(1, 5, 2, 32), z(1, 5, 2, 32))
    refuses("no multiple", f, q, z(1, 5, 3, 64), z(1, 5, 3, 64))
    refuses("no multiple", f, q, z(1, 5, 0, 64), z(1, 5, 0, 64))
    refuses("unsupported dtype", f, q.float(), k.float(), k.float())
    refuses("dtype mismatch", f, q, k.bfloat16(), k.bfloat16())
    refuses("multiple of 8", f, q[..., :60], k[..., :60], k[..., :60])
    refuses("multiple of 8", f, z(1, 5, 4, 264), z(1, 5, 2, 264), z(1, 5, 2, 264))
    refuses("batch size", f, q, z(2, 5, 2, 64), z(2, 5, 2, 64))
    cu = z(2, dtype=I32)
    refuses("go together", f, q[0], k[0], k[0], cu)
    refuses("packed", f, q, k, k, cu, cu)
    for scale in (0.0, -1.0, float("inf"), float("nan"), 1e-60):
        refuses("scale", f, q, k, k, scale=scale)


def test_paged_attention_refusals():
    f = cmpext3.paged_attention
    q, c, t, n = z(2, 4, 64), z(3, 16, 2, 64), z(2, 2, dtype=I32), z(2, dtype=I32)
    refuses("on a GPU", f, q, c, c, t, n)
    refuses(r"\[tokens, heads, dim\]", f, q[0], c, c, t, n)
    refuses("head size mismatch", f, q[..., :32], c, c, t, n)
    refuses("no multiple", f, q[:, :3], c, c, t, n)
    refuses("unsupported dtype", f, q.float(), c, c, t, n)
    refuses("dtype mismatch", f, q.bfloat16(), c, c, t, n)
    refuses("scale must", f, q, c, c, t, n, scale=0.0)
    refuses("only a float8", f, q, c, c, t, n, k_scale=z(3, 16, 2, dtype=torch.float32), v_scale=z(3, 16, 2, dtype=torch.float32))


# ---------------------------------------------------------------- C ABI
def cache_args(**kw):
    c = cabi.KvCache(kv_dtype=cabi.F16, pages=10, page_size=16, kv_heads=2, dim=64, k=0x1000, v=0x2000, k_page=2048, k_token=128,
                     k_head=64, v_page=2048, v_token=128, v_head=64)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def attention_args(cache=None, **kw):
    a = cabi.AttentionArgs(dtype=cabi.F16, batch=2, heads=8, causal=1, scale=0.125, len_q=1, q=0x10000, out=0x20000, q_batch=512,
                           q_token=512, q_head=64, out_batch=512, out_token=512, out_head=64, cache=cache or cache_args(),
                           block_table=0x30000, table_row=5, table_pages=5, seq_lens=0x40000)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def size(a):
    return cabi.lib().cmpext3_attention_workspace_size(ctypes.byref(a))


BAD, NOT, BIG = cabi.ERR_INVALID_ARG, cabi.ERR_UNSUPPORTED, cabi.ERR_TOO_LARGE


@pytest.mark.parametrize("kw,err", [
    (dict(dtype=cabi.F32), NOT), (dict(dtype=9), NOT), (dict(batch=-1), BAD), (dict(heads=7), BAD), (dict(heads=0), BAD),
    (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("inf")), BAD), (dict(scale=float("nan")), BAD),
    (dict(len_q=-1), BAD), (dict(q=None), BAD), (dict(out=None), BAD), (dict(q=0x10008), BAD), (dict(out=0x20004), BAD),
    (dict(q_token=511), BAD), (dict(q_head=60), BAD), (dict(out_token=510), BAD), (dict(table_pages=-1), BAD),
    (dict(seq_lens=None), BAD), (dict(table_pages=1 << 28), BIG), (dict(len_q=1 << 30), BIG), (dict(heads=1 << 17), BIG),
    (dict(batch=1 << 23), BIG),
])
def test_attention_rejects_before_launch(kw, err):
    a = attention_args(**kw)
    assert size(a) == err
    assert cabi.lib().cmpext3_attention(ctypes.byref(a), None, 0, None) == err


@pytest.mark.parametrize("kw,err", [
    (dict(kv_dtype=cabi.BF16), NOT), (dict(kv_dtype=cabi.F32), NOT), (dict(kv_dtype=7), NOT), (dict(kv_heads=0), BAD),
    (dict(dim=0), BAD), (dict(dim=60), NOT), (dict(dim=264), NOT), (dict(k=0x1008), BAD), (dict(v=0x2004), BAD),
    (dict(k_page=2047), BAD), (dict(v_token=124), BAD), (dict(k_head=68), BAD), (dict(pages=-1), BAD), (dict(page_size=0), BAD),
    (dict(k=None), BAD), (dict(kv_dtype=cabi.E4M3), BAD), (dict(kv_heads=1 << 17), BIG),
])
def test_caches_are_checked(kw, err):
    a = attention_args(cache=cache_args(**kw))
    assert cabi.lib().cmpext3_attention(ctypes.byref(a), None, 0, None) == err
    if kw != dict(kv_dtype=cabi.BF16):
        c = cache_args(**kw)
        assert cabi.lib().cmpext3_kv_cache_write(ctypes.byref(c), cabi.F16, 0x1000, 128, 64, 0x2000, 128, 64, 0x3000, 1, None) == err
        assert cabi.lib().cmpext3_kv_cache_read(ctypes.byref(c), 0x1000, 1, 1, 0x2000, 1, 1, cabi.F16, 0x4000, 0x5000, None) == err


def test_packed_attention_rejects():
    def args(**kw):
        a = attention_args(block_table=None, len_k=5)
        for name, value in kw.items():
            setattr(a, name, value)
        return a

    assert size(args()) == 0
    assert size(args(len_k=-1)) == BAD
    assert size(args(cache=cache_args(k=None))) == BAD
    assert size(args(cache=cache_args(k=None, v=None), len_k=0)) == 0
    assert size(args(cache=cache_args(kv_dtype=cabi.E4M3))) == NOT
    assert size(args(cache=cache_args(k_token=1 << 30))) == BIG
    assert size(args(starts_k=0x1000, total_k=-1)) == BAD
    assert size(args(starts_q=0x1000, total_q=-1)) == BAD


def test_workspace_and_nothing_to_do():
    lib = cabi.lib()
    long = attention_args(table_pages=4096)
    need = size(long)
    assert need > 0 and need % 4 == 0
    assert lib.cmpext3_attention(ctypes.byref(long), None, 0, None) == cabi.ERR_WORKSPACE
    assert lib.cmpext3_attention(ctypes.byref(long), 0x1000, need - 1, None) == cabi.ERR_WORKSPACE
    assert lib.cmpext3_attention(ctypes.byref(long), 0x1008, need, None) == cabi.ERR_WORKSPACE
    for kw in (dict(batch=0), dict(len_q=0), dict(starts_q=0x1000, total_q=0)):
        a = attention_args(q=None, out=None, **kw)
        assert lib.cmpext3_attention(ctypes.byref(a), None, 0, None) == 0
    assert lib.cmpext3_attention(None, None, 0, None) == BAD
    c = cache_args()
    assert lib.cmpext3_kv_cache_write(ctypes.byref(c), cabi.F16, None, 0, 0, None, 0, 0, None, 0, None) == 0
    assert lib.cmpext3_kv_cache_read(ctypes.byref(c), None, 0, 0, None, 0, 0, cabi.F16, None, None, None) == 0


def test_plans():
    def plan(**kw):
        buf = ctypes.create_string_buffer(256)
        assert cabi.lib().cmpext3_attention_describe(ctypes.byref(attention_args(**kw)), buf, 256) == 0
        return buf.value.decode()

    assert "attention_few rows=16 groups=1 keys=paged16" in plan()
    assert "attention_few rows=32" in plan(len_q=8)
    assert "attention_tile" in plan(len_q=64) and "splits=1 " in plan(len_q=64)
    assert "keys=paged8" in plan(cache=cache_args(kv_dtype=cabi.E4M3, k_scale=0x100, v_scale=0x200))
    assert "splits=1 " in plan(batch=5000, table_pages=60) and "splits=1 " not in plan(table_pages=4096)
    assert plan(batch=0) == "kernel=none"


def test_qk_norm_rope_c_abi_rejects():
    def call(**kw):
        a = cabi.QkNormRopeArgs(dtype=cabi.F16, heads=4, kv_heads=2, dim=64, rotary_dim=64, tokens=3, q=0x1000, k=0x2000, q_out=0x3000,
                                k_out=0x4000, q_token=256, q_head=64, k_token=128, k_head=64, q_out_token=256, q_out_head=64,
                                k_out_token=128, k_out_head=64, cos=0x5000, sin=0x6000, table_rows=8, table_row=32, positions=0x7000)
        for name, value in kw.items():
            setattr(a, name, value)
        return cabi.lib().cmpext3_qk_norm_rope(ctypes.byref(a), None)

    assert call(dtype=cabi.E4M3) == NOT and call(dim=1025) == NOT
    for kw in (dict(dim=0), dict(tokens=-1), dict(heads=-1), dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=-2), dict(q=None),
               dict(k_out=None), dict(positions=None), dict(cos=None), dict(table_rows=-1)):
        assert call(**kw) == BAD, kw
    assert call(tokens=1 << 40) == BIG and call(heads=1 << 20) == BIG and call(tokens=1 << 24) == BIG
    assert call(tokens=0, q=None) == 0 and call(heads=0, kv_heads=0) == 0


def test_plan_of_many_uneven_tiles():
    """Chunks of up to 62 sequences whose row tiles fill the GPU go in the order of their keys, whole."""
    def plan(**kw):
        buf = ctypes.create_string_buffer(256)
        a = attention_args(starts_q=0x1000, len_q=0, **kw)
        assert cabi.lib().cmpext3_attention_describe(ctypes.byref(a), buf, 256) == 0
        return buf.value.decode()

    kv = attention_args().cache.kv_heads
    for batch, tiles, pages, sorted_ in ((32, 1200, 8, True), (62, 1200, 4096, True), (63, 1200, 8, False), (4, 1200, 8, False),
                                         (32, 560, 8, True), (32, 560, 4096, False), (32, 300, 8, False)):
        rows = (tiles // kv - batch + 1) * 128  # of one kv head
        a = attention_args()
        got = plan(batch=batch, total_q=max(rows, 40 * batch) // (a.heads // kv), table_pages=pages)
        assert ("order=longest" in got) == sorted_, (batch, tiles, pages, got)
        assert not sorted_ or "splits=1 " in got


def test_keys_counted_in_32_bits():
    """Sums of two key numbers are taken in 32 bits: 2^30 keys of a sequence at most."""
    assert size(attention_args(table_pages=2**30 // attention_args().cache.page_size)) == BIG
    assert size(attention_args(table_pages=2**30 // attention_args().cache.page_size - 1)) >= 0


def test_plan_of_short_keys():
    """Few rows: whole keys up to some hundreds, with eight waves for 8 bits; longer ones in splits."""
    def plan(held=cabi.F16, **kw):
        buf = ctypes.create_string_buffer(256)
        a = attention_args(cache=cache_args(kv_dtype=held, k_scale=0x100, v_scale=0x200), **kw)
        assert cabi.lib().cmpext3_attention_describe(ctypes.byref(a), buf, 256) == 0
        return buf.value.decode()

    page = cache_args().page_size
    assert "attention_few " in plan(table_pages=256 // page) and "splits=1 " in plan(table_pages=256 // page)
    assert "splits=1 " not in plan(table_pages=512 // page) and "splits=1 " in plan(table_pages=512 // page, batch=8)
    assert "attention_few8 " in plan(cabi.E4M3, table_pages=512 // page) and "attention_few " in plan(cabi.E4M3, table_pages=64 // page)
    assert "attention_few " in plan(cabi.E4M3, table_pages=1024 // page) and "splits=1 " not in plan(cabi.E4M3, table_pages=1024 // page)
    assert "attention_few8 " in plan(cabi.E4M3, table_pages=1024 // page, batch=128)
    assert "attention_few " in plan(cabi.E4M3, table_pages=512 // page, batch=1000)


def test_plan_of_splits_found_on_the_device():
    """Chunks over long keys: the splits of up to 62 sequences follow from their lengths."""
    def plan(**kw):
        buf = ctypes.create_string_buffer(256)
        a = attention_args(starts_q=0x1000, len_q=0, **kw)
        assert cabi.lib().cmpext3_attention_describe(ctypes.byref(a), buf, 256) == 0
        return buf.value.decode()

    page = cache_args().page_size
    assert "fit=512" in plan(batch=4, total_q=1500, table_pages=8192 // page) and "splits=1 " not in plan(batch=4, total_q=1500, table_pages=8192 // page)
    assert "fit=0" in plan(batch=40, total_q=6000, table_pages=65536 // page)
    assert "fit=0" in plan(batch=63, total_q=3000, table_pages=8192 // page)
    assert "fit=0" in plan(batch=4, total_q=1500, table_pages=2048 // page) and "groups=2" in plan(batch=4, total_q=1500, table_pages=2048 // page)
