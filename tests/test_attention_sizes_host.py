"""Sizes whose products pass 64 bits: refused like any that are too large, before any launch."""
import ctypes

import pytest

from cmp_ext_amd import cabi
from tests.test_attention_host import BIG, attention_args, cache_args, size

MOST = 2**31 - 1


@pytest.mark.parametrize("batch,len_q", [(MOST, MOST), (MOST, 2**30), (2**30, 2**30), (2**29, 2**31 - 2**10), (MOST, 1), (1, MOST)])
@pytest.mark.parametrize("heads", [2, 4, 8, 64, 0xfffe])
@pytest.mark.parametrize("packed", [False, True])
def test_queries_of_all_batch_entries(batch, len_q, heads, packed):
    kw = dict(block_table=None, len_k=5) if packed else {}
    a = attention_args(batch=batch, len_q=len_q, heads=heads, **kw)
    assert size(a) == BIG
    assert cabi.lib().cmpext3_attention(ctypes.byref(a), None, 0, None) == BIG
    assert cabi.lib().cmpext3_attention_describe(ctypes.byref(a), None, 0) == BIG


@pytest.mark.parametrize("pages,page_size", [(MOST, MOST), (2**16, 2**16), (2**20, 2**10)])
def test_keys_of_a_table(pages, page_size):
    assert size(attention_args(table_pages=pages, cache=cache_args(page_size=page_size))) == BIG
    c = cache_args(page_size=page_size)
    read = cabi.lib().cmpext3_kv_cache_read
    if pages * page_size > MOST:
        assert read(ctypes.byref(c), 0x1000, 1, pages, 0x2000, 1, 1, cabi.F16, 0x4000, 0x5000, None) == BIG


@pytest.mark.parametrize("tokens", [2**63 - 1, 2**62, 2**50, 2**31])
def test_rows_of_rotation_and_cache(tokens):
    r = cabi.QkNormRopeArgs(dtype=cabi.F16, heads=0xffff, kv_heads=0xffff, dim=64, rotary_dim=64, tokens=tokens, q=0x1000, k=0x2000,
                            q_out=0x3000, k_out=0x4000, cos=0x5000, sin=0x6000, table_rows=8, table_row=32, positions=0x7000)
    assert cabi.lib().cmpext3_qk_norm_rope(ctypes.byref(r), None) == BIG
    c = cache_args(kv_heads=0xffff)
    assert cabi.lib().cmpext3_kv_cache_write(ctypes.byref(c), cabi.F16, 0x1000, 128, 64, 0x2000, 128, 64, 0x3000, tokens, None) == BIG
