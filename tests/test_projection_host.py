"""The feed-forward operators without a GPU: what the Python surface and the C ABI refuse before any launch."""
import ctypes
import os
import re

import pytest
import torch

import cmpext3
from cmp_ext_amd import cabi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cmpext3_projection.h")
BAD, NOT, BIG, WORK = cabi.ERR_INVALID_ARG, cabi.ERR_UNSUPPORTED, cabi.ERR_TOO_LARGE, cabi.ERR_WORKSPACE


def header():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_exports_match_the_header():
    declared = set(re.findall(r"\b(cmpext3_\w+)\s*\(", header()))
    assert declared == set(cabi.PROJECTION_SIGNATURES)
    for name in declared:
        assert hasattr(cabi.lib(), name)


def test_structures_match_the_header():
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    for cls, name in ((cabi.QuantizeInt8Args, "cmpext3_quantize_int8_args"), (cabi.ProjectionArgs, "cmpext3_projection_args"),
                      (cabi.GatedBackwardArgs, "cmpext3_gated_backward_args")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header(), re.S).group(1)
        want = []
        for line in body.split(";"):
            m = re.match(r"\s*(const )?(\w+)(\*?)\s+(.*)", line.strip(), re.S)
            if not m:
                continue
            for field in m.group(4).split(","):
                pointer = m.group(3) or field.strip().startswith("*")
                want.append((field.strip().lstrip("*"), ctypes.c_void_p if pointer else kinds[m.group(2)]))
        assert [tuple(f) for f in cls._fields_] == want


def test_constants_match_the_header():
    for name, value in re.findall(r"#define CMPEXT3_(ACT_\w+|I8) (\d+)", header()):
        assert getattr(cabi, name) == int(value)


def refuses(match, fn, *args, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def test_python_refusals():
    h, c = torch.zeros(3, 16, dtype=torch.float16), torch.zeros(5, 16, dtype=torch.int8)
    s = torch.ones(5)
    refuses("on a GPU", cmpext3.quantize_int8, h)
    refuses("unsupported dtype", cmpext3.quantize_int8, h.double())
    refuses("unsupported dtype", cmpext3.quantize_int8, c)
    refuses("at least one dimension", cmpext3.quantize_int8, h[0, 0])
    refuses("on a GPU", cmpext3.int8_linear, h, c, s)
    refuses("at least one dimension", cmpext3.int8_linear, h[0, 0], c, s)
    refuses("on a GPU", cmpext3.int8_gated_linear, h, c, c, s, s)
    refuses("unknown activation 'swish'", cmpext3.int8_gated_linear, h, c, c, s, s, "swish")
    refuses("on a GPU", cmpext3.gated_linear, h, c.half(), c.half())


def projection(**kw):
    dtype = kw.get("dtype", cabi.BF16)
    a = cabi.ProjectionArgs(dtype=dtype, x_dtype=dtype, out_dtype=cabi.BF16, activation=cabi.ACT_SILU, M=8, N=64, K=128, x=0x1000, x_row=128,
                            w_gate=0x2000, gate_row=128, w_up=0x3000, up_row=128, out=0x4000, out_row=64)
    if kw.get("dtype") == cabi.I8:
        a.x_scale, a.gate_scale, a.up_scale = 0x5000, 0x6000, 0x7000
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def size(a):
    return cabi.lib().cmpext3_projection_workspace_size(ctypes.byref(a))


def test_projection_c_abi_rejects():
    i8 = dict(dtype=cabi.I8)
    assert size(projection()) >= 0 and size(projection(**i8)) >= 0 and size(projection(out_dtype=cabi.F32, **i8)) >= 0
    assert size(projection(w_up=None, bias=0x8000, **i8)) >= 0
    assert all(size(projection(x_dtype=t, x_scale=None, **i8)) >= 0 for t in (cabi.F16, cabi.BF16, cabi.F32))
    assert cabi.lib().cmpext3_projection_workspace_size(None) == BAD
    for kw in (dict(dtype=cabi.F32), dict(dtype=cabi.E4M3), dict(out_dtype=cabi.F32), dict(out_dtype=cabi.F16), dict(w_up=None),
               dict(activation=4), dict(activation=-1), dict(bias=0x8000), dict(out_dtype=cabi.I8, **i8), dict(x_dtype=cabi.F16),
               dict(x_dtype=cabi.I8), dict(x_dtype=cabi.E4M3, **i8),
               dict(gate_out=0x100, up_out=0x200, pre_row=64, **i8)):
        assert size(projection(**kw)) == NOT, kw
    for kw in (dict(M=-1), dict(N=-1), dict(K=-1), dict(x=None), dict(w_gate=None), dict(out=None), dict(x_row=127), dict(gate_row=127),
               dict(up_row=100), dict(out_row=63), dict(x=0x1001), dict(out=0x4001), dict(gate_out=0x100, pre_row=64),
               dict(gate_out=0x100, up_out=0x200, pre_row=63), dict(x_scale=None, **i8), dict(x_dtype=cabi.F16, **i8), dict(gate_scale=None, **i8),
               dict(up_scale=None, **i8), dict(x_scale=0x5002, **i8), dict(out=0x4002, out_dtype=cabi.F32, **i8),
               dict(w_up=None, bias=0x8001, **i8)):
        assert size(projection(**kw)) == BAD, kw
    for kw in (dict(K=131072, x_row=131072, gate_row=131072, up_row=131072, **i8), dict(x_row=1 << 31), dict(gate_row=1 << 40),
               dict(M=2**31 - 1), dict(N=2**31 - 1, out_row=2**31 - 1), dict(out_row=1 << 31)):
        assert size(projection(**kw)) == BIG, kw
    assert size(projection(M=0, x=None, out=None)) == 0 and size(projection(N=0, w_gate=None)) == 0
    assert size(projection(K=131071, x_row=131071, gate_row=131071, up_row=131071, **i8)) >= 0
    lib = cabi.lib()
    assert lib.cmpext3_projection(ctypes.byref(projection(M=0)), None, 0, None) == 0
    assert lib.cmpext3_projection(ctypes.byref(projection(M=-1)), None, 0, None) == BAD
    assert lib.cmpext3_projection_describe(ctypes.byref(projection(M=-1)), None, 0) == BAD


def plan(**kw):
    buf = ctypes.create_string_buffer(256)
    assert cabi.lib().cmpext3_projection_describe(ctypes.byref(projection(**kw)), buf, 256) == 0
    return buf.value.decode()


def sized(m, n, k, **kw):
    return dict(M=m, N=n, K=k, x_row=k, gate_row=k, up_row=k, out_row=n, **kw)


def test_plans(monkeypatch):
    """Which kernel a call takes, by its sizes, types and alignment."""
    monkeypatch.delenv("CMPEXT3_PROJECTION_CONFIG", raising=False)
    i8 = dict(dtype=cabi.I8)
    assert plan(M=0) == "kernel=none" and plan(**sized(8, 64, 7)) == "kernel=any64x64" and plan(**sized(8, 64, 0)) == "kernel=any64x64"
    assert plan(**sized(16, 14336, 4096)) == "kernel=rows" and plan(**sized(64, 4096, 4096)) == "kernel=rows"
    assert plan(**sized(64, 14336, 4096)) != "kernel=rows"  # fills the CUs: tiles are as fast
    assert "small64x64" in plan(**sized(16, 4099, 1001))  # odd rows: no strips of 16 bytes
    assert "small64x64" in plan(x=0x1002, **sized(16, 4096, 1024))
    assert "tile256x256" in plan(**sized(4096, 14336, 4096)) and "copies=0" in plan(**sized(4096, 14336, 4096))
    assert "copies=3" in plan(**sized(4096, 14336, 4097)) and "tile256x256" in plan(**sized(4096, 14336, 4097))
    assert "tile256x128" in plan(**sized(256, 14336, 4096))
    assert "groups=2" in plan(w_up=None, **sized(256, 4096, 4096, **i8)) and "splits=1 " not in plan(**sized(100, 512, 16384))
    codes = dict(x_scale=None, x_dtype=cabi.BF16, w_up=None, **i8)
    assert plan(**sized(1, 4096, 4096, **codes)) == "kernel=rows codes=inside"
    assert plan(**sized(2, 4096, 4096, **codes)) == "kernel=rows"
    assert plan(**sized(1, 4096, 4000, **codes)) == "kernel=rows" and "codes=inside" in plan(**sized(8, 4096, 512, **codes))
    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=tile128x128,splits=3")
    assert "tile128x128" in plan(**sized(256, 4096, 4096)) and "splits=3" in plan(**sized(256, 4096, 4096))
    monkeypatch.setenv("CMPEXT3_PROJECTION_CONFIG", "kernel=nothing")
    assert plan(**sized(16, 14336, 4096)) == "kernel=rows"


def test_workspace_covers_what_a_plan_needs(monkeypatch):
    monkeypatch.delenv("CMPEXT3_PROJECTION_CONFIG", raising=False)
    assert size(projection(**sized(4096, 14336, 4096))) == 0
    pitch = 4104 * 2  # of 4097 elements in whole 16 bytes
    assert size(projection(**sized(4096, 14336, 4097))) >= pitch * (4096 + 2 * 14336)
    i8 = dict(dtype=cabi.I8, x_dtype=cabi.F32, x_scale=None)
    assert size(projection(**sized(100, 512, 1000, **i8))) >= 100 * 1008 + 100 * 4
    a = projection(**sized(100, 512, 1000, **i8))
    assert cabi.lib().cmpext3_projection(ctypes.byref(a), None, 0, None) == WORK


def backward(**kw):
    a = cabi.GatedBackwardArgs(dtype=cabi.F16, activation=cabi.ACT_GELU, M=8, N=64, K=128, grad_out=0x1000, grad_row=64, gate=0x2000,
                               up=0x3000, pre_row=64, x=0x4000, x_row=128, w_gate=0x5000, gate_row=128, w_up=0x6000, up_row=128,
                               dx=0x7000, dx_row=128, dw_gate=0x8000, dgate_row=128, dw_up=0x9000, dup_row=128)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_gated_backward_c_abi_rejects():
    lib = cabi.lib()

    def need(a):
        return lib.cmpext3_gated_backward_workspace_size(ctypes.byref(a))

    assert need(backward()) >= 2 * 2 * 8 * 64
    assert lib.cmpext3_gated_backward_workspace_size(None) == BAD
    for kw in (dict(dtype=cabi.F32), dict(dtype=cabi.I8), dict(activation=4), dict(activation=-1)):
        assert need(backward(**kw)) == NOT, kw
    for kw in (dict(M=-1), dict(N=-1), dict(K=-1), dict(grad_out=None), dict(gate=None), dict(up=None), dict(x=None), dict(w_gate=None),
               dict(w_up=None), dict(grad_row=63), dict(pre_row=63), dict(x_row=127), dict(gate_row=127), dict(up_row=127), dict(dx_row=127),
               dict(dgate_row=127), dict(dup_row=127), dict(dx=0x7001)):
        assert need(backward(**kw)) == BAD, kw
    for kw in (dict(M=2**31 - 1), dict(x_row=1 << 31), dict(M=1 << 25)):
        assert need(backward(**kw)) == BIG, kw
    # what is not asked for needs no operands
    assert need(backward(dx=None, w_gate=None, w_up=None)) >= 0
    assert need(backward(dw_gate=None, dw_up=None, x=None)) >= 0
    a = backward()
    assert lib.cmpext3_gated_backward(ctypes.byref(a), None, 0, None) == WORK
    assert lib.cmpext3_gated_backward(ctypes.byref(a), 0x10000, need(a) - 1, None) == WORK
    assert lib.cmpext3_gated_backward(ctypes.byref(a), 0x10008, need(a), None) == WORK


def test_quantize_c_abi_rejects():
    def call(**kw):
        a = cabi.QuantizeInt8Args(dtype=cabi.F16, cols=64, rows=3, x=0x1000, x_row=64, codes=0x2000, codes_row=64, scale=0x3000)
        for name, value in kw.items():
            setattr(a, name, value)
        return cabi.lib().cmpext3_quantize_int8(ctypes.byref(a), None)

    assert cabi.lib().cmpext3_quantize_int8(None, None) == BAD
    assert call(dtype=cabi.I8) == NOT and call(dtype=cabi.E4M3) == NOT
    for kw in (dict(rows=-1), dict(cols=-1), dict(x=None), dict(codes=None), dict(scale=None), dict(x_row=63), dict(codes_row=63),
               dict(x=0x1001), dict(scale=0x3002)):
        assert call(**kw) == BAD, kw
    assert call(rows=1 << 40) == BIG
    assert call(rows=0) == 0
