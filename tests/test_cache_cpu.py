"""The cached-attention operators without a GPU: what the host side refuses, and the C entries' checks."""

import ctypes

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tinygrad_dx12_b200 import _lib
from tinygrad_dx12_b200 import attention as A


def cache(**kw):
    a = dict(pages=2, page_size=16, kv_heads=2, head_dim=64, format="int8", device="cpu")
    return tg.PackedCache.empty(**{**a, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(format="int3"), "unknown cache format"),
    (dict(head_dim=96), "head_dim"),
    (dict(block_size=16), "block_size"),
    (dict(block_size=0), "block_size"),
    (dict(page_size=24), "page_size"),
    (dict(page_size=8), "page_size"),
    (dict(kv_heads=0), "key head"),
    (dict(scale_dtype=torch.float16), "scales"),
    (dict(order="pages"), "order"),
    (dict(pages=-1), "pages"),
])
def test_cache_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        cache(**kw)


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("fmt,row", [("int8", 64), ("fp8e4m3", 64), ("int4", 32), ("fp4_e2m1", 32)])
def test_cache_layout(order, fmt, row):
    c = cache(format=fmt, block_size=32, order=order, scale_dtype=torch.float8_e8m0fnu)
    assert c.k.shape == (2, 2, 16, row) and c.k_scales.shape == (2, 2, 16, 2)
    assert (c.pages, c.kv_heads, c.page_size) == (2, 2, 16)
    assert c.k.stride(1) == (16 * row if order == "heads" else row)
    assert c.token_bytes() == 2 * 2 * (row + 2)


def test_cache_parts_must_agree():
    c = cache()
    ok = (c.k, c.v, c.k_scales, c.v_scales, "int8", 64, 64)
    tg.PackedCache(*ok)
    for i, t in [(0, c.k.int()), (1, c.v[:1]), (2, c.k_scales.float()), (3, c.v_scales[:, :1]), (0, c.k[..., :32]),
                 (1, c.v.transpose(1, 2).contiguous().transpose(1, 2))]:
        bad = list(ok)
        bad[i] = t
        with pytest.raises(ValueError):
            tg.PackedCache(*bad)


def test_caches_compare_by_identity():
    a, b = cache(), cache()
    assert a == a and a != b and len({a, b, a}) == 2 and [b, a].index(a) == 1


def test_no_cpu_path():
    c = cache()
    x = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        tg.cache_write(c, x, x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        tg.cache_read(c, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        tg.cache_attention(x.half(), c, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        tg.RotaryTable(torch.zeros(4, 8), torch.zeros(4, 8))


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rows=0), dict(base=0.0), dict(factor=0.0),
                                dict(scaling="other"), dict(scaling="base", rotary_dim=2, factor=2.0)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        tg.RotaryTable.build(**{**dict(rotary_dim=8, rows=4, device="cpu"), **kw})


def _desc(**kw):
    d = A.CacheDesc(4096, 4096, 4096, 4096, 2, 16, 2, 64, 64, 0, _lib.DT["bfloat16"], (ctypes.c_int64 * 3)(2048, 1024, 64),
                    (ctypes.c_int64 * 3)(32, 16, 1))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,msg", [
    (dict(format=4), "unknown cache format"), (dict(scale_dtype=12), "scales must be"), (dict(head_dim=65), "head_dim"),
    (dict(block_size=16), "block_size"), (dict(page_size=48), "page_size"), (dict(pages=-1), "pages"),
    (dict(kv_heads=0), "kv_heads"), (dict(k=None), "null cache storage"), (dict(v=4097), "16-byte"),
    (dict(strides=(ctypes.c_int64 * 3)(2048, 1024, 60)), "multiples of 16"),
])
def test_c_entries_check_the_cache(kw, msg):
    lib, d = _lib.lib(), _desc(**kw)
    a = A.AttentionArgs()
    for rc in (lib.b200_cache_attention(ctypes.byref(d), ctypes.byref(a), None),
               lib.b200_cache_read(ctypes.byref(d), None, 6, 0, None, None, 12, None),
               lib.b200_cache_write(ctypes.byref(d), None, 0, 0, None, 0, 0, 12, 0, None, 6, None, None, 0, None, 0, 0, 0, None, None)):
        assert rc == _lib.ERR_INVALID and msg in _lib.last_error()


def test_c_entries_check_arguments():
    lib, d = _lib.lib(), _desc()
    ref = ctypes.byref(d)

    def attention(**kw):
        a = A.AttentionArgs()
        a.q = a.out = a.tables = a.lengths = 4096
        a.batch, a.queries, a.heads, a.q_dtype, a.max_pages, a.table_stride = 1, 1, 4, 12, 1, 1
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.b200_cache_attention(ref, ctypes.byref(a), None)

    for kw in (dict(q_dtype=14), dict(heads=3), dict(heads=0), dict(batch=-1), dict(max_pages=-1), dict(prefix_length=1),
               dict(q=None), dict(out=4100), dict(lengths=None), dict(tables=None), dict(prefix_pages=1, prefix_length=17)):
        assert attention(**kw) == _lib.ERR_INVALID, kw
    assert attention(max_pages=2 ** 31) == _lib.ERR_UNSUPPORTED
    assert attention(batch=0) == 0 and attention(queries=0) == 0
    assert lib.b200_cache_attention(ref, None, None) == _lib.ERR_INVALID
    assert lib.b200_cache_read(ref, None, 6, 1, None, None, 12, None) == _lib.ERR_INVALID
    assert lib.b200_cache_read(ref, None, 12, 0, None, None, 12, None) == _lib.ERR_INVALID
    assert lib.b200_cache_read(ref, None, 6, 0, None, None, 2, None) == _lib.ERR_INVALID
    assert lib.b200_cache_write(ref, None, 0, 0, None, 0, 0, 12, -1, None, 6, None, None, 0, None, 0, 0, 0, None, None) == _lib.ERR_INVALID
    assert lib.b200_cache_write(ref, None, 0, 0, None, 0, 0, 12, 1, None, 6, None, None, 0, None, 0, 0, 0, None, None) == _lib.ERR_INVALID
    t = A.RotaryDesc(4096, 4096, 10, 66, 0)
    assert lib.b200_rotary(4096, 12, 1, 1, 1, 64, 0, 0, 0, 4096, 0, 0, 0, ctypes.byref(t), 4096, 6, 0, None) == _lib.ERR_INVALID
    assert "rotary_dim" in _lib.last_error()
    assert lib.b200_rotary(4096, 12, 1, 1, 1, 64, 0, 0, 0, 4096, 0, 0, 0, None, 4096, 6, 0, None) == _lib.ERR_INVALID
    assert lib.b200_rotary(None, 12, 0, 1, 1, 64, 0, 0, 0, None, 0, 0, 0, None, None, 6, 0, None) == 0
    assert lib.b200_cache_attention_scratch(2, 3, 4, 64, 10) == 2 * 3 * 4 * 66 * 4
    assert lib.b200_cache_attention_scratch(2, 3, 4, 64, 0) == 0


def test_c_entries_of_captures():
    lib = _lib.lib()
    assert lib.b200_capture_release(0) == 0 and lib.b200_capture_release(12345) == 0
    assert lib.b200_capture_id(None, None) == _lib.ERR_INVALID and "null" in _lib.last_error()
    n = ctypes.c_uint64(7)
    assert lib.b200_capture_id(None, ctypes.byref(n)) == 0 and n.value == 0  # the legacy stream is never captured
