"""Refusals of the 8-bit KV cache operators that need no GPU, and their plain forms' own rules."""
import ctypes
import math

import pytest
import torch

import _kv8
from flash_attn_triton import (_native, flash_attn_with_kvcache_8bit, kvcache_append_8bit,
                               paged_kvcache_slots)


def _cache(pages=2, page=32, block=16, heads=2, dim=64, store=torch.float8_e4m3fn):
    c = torch.zeros(pages, page, heads, dim).to(store)
    s = torch.zeros(pages, page // block, heads, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return c, c.clone(), s, s.clone()


@pytest.mark.parametrize("change,match", [
    (dict(dim=32), "head dimension"), (dict(block=8), "scale block"), (dict(page=48, block=48), "scale block"),
    (dict(store=torch.float16), "float8_e4m3fn"), ({}, "CUDA"),
])
def test_cache_shapes(change, match):
    c = _cache(**change)
    heads, dim = c[0].shape[2:]
    rows = torch.zeros(3, heads, dim).half()
    with pytest.raises(ValueError, match=match):
        kvcache_append_8bit(rows, rows, *c, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match=match):
        flash_attn_with_kvcache_8bit(torch.zeros(1, 1, heads, dim).half(), *c)


def test_cache_tensors_must_match():
    kc, vc, ks, vs = _cache()
    q = torch.zeros(1, 1, 2, 64).half()
    with pytest.raises(ValueError, match="same shape"):
        flash_attn_with_kvcache_8bit(q, kc, vc[:1], ks, vs)
    with pytest.raises(ValueError, match="both float8"):
        flash_attn_with_kvcache_8bit(q, kc, vc.float().to(torch.float8_e5m2), ks, vs)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        flash_attn_with_kvcache_8bit(q, kc, vc, ks.view(torch.uint8), vs)
    with pytest.raises(ValueError, match="must have shape"):
        flash_attn_with_kvcache_8bit(q, kc, vc, ks[:, :, :1], vs[:, :, :1])


def test_queries_and_rows():
    c = _cache()
    with pytest.raises(ValueError, match="FP16 or BF16"):
        flash_attn_with_kvcache_8bit(torch.zeros(1, 1, 2, 64), *c)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        flash_attn_with_kvcache_8bit(torch.zeros(1, 2, 64).half(), *c)
    with pytest.raises(ValueError, match="tokens, nheads_k, headdim"):
        kvcache_append_8bit(torch.zeros(1, 1, 2, 64), torch.zeros(1, 1, 2, 64), *c, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="FP16, BF16 or FP32"):
        kvcache_append_8bit(torch.zeros(1, 2, 64).half(), torch.zeros(1, 2, 64), *c, torch.zeros(1, dtype=torch.int64))


def test_strides_that_share_memory():
    from flash_attn_triton.kvcache_8bit import _apart
    assert _apart((2, 3, 4), (12, 4, 1), (1, 8, 2), (100, 4, 1)) and _apart((1, 3, 1), (0, 1, 0)) and _apart((2, 0), (0, 1))
    assert not _apart((2, 3, 4), (0, 4, 1)) and not _apart((2, 3, 4), (12, 3, 1)) and not _apart((2, 2), (1, 1))


def test_slots_arguments():
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32 tensor of shape"):
        paged_kvcache_slots(torch.zeros(1, 2, dtype=torch.int64), one, one, one, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        paged_kvcache_slots(torch.zeros(1, 2, dtype=torch.int32), one, one, one, 16, 4)


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def _error(lib):
    return lib.fa_last_error_string().decode()


def test_c_slots_checks(lib):
    one = ctypes.c_void_p(16)   # never dereferenced

    def call(batch=1, cols=2, n_free=1, page=16, rows=4, stride=2, table=one, slots=one):
        return lib.fa_kvcache_slots(table, stride, cols, one, one, batch, one, n_free, None, page, rows, slots, one, one,
                                    one, one, None)
    assert call(page=0) == _native.FA_ERR_INVALID
    assert call(batch=-1) == _native.FA_ERR_INVALID
    assert call(table=None) == _native.FA_ERR_INVALID and "null" in _error(lib)
    assert call(slots=None) == _native.FA_ERR_INVALID
    assert call(batch=2, stride=1) == _native.FA_ERR_INVALID and "overlap" in _error(lib)
    assert call(cols=1 << 20, page=1 << 20, stride=1 << 20) == _native.FA_ERR_UNSUPPORTED


def test_c_append_checks(lib):
    one, st = ctypes.c_void_p(16), _native._strides((1024, 512, 64))

    def call(k=one, dtype=0, store=0, tokens=1, pages=1, page=32, block=16, heads=1, dim=64, strides=st):
        return lib.fa_kvcache8_append(k, one, strides, strides, dtype, one, one, st, st, store, one, one, st, st, one,
                                      tokens, pages, page, block, heads, dim, None)
    assert call(store=2) == _native.FA_ERR_UNSUPPORTED
    assert call(block=24) == _native.FA_ERR_UNSUPPORTED
    assert call(block=8) == _native.FA_ERR_UNSUPPORTED
    assert call(page=24) == _native.FA_ERR_INVALID
    assert call(dim=32) == _native.FA_ERR_UNSUPPORTED
    assert call(dtype=3) == _native.FA_ERR_UNSUPPORTED
    assert call(k=None) == _native.FA_ERR_INVALID
    assert call(strides=_native._strides((1024, 516, 0))) == _native.FA_ERR_INVALID and "aligned" in _error(lib)
    assert call(pages=1 << 31) == _native.FA_ERR_UNSUPPORTED
    assert call(tokens=0) == _native.FA_OK


def test_c_attention_checks(lib):
    one, st = ctypes.c_void_p(16), _native._strides((4096, 1024, 64))

    def call(q=one, dtype=0, store=0, table=one, cols=4, pages=8, page=32, block=16, cu=None, batch=2, max_q=1, total=2,
             max_keys=128, hq=2, hk=1, dim=64, less=0, ws=one, kst=st, softcap=0.0):
        need = ctypes.c_int64(0)
        lib.fa_fwd_kvcache8_plan(batch, max_q, total, hq, hk, dim, max_keys, ctypes.byref(need))
        return lib.fa_fwd_kvcache8(q, one, st, st, dtype, one, one, kst, kst, store, one, one, st, st, one, table, 4, cols,
                                   pages, page, block, cu, batch, max_q, total, max_keys, hq, hk, dim, 1.0, 1, -1, -1,
                                   softcap, None, 0, ws, need.value - less, None)
    assert call(q=None) == _native.FA_ERR_INVALID
    assert call(dtype=2) == _native.FA_ERR_UNSUPPORTED
    assert call(max_keys=129) == _native.FA_ERR_INVALID and "block table" in _error(lib)
    assert call(table=None, max_keys=33) == _native.FA_ERR_INVALID
    assert call(total=3) == _native.FA_ERR_INVALID
    assert call(hq=3, hk=2) == _native.FA_ERR_INVALID
    assert call(cols=40, max_keys=1280, less=4) == _native.FA_ERR_INVALID and "plan" in _error(lib)
    assert call(cols=40, max_keys=1280, ws=None) == _native.FA_ERR_INVALID
    assert call(softcap=-1.0) == _native.FA_ERR_INVALID
    assert call(softcap=math.nan) == _native.FA_ERR_INVALID
    assert call(kst=_native._strides((4096, 32, 64))) == _native.FA_ERR_UNSUPPORTED and "overlap" in _error(lib)
    assert call(kst=_native._strides((4096, 1 << 27, 64))) == _native.FA_ERR_UNSUPPORTED
    assert call(batch=0, total=0) == _native.FA_OK


def test_plan_of_the_workspace(lib):
    def plan(*args):
        need = ctypes.c_int64(-1)
        assert lib.fa_fwd_kvcache8_plan(*args, ctypes.byref(need)) == _native.FA_OK
        return need.value
    # stretches of single tokens: a row per sequence and stretch, K/V head and query head, its sum, and the starts
    assert plan(64, 1, 64, 32, 8, 128, 8192) == (64 + 64) * 32 * 129 * 4 + 66 * 4
    # however long, and whatever the number of sequences
    assert plan(1, 1, 1, 32, 8, 128, 1 << 20) == (1 + 64) * 32 * 129 * 4 + 3 * 4
    assert plan(5000, 1, 5000, 32, 8, 128, 8192) == (256 + 64) * 32 * 129 * 4 + 258 * 4
    assert plan(64, 1, 64, 32, 8, 128, 512) == 0
    # chunks: whole rows of q, for each split
    assert plan(4, 512, 2048, 32, 8, 128, 8192) == 0
    assert plan(1, 40, 40, 16, 4, 64, 4000) % (40 * 16 * 65 * 4) == 0


def test_scale_rule():
    # the least power of two that holds the number, at and around the type's largest
    for store, top in ((torch.float8_e4m3fn, 448.0), (torch.float8_e5m2, 57344.0)):
        for j in (-20, 0, 7):
            assert _kv8.scale_of(top * 2.0 ** j, store) == 127 + j
            assert _kv8.scale_of(math.nextafter(top * 2.0 ** j, math.inf), store) == 128 + j
            assert _kv8.scale_of(top * 2.0 ** (j - 1) * 1.01, store) == 127 + j
