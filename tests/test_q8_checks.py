"""Refusals of 8-bit KV pools that come before any GPU call."""

import ctypes

import pytest
import torch

from flint_amd import KvPool, ThubanError, _lib, ops


class _Pool:
    """Only what the checks read from a KvPool (no device memory)."""

    kv_heads, head_dim, handle, _hd_arr, kv_dtype = 2, 64, 0, None, "e4m3"


class _Rows:
    handle = 0


def _raises(fn, text):
    with pytest.raises(ThubanError) as e:
        fn()
    assert text in str(e.value), str(e.value)


def test_kv_load_rejects_bad_buffers():
    pool = _Pool()
    k = torch.zeros(3, 2, 64)
    _raises(lambda: ops.kv_load(k[:2], k, pool, 0, 3, _Rows()), "k_dst holds 256 elements, the call needs 384")
    _raises(lambda: ops.kv_load(k, k[:, :1], pool, 0, 3, _Rows()), "v_dst must be contiguous")
    _raises(lambda: ops.kv_load(k, k.half(), pool, 0, 3, _Rows()), "dtypes differ")
    _raises(lambda: ops.kv_load(k.int(), k, pool, 0, 3, _Rows()), "k_dst: dtype int32")
    _raises(lambda: ops.kv_load(k, k, pool, 0, 3, _Rows()), "must be a GPU tensor")


def test_kv_load_c_entry_rejects_null():
    rc = _lib.lib().thb_kv_load(None, 0, 16, 16, 0, None, 0, 1, None)
    assert rc == _lib.THB_ERR_INVALID


def _desc(page_len, kv_dtype=_lib.KV_E4M3, head_dim=128, part_len=0):
    d = _lib.PoolDesc()
    lens = (ctypes.c_uint32 * 1)(64)
    d.layers, d.kv_heads, d.head_dim, d.pages = 1, 1, head_dim, 8
    d.page_len, d.kv_dtype, d.part_len = page_len, kv_dtype, part_len
    d.seqs, d.seq_lens = 1, lens
    return d, lens


@pytest.mark.parametrize("page_len,kv_dtype,text", [
    (8, _lib.KV_E4M3, "at least 16 in an 8-bit pool"),
    (24, _lib.KV_E4M3, "power of two"),
    (512, _lib.KV_E4M3, "power of two"),
    (16, 3, "unknown kv_dtype 3"),
])
def test_pool_create_refuses(page_len, kv_dtype, text):
    d, keep = _desc(page_len, kv_dtype)
    h = ctypes.c_void_p()
    rc = _lib.lib().thb_pool_create(ctypes.byref(d), ctypes.byref(h))
    assert rc == _lib.THB_ERR_CONFIG and not h.value
    with pytest.raises(ThubanError) as e:
        _lib.check(rc)
    assert text in str(e.value)


def test_unknown_pool_type_name():
    with pytest.raises((KeyError, ThubanError)):
        KvPool(None, kv_heads=1, head_dim=64, layers=1, page_len=16, kv_dtype="e5m2")
