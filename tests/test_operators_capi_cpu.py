"""The cache's, cached attention's and token scores' entry points on a host without a GPU: arguments are checked before the
first HIP call."""

import ctypes

import numpy as np
import pytest

from dirktensor_amd import _capi as C

FAKE = 0x10000  # aligned non-NULL address; never dereferenced because validation fails first


def error():
    return C.lib().dt_last_error().decode()


def refused(rc, code, msg):
    assert rc == code and msg in error(), (rc, error())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(D=64), C.DT_ERR_UNSUPPORTED, "head_dim"),
    (dict(slots=0), C.DT_ERR_INVALID_ARG, "slots"),
    (dict(capacity=0), C.DT_ERR_INVALID_ARG, "capacity"),
    (dict(capacity=(1 << 20) + 1), C.DT_ERR_INVALID_ARG, "capacity"),
    (dict(heads=0), C.DT_ERR_INVALID_ARG, "n_heads"),
    (dict(fmt=3), C.DT_ERR_INVALID_ARG, "format"),
    ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL"),
])
def test_cache_create(kw, code, msg):
    a = dict(ctx=None, slots=1, capacity=8, heads=2, D=128, fmt=C.DT_KV_INT8)
    a.update(kw)
    h = ctypes.c_void_p()
    refused(C.lib().dt_kv_cache_create(*a.values(), ctypes.byref(h)), code, msg)
    assert not h


@pytest.mark.parametrize("kw,code,msg", [
    (dict(k=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(B=0), C.DT_ERR_INVALID_ARG, "B=0"),
    (dict(B=257), C.DT_ERR_UNSUPPORTED, "B=257"),
    (dict(T=0), C.DT_ERR_INVALID_ARG, "tokens"),
    (dict(dtype=4), C.DT_ERR_INVALID_ARG, "dtype"),
    (dict(mem=4), C.DT_ERR_INVALID_ARG, "mem"),
    (dict(v=FAKE + 8), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(ldk=260), C.DT_ERR_INVALID_ARG, "aligned"),
    ({}, C.DT_ERR_INVALID_ARG, "cache is NULL"),
])
def test_cache_append(kw, code, msg):
    a = dict(cache=None, k=FAKE, v=FAKE, B=1, T=4, ldk=256, ldv=256, slots=None, counts=None, dtype=C.DT_BF16,
             mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_kv_cache_append(*a.values()), code, msg)


def test_cache_read_lengths_truncate_destroy():
    lib = C.lib()
    refused(lib.dt_kv_cache_read(None, None, FAKE, 1, 1, None, None, 0, 0, None), C.DT_ERR_INVALID_ARG, "non-NULL")
    refused(lib.dt_kv_cache_read(None, FAKE, FAKE, 1, 0, None, None, 0, 0, None), C.DT_ERR_INVALID_ARG, "tokens")
    refused(lib.dt_kv_cache_read(None, FAKE, FAKE + 4, 1, 1, None, None, 0, 0, None), C.DT_ERR_INVALID_ARG, "aligned")
    refused(lib.dt_kv_cache_read(None, FAKE, FAKE, 1, 1, None, None, 0, 0, None), C.DT_ERR_INVALID_ARG, "cache is NULL")
    n = np.zeros(1, np.int32)
    refused(lib.dt_kv_cache_lengths(None, n.ctypes.data), C.DT_ERR_INVALID_ARG, "cache is NULL")
    refused(lib.dt_kv_cache_truncate(None, 1, None, None), C.DT_ERR_INVALID_ARG, "lengths is NULL")
    refused(lib.dt_kv_cache_truncate(None, 0, None, n.ctypes.data), C.DT_ERR_INVALID_ARG, "B=0")
    refused(lib.dt_kv_cache_truncate(None, 1, None, n.ctypes.data), C.DT_ERR_INVALID_ARG, "cache is NULL")
    assert lib.dt_kv_cache_destroy(None) == C.DT_OK


@pytest.mark.parametrize("kw,code,msg", [
    (dict(q=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(mem=2), C.DT_ERR_INVALID_ARG, "mem"),
    (dict(scale=-1.0), C.DT_ERR_INVALID_ARG, "scale"),
    (dict(scale=float("nan")), C.DT_ERR_INVALID_ARG, "scale"),
    (dict(causal=2), C.DT_ERR_INVALID_ARG, "causal"),
    (dict(D=96), C.DT_ERR_UNSUPPORTED, "head_dim"),
    (dict(B=0), C.DT_ERR_INVALID_ARG, ">= 1"),
    (dict(B=257), C.DT_ERR_UNSUPPORTED, "B=257"),
    (dict(T=8193), C.DT_ERR_INVALID_ARG, "max_seq_len"),
    (dict(dtype=2), C.DT_ERR_INVALID_ARG, "dtype"),
    ({}, C.DT_ERR_INVALID_ARG, "cache is NULL"),
])
def test_cached_attn(kw, code, msg):
    a = dict(cache=None, q=FAKE, o=FAKE, m=None, l=None, B=1, T=1, H=2, D=128, ldq=256, scale=0.1, causal=1, slots=None,
             counts=None, prefix=None, prefix_slot=0, ws=None, ws_bytes=0, dtype=C.DT_BF16, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_cached_attn_fwd(*a.values()), code, msg)


def test_cached_attn_workspace():
    n = ctypes.c_int64()
    lib = C.lib()
    refused(lib.dt_cached_attn_workspace(None, 1, 1, 2, 128, None, None, None, 0, 0, None), C.DT_ERR_INVALID_ARG, "bytes")
    refused(lib.dt_cached_attn_workspace(None, 1, 1, 2, 128, None, None, None, 0, 0, ctypes.byref(n)), C.DT_ERR_INVALID_ARG,
            "cache is NULL")
