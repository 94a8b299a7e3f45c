"""The cache's format in 4 bits on a host without a GPU."""

import ctypes

from dirktensor_amd import _capi as C


def test_the_format_is_known():
    h = ctypes.c_void_p()
    rc = C.lib().dt_kv_cache_create(None, 1, 8, 2, 128, C.DT_KV_FP4, ctypes.byref(h))
    assert rc == C.DT_ERR_INVALID_ARG and "ctx is NULL" in C.lib().dt_last_error().decode() and not h
