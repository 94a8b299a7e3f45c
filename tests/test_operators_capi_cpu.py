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


@pytest.mark.parametrize("kw,code,msg", [
    (dict(logits=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(m=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(B=0), C.DT_ERR_INVALID_ARG, ">= 1"),
    (dict(V=(1 << 24) + 1), C.DT_ERR_UNSUPPORTED, "V="),
    (dict(T=1 << 24), C.DT_ERR_UNSUPPORTED, "rows"),
    (dict(ldt=-1), C.DT_ERR_INVALID_ARG, "strides"),
    (dict(token_bytes=2), C.DT_ERR_INVALID_ARG, "token_bytes"),
    (dict(top_k=65), C.DT_ERR_INVALID_ARG, "top_k"),
    (dict(top_k=3, top_index=None), C.DT_ERR_INVALID_ARG, "top_index"),
    (dict(logits=FAKE + 2), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(ws=FAKE + 8), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(tokens=FAKE + 4, token_bytes=8), C.DT_ERR_INVALID_ARG, "tokens are not aligned"),
    (dict(V=100352, ws=None), C.DT_ERR_INVALID_ARG, "the workspace has 0"),
    (dict(dtype=9), C.DT_ERR_INVALID_ARG, "dtype"),
    (dict(mem=9), C.DT_ERR_INVALID_ARG, "mem"),
    ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL"),
])
def test_token_logprobs(kw, code, msg):
    a = dict(ctx=None, logits=FAKE, tokens=FAKE, B=1, T=1, V=100, ldb=0, ldt=0, token_bytes=4, ignore=C.DT_NO_IGNORE, top_k=0,
             logprob=FAKE, entropy=None, m=FAKE, l=FAKE, top_index=FAKE, top_logprob=FAKE, ws=FAKE, ws_bytes=0,
             dtype=C.DT_FP32_EXACT, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_token_logprobs(*a.values()), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(g=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(h=FAKE, entropy=None), C.DT_ERR_INVALID_ARG, "entropy"),
    (dict(T=2, ldt_out=99), C.DT_ERR_INVALID_ARG, "overlap"),
    (dict(B=2, T=2, ldt_out=100, ldb_out=199), C.DT_ERR_INVALID_ARG, "overlap"),
    (dict(dx=FAKE + 1), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(token_bytes=0), C.DT_ERR_INVALID_ARG, "token_bytes"),
    ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL"),
])
def test_token_logprobs_bwd(kw, code, msg):
    a = dict(ctx=None, g=FAKE, h=None, logits=FAKE, tokens=FAKE, m=FAKE, l=FAKE, entropy=FAKE, B=1, T=1, V=100, ldb=0, ldt=0,
             token_bytes=4, ignore=0, dx=FAKE, ldb_out=0, ldt_out=0, dtype=C.DT_BF16, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_token_logprobs_bwd(*a.values()), code, msg)


def test_token_logprobs_host_tokens_are_checked():
    tok = np.array([3, 100], np.int64)
    args = [None, FAKE, tok.ctypes.data, 1, 2, 100, 200, 100, 8, C.DT_NO_IGNORE, 0, FAKE, None, FAKE, FAKE, None, None, None, 0, 0,
            C.DT_MEM_HOST, None]
    refused(C.lib().dt_token_logprobs(*args), C.DT_ERR_INVALID_ARG, "token 100 of row 1")
    args[9] = 100  # ignored
    refused(C.lib().dt_token_logprobs(*args), C.DT_ERR_INVALID_ARG, "ctx is NULL")


def test_token_logprobs_workspace():
    n = ctypes.c_int64(-1)
    lib = C.lib()
    assert lib.dt_token_logprobs_workspace(2048, 2, 100352, 5, ctypes.byref(n)) == C.DT_OK and n.value == 0  # rows enough
    assert lib.dt_token_logprobs_workspace(1, 1, 100352, 20, ctypes.byref(n)) == C.DT_OK and n.value > 0
    refused(lib.dt_token_logprobs_workspace(1, 1, 10, 11, ctypes.byref(n)), C.DT_ERR_INVALID_ARG, "top_k")
    refused(lib.dt_token_logprobs_workspace(1, 1, 10, 1, None), C.DT_ERR_INVALID_ARG, "bytes")


def test_leading_dimensions_as_two_strides():
    from dirktensor_amd.logprobs import _two_strides

    assert _two_strides((), ()) == (1, 1, 0, 0)
    assert _two_strides((5,), (7,)) == (1, 5, 0, 7)
    assert _two_strides((3, 5), (35, 7)) == (1, 15, 0, 7)
    assert _two_strides((3, 5), (42, 7)) == (3, 5, 42, 7)
    assert _two_strides((3, 1, 5), (42, 9, 7)) == (3, 5, 42, 7)
    assert _two_strides((2, 3, 5), (105, 35, 7)) == (1, 30, 0, 7)
    assert _two_strides((2, 3, 5), (126, 42, 7)) == (6, 5, 42, 7)
    assert _two_strides((2, 3, 5), (200, 42, 7)) is None
    assert _two_strides((4, 5), (0, 7)) == (4, 5, 0, 7)


def test_kernels_use_no_scratch_memory():
    """Scratch memory would be allocated at a kernel's first launch, at the latest: a captured call cannot have that."""
    from test_kernel_scratch_cpu import _code_objects, _kernels

    import dirktensor_amd as dt

    if not dt.LIB_PATH.exists():
        pytest.skip("the library is not built")
    sizes = {k[".name"]: (k[".private_segment_fixed_size"], bool(k.get(".uses_dynamic_stack")))
             for elf in _code_objects(dt.LIB_PATH.read_bytes()) for k in _kernels(elf)}
    mine = {n: s for n, s in sizes.items() if any(x in n for x in ("cached_attn", "kv_append", "kv_read", "logprob"))}
    assert len(mine) >= 40, sorted(mine)
    assert {n: s for n, s in mine.items() if s != (0, False)} == {}
