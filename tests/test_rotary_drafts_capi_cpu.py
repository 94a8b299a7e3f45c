"""The rotary's and the verified drafts' entry points on a host without a GPU: frequencies, and arguments that are checked before the
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


def rotary(**kw):
    a = dict(dims=128, layout=0, theta=500000.0, scaling=0, factor=1.0, original=8192.0, low=1.0, high=32.0, magnitude=1.0)
    a.update(kw)
    r = C.DTRotary()
    return r, C.lib().dt_rotary_init(ctypes.addressof(r), *a.values())


@pytest.mark.parametrize("dims", [16, 48, 128])
@pytest.mark.parametrize("scaling", [C.DT_ROTARY_UNSCALED, C.DT_ROTARY_LINEAR, C.DT_ROTARY_THETA, C.DT_ROTARY_RAMP])
def test_frequencies(dims, scaling):
    r, rc = rotary(dims=dims, scaling=scaling, factor=8.0, theta=10000.0, magnitude=1.5)
    assert rc == C.DT_OK and (r.dims, r.layout, r.magnitude) == (dims, 0, 1.5)
    f = np.array(r.frequency[:dims // 2])
    plain = 10000.0 ** (-np.arange(0, dims, 2) / dims)
    if scaling == C.DT_ROTARY_UNSCALED:
        want = plain
    elif scaling == C.DT_ROTARY_LINEAR:
        want = plain / 8
    elif scaling == C.DT_ROTARY_THETA:
        want = plain * 8.0 ** (-np.arange(dims // 2) / (dims // 2 - 1))
    else:
        turns = plain * 8192 / (2 * np.pi)
        want = plain * np.interp(turns, [1, 32], [1 / 8, 1])
    np.testing.assert_allclose(f, want, rtol=1e-13)
    assert all(v == 0 for v in r.frequency[dims // 2:])


@pytest.mark.parametrize("kw,msg", [
    (dict(dims=0), "dims"), (dict(dims=24), "dims"), (dict(dims=144), "dims"), (dict(layout=2), "layout"), (dict(scaling=4), "scaling"),
    (dict(theta=1.0), "theta"), (dict(theta=float("inf")), "theta"), (dict(scaling=1, factor=0.5), "factor"),
    (dict(scaling=3, factor=2.0, low=4.0, high=4.0), "low"), (dict(scaling=3, factor=2.0, original=0.0), "ramp"),
    (dict(magnitude=0.0), "magnitude"), (dict(magnitude=float("nan")), "magnitude"), (dict(magnitude=1e39), "magnitude"), (dict(magnitude=1e-60), "magnitude"), (dict(scaling=2, factor=1e300), "theta"),
])
def test_rotary_init_refusals(kw, msg):
    refused(rotary(**kw)[1], C.DT_ERR_INVALID_ARG, msg)


def test_rotary_init_null():
    refused(C.lib().dt_rotary_init(None, 128, 0, 1e4, 0, 1.0, 1.0, 1.0, 2.0, 1.0), C.DT_ERR_INVALID_ARG, "rotary is NULL")


ROWS = [
    (dict(B=0), C.DT_ERR_INVALID_ARG, "B=0"), (dict(T=0), C.DT_ERR_INVALID_ARG, "T=0"), (dict(H=0), C.DT_ERR_INVALID_ARG, "H=0"),
    (dict(Hk=-1), C.DT_ERR_INVALID_ARG, "Hk=-1"), (dict(q=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(k=None), C.DT_ERR_INVALID_ARG, "non-NULL"), (dict(rot=None), C.DT_ERR_INVALID_ARG, "rotary is NULL"),
    (dict(D=64), C.DT_ERR_UNSUPPORTED, "head_dim"), (dict(H=1000, Hk=25), C.DT_ERR_UNSUPPORTED, "heads"),
    (dict(B=1 << 20, T=1 << 20), C.DT_ERR_UNSUPPORTED, "tokens"), (dict(dtype=5), C.DT_ERR_INVALID_ARG, "dtype"),
    (dict(mem=5), C.DT_ERR_INVALID_ARG, "mem"), (dict(positions=FAKE, starts=FAKE), C.DT_ERR_INVALID_ARG, "exclude"),
    (dict(positions=FAKE, pos_bytes=2), C.DT_ERR_INVALID_ARG, "pos_bytes"), (dict(positions=FAKE + 4, pos_bytes=8), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(B=257, starts=FAKE), C.DT_ERR_UNSUPPORTED, "starts"), (dict(ldq=255), C.DT_ERR_INVALID_ARG, "strides"),
    (dict(ldko=127), C.DT_ERR_INVALID_ARG, "strides"), (dict(ldq=260), C.DT_ERR_INVALID_ARG, "aligned"), (dict(oq=FAKE + 8), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(ok=FAKE), C.DT_ERR_INVALID_ARG, "the other"), (dict(oq=FAKE + 4096, ok=FAKE + 8192), C.DT_ERR_INVALID_ARG, "the other"),
    (dict(ldqo=264), C.DT_ERR_INVALID_ARG, "same stride"), (dict(ldko=136), C.DT_ERR_INVALID_ARG, "same stride"),
    (dict(T=1, ldqo=264), C.DT_ERR_INVALID_ARG, "ctx is NULL"), ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL"),
]


@pytest.mark.parametrize("kw,code,msg", ROWS + [(dict(backward=2), C.DT_ERR_INVALID_ARG, "backward")])
def test_rotary_fwd(kw, code, msg):
    r, _ = rotary()
    a = dict(ctx=None, q=FAKE, k=FAKE + 4096, oq=FAKE, ok=FAKE + 4096, B=1, T=4, H=2, Hk=1, D=128, ldq=256, ldk=128, ldqo=256, ldko=128, positions=None,
             pos_bytes=4, starts=None, rot=ctypes.addressof(r), backward=0, dtype=C.DT_BF16, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_rotary_fwd(*a.values()), code, msg)


def test_a_rotary_filled_by_hand_is_checked():
    for field, value in (("dims", 8), ("dims", 130), ("layout", 7), ("magnitude", -1.0)):
        r, _ = rotary()
        setattr(r, field, value)
        refused(C.lib().dt_rotary_fwd(None, FAKE, None, FAKE, None, 1, 1, 1, 0, 128, 128, 0, 128, 0, None, 0, None, ctypes.addressof(r), 0, 0, 0,
                                      None), C.DT_ERR_INVALID_ARG, "dims")
    r, _ = rotary()
    r.frequency[3] = float("nan")
    refused(C.lib().dt_rotary_fwd(None, FAKE, None, FAKE, None, 1, 1, 1, 0, 128, 128, 0, 128, 0, None, 0, None, ctypes.addressof(r), 0, 0, 0, None),
            C.DT_ERR_INVALID_ARG, "finite")


@pytest.mark.parametrize("kw,code,msg", ROWS + [
    (dict(wq=None), C.DT_ERR_INVALID_ARG, "weights"), (dict(wk=None), C.DT_ERR_INVALID_ARG, "weights"), (dict(wk=FAKE + 4), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(eps=0.0), C.DT_ERR_INVALID_ARG, "eps"), (dict(eps=float("inf")), C.DT_ERR_INVALID_ARG, "eps")])
def test_head_norm_fwd(kw, code, msg):
    r, _ = rotary()
    a = dict(ctx=None, q=FAKE, k=FAKE + 4096, wq=FAKE, wk=FAKE + 4096, oq=FAKE, ok=FAKE + 4096, B=1, T=4, H=2, Hk=1, D=128, ldq=256, ldk=128, ldqo=256, ldko=128,
             positions=None, pos_bytes=4, starts=None, rot=ctypes.addressof(r), eps=1e-6, dtype=C.DT_BF16, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_head_norm_rotary_fwd(*a.values()), code, msg)


@pytest.mark.parametrize("kw,code,msg", [r for r in ROWS if "ctx" not in r[2]] + [
    (dict(xq=None), C.DT_ERR_INVALID_ARG, "forward's inputs"), (dict(dwk=None), C.DT_ERR_INVALID_ARG, "forward's inputs"),
    (dict(ldxk=64), C.DT_ERR_INVALID_ARG, "strides"), (dict(ldxk=136), C.DT_ERR_INVALID_ARG, "same stride"), (dict(xk=FAKE + 8), C.DT_ERR_INVALID_ARG, "aligned"), ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL")])
def test_head_norm_bwd(kw, code, msg):
    r, _ = rotary()
    a = dict(ctx=None, q=FAKE, k=FAKE + 4096, xq=FAKE, xk=FAKE + 4096, wq=FAKE, wk=FAKE + 4096, oq=FAKE, ok=FAKE + 4096, dwq=FAKE, dwk=FAKE, B=1, T=4, H=2, Hk=1, D=128, ldq=256,
             ldk=128, ldxq=256, ldxk=128, ldqo=256, ldko=128, positions=None, pos_bytes=4, starts=None, rot=ctypes.addressof(r), eps=1e-6, ws=FAKE,
             ws_bytes=1 << 30, dtype=C.DT_BF16, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_head_norm_rotary_bwd(*a.values()), code, msg)


def test_workspaces():
    n = ctypes.c_int64(-1)
    lib = C.lib()
    assert lib.dt_head_norm_rotary_bwd_workspace(1, 1, 1, 0, ctypes.byref(n)) == C.DT_OK and n.value >= 512
    refused(lib.dt_head_norm_rotary_bwd_workspace(1, 1, 1, 0, None), C.DT_ERR_INVALID_ARG, "bytes")
    refused(lib.dt_head_norm_rotary_bwd_workspace(0, 1, 1, 0, ctypes.byref(n)), C.DT_ERR_INVALID_ARG, "B=0")
    refused(lib.dt_head_norm_rotary_bwd_workspace(1, 1, 2**31 - 1, 2**31 - 1, ctypes.byref(n)), C.DT_ERR_UNSUPPORTED, "heads")
    refused(lib.dt_head_norm_rotary_bwd_workspace(1 << 20, 1 << 20, 16, 16, ctypes.byref(n)), C.DT_ERR_UNSUPPORTED, "tokens")
    assert lib.dt_verify_drafts_workspace(4, 3, 1000, 1, 1.0, ctypes.byref(n)) == C.DT_OK and n.value > 0
    refused(lib.dt_verify_drafts_workspace(4, 3, 1000, 1, 1.0, None), C.DT_ERR_INVALID_ARG, "bytes")
    refused(lib.dt_verify_drafts_workspace(4, 65, 1000, 1, 1.0, ctypes.byref(n)), C.DT_ERR_UNSUPPORTED, "K=65")


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=0), C.DT_ERR_INVALID_ARG, "B=0"), (dict(B=257), C.DT_ERR_UNSUPPORTED, "B=257"), (dict(K=-1), C.DT_ERR_INVALID_ARG, "K=-1"),
    (dict(K=65), C.DT_ERR_UNSUPPORTED, "K=65"), (dict(V=0), C.DT_ERR_INVALID_ARG, "V=0"), (dict(V=(1 << 24) + 1), C.DT_ERR_UNSUPPORTED, "V="),
    (dict(temperature=-0.5), C.DT_ERR_INVALID_ARG, "temperature"), (dict(temperature=float("inf")), C.DT_ERR_INVALID_ARG, "temperature"),
    (dict(logits=None), C.DT_ERR_INVALID_ARG, "non-NULL"), (dict(drafts=None), C.DT_ERR_INVALID_ARG, "non-NULL"),
    (dict(tokens=None), C.DT_ERR_INVALID_ARG, "non-NULL"), (dict(uniforms=None), C.DT_ERR_INVALID_ARG, "uniforms"),
    (dict(dtype=3), C.DT_ERR_INVALID_ARG, "dtype"), (dict(mem=3), C.DT_ERR_INVALID_ARG, "mem"), (dict(token_bytes=2), C.DT_ERR_INVALID_ARG, "token_bytes"),
    (dict(ldt=-1), C.DT_ERR_INVALID_ARG, "strides"), (dict(ldb_draft=-4), C.DT_ERR_INVALID_ARG, "strides"), (dict(ldb=1 << 60), C.DT_ERR_INVALID_ARG, "strides"),
    (dict(logits=FAKE + 2), C.DT_ERR_INVALID_ARG, "aligned"), (dict(drafts=FAKE + 4, token_bytes=8), C.DT_ERR_INVALID_ARG, "aligned"),
    (dict(ws=FAKE + 8), C.DT_ERR_INVALID_ARG, "workspace"), (dict(ws_bytes=16), C.DT_ERR_INVALID_ARG, "the call needs"),
    (dict(ws=None), C.DT_ERR_INVALID_ARG, "the workspace has 0"), ({}, C.DT_ERR_INVALID_ARG, "ctx is NULL"),
])
def test_verify_drafts(kw, code, msg):
    a = dict(ctx=None, logits=FAKE, drafts=FAKE, uniforms=FAKE, draft_logits=FAKE, B=2, K=3, V=100, ldb=400, ldt=100, ldb_draft=300, ldt_draft=100,
             token_bytes=4, counts=None, temperature=1.0, accepted=FAKE, tokens=FAKE, logprob=FAKE, ws=FAKE, ws_bytes=1 << 30,
             dtype=C.DT_FP32_EXACT, mem=C.DT_MEM_DEVICE, stream=None)
    a.update(kw)
    refused(C.lib().dt_verify_drafts(*a.values()), code, msg)


def test_verify_drafts_host_arguments_are_checked():
    counts = np.array([3, 4], np.int32)
    drafts = np.array([[0, 1, 2], [3, 100, 5]], np.int64)
    a = [None, FAKE, drafts.ctypes.data, FAKE, None, 2, 3, 100, 400, 100, 0, 0, 8, counts.ctypes.data, 1.0, FAKE, FAKE, FAKE, None, 0, 0, C.DT_MEM_HOST,
         None]
    refused(C.lib().dt_verify_drafts(*a), C.DT_ERR_INVALID_ARG, "counts[1]=4")
    counts[1] = 2
    refused(C.lib().dt_verify_drafts(*a), C.DT_ERR_INVALID_ARG, "draft 100 of row 1")
    counts[1] = 1
    refused(C.lib().dt_verify_drafts(*a), C.DT_ERR_INVALID_ARG, "ctx is NULL")


def test_kernels_use_no_scratch_memory():
    """Scratch memory would be allocated at a kernel's first launch, at the latest: a captured call cannot have that."""
    from test_kernel_scratch_cpu import _code_objects, _kernels

    import dirktensor_amd as dt

    if not dt.LIB_PATH.exists():
        pytest.skip("the library is not built")
    sizes = {k[".name"]: (k[".private_segment_fixed_size"], bool(k.get(".uses_dynamic_stack")))
             for elf in _code_objects(dt.LIB_PATH.read_bytes()) for k in _kernels(elf)}
    mine = {n: s for n, s in sizes.items() if any(x in n for x in ("rotary", "head_norm", "verify_"))}
    assert len(mine) >= 30, sorted(mine)
    assert {n: s for n, s in mine.items() if s != (0, False)} == {}
