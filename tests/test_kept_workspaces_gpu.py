"""Workspaces that calls on torch tensors keep for the next: whose they are and how long they are held."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 128


def randn(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def hip():
    """The HIP runtime that torch has loaded."""
    with open("/proc/self/maps") as f:
        path = next(ln.split()[-1] for ln in f if "libamdhip64" in ln)
    return ctypes.CDLL(path)


@pytest.fixture
def kept():
    from dirktensor_amd import _workspace

    _workspace._kept.by_stream.clear()
    return _workspace._kept.by_stream


@pytest.fixture
def calls():
    """An attention and scores that need workspaces, and whether their results are what the first ones were."""
    from dirktensor_amd import KVCache, cached_attention, token_logprobs

    c = KVCache(2, 3000, 4)
    c.append(randn((2, 3000, 4, D), 1), randn((2, 3000, 4, D), 2))
    q, x, tok = randn((2, 1, 4, D), 3), randn((2, 50021), 4), torch.arange(2, device="cuda")
    torch.cuda.synchronize()
    run = lambda: (cached_attention(q, c, 0.09).output, token_logprobs(x, tok, top_k=9).top_logprob)
    want = run()
    torch.cuda.synchronize()

    def same():
        got = run()
        torch.cuda.current_stream().synchronize()
        return all(torch.equal(a, b) for a, b in zip(got, want))

    return same


def test_streams_from_elsewhere_keep_none(kept, calls):
    lib, raw = hip(), ctypes.c_void_p()
    assert lib.hipStreamCreateWithFlags(ctypes.byref(raw), ctypes.c_uint(1)) == 0
    try:
        with torch.cuda.stream(torch.cuda.ExternalStream(raw.value)):
            assert calls() and calls()
            assert not any(stream == raw.value for _, stream in kept)
        torch.cuda.synchronize()
    finally:
        assert lib.hipStreamDestroy(raw) == 0
    pool = torch.cuda.Stream()
    with torch.cuda.stream(pool):
        assert calls() and calls()
    assert (0, pool.cuda_stream) in kept
    # the same stream by its address: its work is in the same order, so it takes what the stream has
    with torch.cuda.stream(torch.cuda.ExternalStream(pool.cuda_stream)):
        n = len(kept)
        assert calls() and len(kept) == n


def test_a_thread_keeps_them_for_few_streams(kept, calls):
    streams = {}
    for _ in range(40):
        s = torch.cuda.Stream()
        streams[s.cuda_stream] = s
        with torch.cuda.stream(s):
            assert calls()
        assert len(kept) <= 8 and (0, s.cuda_stream) in kept
    assert len(streams) > 8


def test_they_are_given_back(kept, calls):
    import gc
    import threading

    import dirktensor_amd as dt

    def held():
        gc.collect()  # (what earlier tests left in cycles)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        return torch.cuda.memory_allocated()

    dt.release_workspaces()
    before = held()
    done, go, ok = threading.Event(), threading.Event(), []

    def work():
        ok.append(calls())
        done.set()
        go.wait(60)
        ok.append(calls())

    t = threading.Thread(target=work)
    t.start()
    done.wait(60)
    assert calls() and held() >= before + 2 * (1 << 20)  # this thread's and the other's
    dt.release_workspaces()
    assert held() == before
    go.set()
    t.join()
    assert ok == [True, True] and calls()
    dt.release_workspaces()
    assert held() == before
