"""Errors that the device reports reach the caller of cached_attention, also where the call has a kept workspace at hand."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_an_error_of_the_first_attempt_is_raised(monkeypatch):
    """The library's answer to the first attempt is replaced by a device error: a second attempt would succeed and hide it."""
    from dirktensor_amd import DTError, KVCache, _capi as C, cache, cached_attention

    c = KVCache(1, 3000, 2)
    x = torch.randn((1, 3000, 2, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    c.append(x, x)
    q = x[:, -1:].contiguous()
    want = cached_attention(q, c, 0.09).output  # (keeps a workspace)
    lib, answers = C.lib(), [C.DT_ERR_HIP]

    class Library:
        def __getattr__(self, name):
            f = getattr(lib, name)
            if name != "dt_cached_attn_fwd":
                return f
            return lambda *a: answers.pop() if answers else f(*a)

    monkeypatch.setattr(cache.C, "lib", Library)
    with pytest.raises(DTError) as e:
        cached_attention(q, c, 0.09)
    assert e.value.code == C.DT_ERR_HIP and not answers
    assert torch.equal(cached_attention(q, c, 0.09).output, want)
