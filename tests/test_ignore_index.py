"""Which tokens a score skips at the ends of 64 bits, on a host without a GPU: the check of host tokens runs before the first HIP call."""

import numpy as np
import pytest

from dirktensor_amd import _capi as C
from dirktensor_amd import logprobs

FAKE = 0x10000  # aligned non-NULL address; never dereferenced because validation fails first
LEAST = -(2 ** 63)


def scores(tok, ignore):
    rc = C.lib().dt_token_logprobs(None, FAKE, tok.ctypes.data, 1, len(tok), 100, 100 * len(tok), 100, 8, ignore, 0, FAKE, None, FAKE, FAKE,
                                   None, None, None, 0, 0, C.DT_MEM_HOST, None)
    return rc, C.lib().dt_last_error().decode()


def gradient(tok, ignore):
    rc = C.lib().dt_token_logprobs_bwd(None, FAKE, None, FAKE, tok.ctypes.data, FAKE, FAKE, None, 1, len(tok), 100, 100 * len(tok), 100, 8,
                                       ignore, FAKE, 100 * len(tok), 100, 0, C.DT_MEM_HOST, None)
    return rc, C.lib().dt_last_error().decode()


@pytest.mark.parametrize("call", [scores, gradient])
def test_without_an_ignored_index_no_token_is_skipped(call):
    rc, msg = call(np.array([3, LEAST], np.int64), C.DT_NO_IGNORE)
    assert rc == C.DT_ERR_INVALID_ARG and f"token {LEAST} of row 1" in msg
    rc, msg = call(np.array([3, -100], np.int64), -100)
    assert "ctx is NULL" in msg


def test_indices_that_64_bits_do_not_hold():
    assert logprobs._ignore_of(None) == C.DT_NO_IGNORE
    for i in (-100, 0, 100277, 2 ** 63 - 1, LEAST + 1):
        assert logprobs._ignore_of(i) == i
    for i in (2 ** 63, 2 ** 64 - 100, LEAST, LEAST - 1):  # (the second would arrive as -100)
        with pytest.raises(ValueError, match="ignore_index"):
            logprobs._ignore_of(i)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 2100])
def test_the_least_token_on_the_device(rows):
    torch = pytest.importorskip("torch")
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    x = torch.randn((rows, 5003), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    tok = torch.full((rows,), 7, dtype=torch.int64, device="cuda")
    tok[1] = LEAST
    r = token_logprobs(x, tok)
    nan = [i == 1 for i in range(rows)]
    assert torch.isnan(r.logprob).tolist() == nan and bool(torch.isfinite(r.entropy).all())
    d = token_logprobs_backward(torch.ones(rows, device="cuda"), x, tok, r)
    assert torch.isnan(d).all(-1).tolist() == nan and bool(torch.isfinite(d[[0, 2]]).all())
    tok[1] = -100
    r = token_logprobs(x, tok, ignore_index=-100)
    assert float(r.logprob[1]) == 0.0
    with pytest.raises(ValueError, match="ignore_index"):
        token_logprobs(x, tok, ignore_index=2 ** 64 - 100)
