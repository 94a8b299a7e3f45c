"""Drafts of full batches verified: vocabularies whose rows are read in whole batches of 4096 values (an odd and an even number of
them, with and without a remainder), chunks that a wave takes one after another, and rows of many segments. Against the
definition in 64 bits, with the bounds of test_verify_drafts_gpu."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_verify_drafts_gpu import TYPES, check, dt, inputs, reference

pytestmark = pytest.mark.gpu


def spread(u):
    """Uniforms at both ends for some of the rows: their borders lie in the first and in the last chunks."""
    u[0::5, -1], u[1::5, -1], u[2::5, -1] = 0.0, 1.0 - 2.0 ** -24, 2.0 ** -12
    u[3::5, :-1] *= 0.1  # (more drafts accepted)
    return u


# (64 x 5 drafts with draft logits are 704 rows, three segments each: of 5 batches and 2 with a remainder; of 2 and a remainder alone; of 2;
# of 9, and 6 with a remainder)
@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("T", [0.8, 0.0])
@pytest.mark.parametrize("B,K,V", [(64, 5, 50021), (64, 5, 20011), (64, 5, 24576), (64, 5, 100352), (64, 2, 100352), (64, 2, 99991), (40, 8, 65537), (64, 0, 131101), (256, 1, 33333)])
def test_full_batches(gpu, tdt, draft, T, B, K, V):
    print(f"verify {tdt} draft={draft} T={T} B={B} K={K} V={V}", flush=True)
    x, d, u, y = inputs(B, K, V, 100 + K, tdt, draft)
    spread(u)
    check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T), reference(x, d, u, y, T))


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("T", [1.0, 0.0])
def test_ragged_and_masked(gpu, tdt, draft, T):
    B, K, V = 64, 5, 50021
    x, d, u, y = inputs(B, K, V, 31, tdt, draft, masked=True)
    spread(u)
    counts = np.arange(B) * 5 % (K + 1)
    want = reference(x, d, u, y, T, counts)
    for b in range(B):  # (the rows behind the counts are not read)
        x[b, counts[b] + 1:] = float("nan")
        if y is not None:
            y[b, counts[b]:] = float("nan")
    check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T, counts=counts), want)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("V", [100352, 50021])
def test_values_that_end_a_row(gpu, tdt, V):
    """The largest logit, the draft and what a token is drawn from at the ends of batches, segments and chunks."""
    B, K = 64, 5
    x, d, u, y = inputs(B, K, V, 37, tdt)
    places = [0, 7, 4095, 4096, 8191, 8192, 20479, 20480, 36863, 36864, 40959, 40960, V - 4097, V - 513, V - 512, V - 9, V - 8, V - 7, V - 2, V - 1]
    for b in range(B):
        for i in range(K):
            at = places[(b + 7 * i) % len(places)]
            x[b, i, at] = 14.0
            y[b, i, at] = 12.0 + 3 * ((b + i) % 2)
            if (b + i) % 3:
                d[b, i] = at
    for T in (1.0, 0.0):
        check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T), reference(x, d, u, y, T))


@pytest.mark.parametrize("tdt", TYPES)
def test_equal_logits_of_far_segments(gpu, tdt):
    """At temperature 0 the first of equals, in rows of 293 segments that 16 lanes join in several rounds."""
    B, V = 8, 600011
    x = torch.randn((B, 1, V), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(tdt)
    ties = [[V - 1], [0, V - 1], [2047, 2048], [131071, 131072, 300000], [262143, 5000], [599999, 200000, 400000], [2048 * 16 * 4, 2048 * 16 * 8], [599040, 1]]
    for b, t in enumerate(ties):
        x[b, 0, t] = 9.0
    d, u = torch.zeros((B, 0), dtype=torch.int32, device="cuda"), torch.full((B, 1), 0.5, device="cuda")
    r = dt().verify_drafts(x, d, u, temperature=0)
    assert r.tokens[:, 0].tolist() == [min(t) for t in ties]
    check(r, reference(x, d, u, None, 0))
    one = x[:1].clone()  # (one row: 293 segments; eight of them: 256)
    one[0, 0, [70000, 550000]] = 11.0
    r = dt().verify_drafts(one, d[:1], u[:1], temperature=0)
    assert r.tokens.tolist() == [[70000]]
    x[:, :, 10:] = float("-inf")
    check(dt().verify_drafts(x, d, u, temperature=1.0), reference(x, d, u, None, 1.0))
