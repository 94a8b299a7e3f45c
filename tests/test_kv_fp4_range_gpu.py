"""Attention over a cache in 4 bits at the ends of fp32's range: what the other formats' tests ask (test_cached_attn_range_gpu,
test_cached_attn_gpu), of 4 bits; several key tiles of a long prompt in parts; one (head, sequence) a wave."""

import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn
import test_cached_attn_range_gpu as ends

pytestmark = pytest.mark.gpu

D = 128
TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("tdt", TYPES)
def test_scores_that_rise(gpu, tdt):
    ends.test_scores_that_rise("fp4", tdt)


@pytest.mark.parametrize("tdt", TYPES)
def test_a_mean_of_many_large_values(gpu, tdt):
    ends.test_a_mean_of_many_large_values("fp4", tdt)


@pytest.mark.parametrize("tdt", TYPES)
def test_nan_rows_beside_large_values(gpu, tdt):
    ends.test_nan_rows_beside_large_values("fp4", tdt)


@pytest.mark.parametrize("qsize,ksize", [(1e-34, 3e37), (1e-36, 2.5e38), (1e-30, 1e30), (1e30, 1e-30), (1e34, 1e-34), (1.0, 1.0)])
def test_large_keys_and_small_queries_in_fp32(gpu, qsize, ksize):
    ends.test_large_keys_and_small_queries_in_fp32("fp4", qsize, ksize)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("T,H,Hk,P", [(256, 2, 1, 0), (130, 4, 4, 1000), (300, 2, 2, 0)])
def test_parts_of_a_prompt(gpu, tdt, T, H, Hk, P):
    """Hundreds of new tokens behind what the cache holds."""
    from dirktensor_amd import KVCache

    L = T + 170
    c, p = KVCache(1, L, Hk, format="fp4"), None
    c.append(attn.randn((1, L, Hk, D), 1), attn.randn((1, L, Hk, D), 2))
    if P:
        p = KVCache(1, P, Hk, format="fp4")
        p.append(attn.randn((1, P, Hk, D), 3), attn.randn((1, P, Hk, D), 4))
    attn.run(attn.randn((1, T, H, D), 5, tdt), c, prefix=p)
