"""Attention over cached values near the end of fp32's range: the sums before the division by l pass it, the results do not. Against
64 bits on the values the cache holds, with the bounds of test_cached_attn_gpu (relative to sum p |v| / l, whatever its size), and every
result a number."""

import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn

pytestmark = pytest.mark.gpu

D, SCALE = attn.D, attn.SCALE
FORMATS, DTYPES = attn.FORMATS, [torch.bfloat16, torch.float32]
TOP = 2.5e38  # (a mean of such values, off by 2^-7 at most, and its rounding to bf16 stay below 3.39e38)


def numbers(r):
    return all(not bool(torch.isnan(x).any()) for x in (r.output, r.softmax_m, r.softmax_l)) and bool(torch.isfinite(r.output).all())


def values(shape, seed, size=TOP):
    return attn.randn(shape, seed).clamp(-1, 1) * size


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", DTYPES)
@pytest.mark.parametrize("B,L,T,H,Hk,P", [(1, 5, 1, 2, 2, 0), (1, 1000, 1, 2, 2, 0), (2, 3000, 3, 4, 2, 0), (20, 100, 1, 2, 2, 300),
                                          (64, 100, 1, 16, 16, 0), (3, 400, 40, 4, 2, 1500)])
def test_large_values_everywhere(fmt, tdt, B, L, T, H, Hk, P):
    """Every form of the call: one workgroup's keys, shares of a list and their join, one (head, sequence) a wave, a prefix, several
    query tiles a wave."""
    from dirktensor_amd import KVCache

    print(f"large values {fmt} {tdt} B={B} L={L} T={T} H={H} Hk={Hk} P={P}", flush=True)
    c, p = KVCache(B, L, Hk, format=fmt), None
    c.append(attn.randn((B, L, Hk, D), 1), values((B, L, Hk, D), 2))
    if P:
        p = KVCache(1, P, Hk, format=fmt)
        p.append(attn.randn((1, P, Hk, D), 3), values((1, P, Hk, D), 4))
    assert numbers(attn.run(attn.randn((B, T, H, D), 5, tdt), c, prefix=p))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", DTYPES)
@pytest.mark.parametrize("at", ["first", "last", "one_head", "prefix", "one_column"])
def test_large_values_in_one_place(fmt, tdt, at):
    """Some waves' sums are too large and others' are not: they meet in a workgroup, in the join, and behind a prefix."""
    from dirktensor_amd import KVCache

    print(f"large values {at} {fmt} {tdt}", flush=True)
    B, L, T, H, P = 2, 4000, 2, 3, 700
    k, v = attn.randn((B, L, H, D), 11), attn.randn((B, L, H, D), 12)
    pk, pv = attn.randn((1, P, H, D), 13), attn.randn((1, P, H, D), 14)
    if at == "first":
        v[:, :40] = values((B, 40, H, D), 15)
    elif at == "last":
        v[:, -300:] = values((B, 300, H, D), 15)
    elif at == "one_head":
        v[:, :, 1] = values((B, L, D), 15)
    elif at == "prefix":
        pv = values((1, P, H, D), 15)
    else:
        v[:, :, :, 77] = values((B, L, H), 15)
    q = attn.randn((B, T, H, D), 16, tdt)
    c, p = KVCache(B, L, H, format=fmt), KVCache(1, P, H, format=fmt)
    c.append(k, v)
    p.append(pk, pv)
    assert numbers(attn.run(q, c))
    assert numbers(attn.run(q, c, prefix=p))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", DTYPES)
def test_scores_that_rise(fmt, tdt):
    """Each key's score is higher than the one before by little: the terms are largest relative to the running base."""
    from dirktensor_amd import KVCache

    L = 600
    c = KVCache(1, L, 1, format=fmt)
    k = torch.zeros((1, L, 1, D), device="cuda")
    k[..., 0] = torch.linspace(0, 40, L, device="cuda")[None, :, None]
    q = torch.zeros((1, 1, 1, D), device="cuda", dtype=tdt)
    q[..., 0] = 8.0
    for size in (1e36, 1e37, TOP):
        c.truncate([0])
        c.append(k, values((1, L, 1, D), 21, size))
        assert numbers(attn.run(q, c))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", DTYPES)
def test_a_mean_of_many_large_values(fmt, tdt):
    """40000 keys of one score and value: that value, to the rounding of the sums' arithmetic."""
    from dirktensor_amd import KVCache, cached_attention

    L = 40000
    c = KVCache(1, L, 2, format=fmt)
    k, v = attn.randn((1, L, 2, D), 31), torch.full((1, L, 2, D), 2.0 ** 127, device="cuda")
    v[:, :, 1] *= -1
    c.append(k, v)
    held = c.read([0], 1, mode="fp32")[1][:, :1].double()
    r = cached_attention(torch.zeros((1, 1, 2, D), device="cuda", dtype=tdt), c, SCALE)
    assert bool((r.softmax_l == L).all())
    # 1250 blocks of 32 keys: however they are cut, no term meets more than 1250 + 32 additions one after another, and the scales, the
    # division and the waves' factors round it 6 times; bf16: the term and the result once each
    tol = 1300 * 2.0 ** -24 + (2.0 ** -7 if tdt == torch.bfloat16 else 0.0)
    assert numbers(r) and bool(((r.output.double() / held - 1).abs() <= tol).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", DTYPES)
def test_nan_rows_beside_large_values(fmt, tdt):
    """A NaN in a large row reaches the queries that see it, the others stay as they are without it."""
    from dirktensor_amd import KVCache, cached_attention

    T, L, H = 6, 150, 2
    k, v, q = attn.randn((1, L, H, D), 41), values((1, L, H, D), 42), attn.randn((1, T, H, D), 43, tdt)
    clean, c = KVCache(1, L, H, format=fmt), KVCache(1, L, H, format=fmt)
    clean.append(k, v)
    v[0, L - 3, 0, 5] = float("nan")
    c.append(k, v)
    want, r = attn.run(q, clean), cached_attention(q, c, SCALE)
    assert numbers(want)
    assert bool(torch.isnan(r.output[0, T - 3:, 0]).all())
    assert torch.equal(r.output[0, :T - 3], want.output[0, :T - 3]) and torch.equal(r.output[0, :, 1], want.output[0, :, 1])


@pytest.mark.parametrize("tdt", DTYPES)
def test_ordinary_sequences_beside_large_ones(tdt):
    """One batch: sequences of unit size and of 2.5e38 behind one prefix, whose chunks serve them together; each sequence's result is what
    it is alone, within the bounds."""
    from dirktensor_amd import KVCache

    B, L, H, P = 12, 200, 2, 1000
    c, p = KVCache(B, L, H), KVCache(1, P, H)
    v = attn.randn((B, L, H, D), 51)
    v[::3] = values((len(range(0, B, 3)), L, H, D), 52)
    c.append(attn.randn((B, L, H, D), 53), v)
    p.append(attn.randn((1, P, H, D), 54), attn.randn((1, P, H, D), 55))
    assert numbers(attn.run(attn.randn((B, 2, H, D), 56, tdt), c, prefix=p))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("qsize,ksize", [(1e-34, 3e37), (1e-36, 2.5e38), (1e-30, 1e30), (1e30, 1e-30), (1.0, 1.0)])
def test_large_keys_and_small_queries_in_fp32(fmt, qsize, ksize):
    """Scores of ordinary size from keys near the end of the range: no sum on the way to them may pass it."""
    from dirktensor_amd import KVCache

    L, H, T = 300, 2, 3
    c = KVCache(1, L, H, format=fmt)
    c.append(values((1, L, H, D), 61, ksize), attn.randn((1, L, H, D), 62))
    assert numbers(attn.run(attn.randn((1, T, H, D), 63, scale=qsize), c))
    # the same sign everywhere: the largest sums that such values have
    c.truncate([0])
    c.append(values((1, L, H, D), 64, ksize).abs(), attn.randn((1, L, H, D), 65))
    assert numbers(attn.run(attn.randn((1, T, H, D), 66, scale=qsize).abs(), c))
