"""The cache in 4 bits and the attention over it: held values against the format's definition in 64 bits, and what the other formats'
tests ask of the cache and its attention."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn
import test_cached_attn_range_gpu as ends
import test_kv_cache_gpu as cache

pytestmark = pytest.mark.gpu

D = 128
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
TYPES = [torch.float32, torch.bfloat16]


def held64(x, fmt="fp4"):
    """What the cache stands for, in 64 bits, of finite rows x [..., 128]."""
    assert fmt == "fp4"
    g = x.detach().cpu().double().unflatten(-1, (4, 32))
    amax = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -120.0)
    for cand in range(-120, 127):  # the smallest power of two that brings the group within 6
        e = torch.where(amax > 6 * 2.0 ** (cand - 1), torch.full_like(e, float(cand)), e) if cand > -120 else e
    s = 2.0 ** e
    y = (g / s).abs()
    d = (y[..., None] - LEVELS).abs()
    near = d.amin(-1, keepdim=True)
    code = torch.where(d == near, torch.arange(8) + 10.0 * (torch.arange(8) % 2), 100.0).argmin(-1)  # (of two, the even one)
    q = LEVELS[code] * torch.sign(g)
    return (torch.where((q * s).abs() < 2.0 ** 128, q, 3 * torch.sign(q)) * s).flatten(-2)


@pytest.fixture(autouse=True)
def _definition(monkeypatch):
    monkeypatch.setattr(cache, "held64", held64)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 31, 3), (3, 32, 2), (1, 33, 16), (2, 200, 5), (2, 8, 3), (1, 9, 2)])
def test_held_values(gpu, tdt, B, T, H):
    cache.test_held_values("fp4", tdt, B, T, H)


def test_every_level_and_the_middles_between(gpu):
    from dirktensor_amd import KVCache

    mids = (LEVELS[1:] + LEVELS[:-1]) / 2
    points = torch.cat([LEVELS, mids, mids * (1 + 2.0 ** -20), mids * (1 - 2.0 ** -20)]).float()
    x = torch.zeros((1, 4, 2, D))
    x[..., :len(points)] = points
    x[..., 64:64 + len(points)] = -points
    x[..., 40], x[..., 104] = 6.0, -6.0
    x = x * 2.0 ** torch.tensor([0.0, -30.0, 77.0, -110.0])[None, :, None, None]
    c = KVCache(1, 4, 2, format="fp4")
    c.append(x.cuda(), x.cuda())
    for got in c.read([0], 4, mode="fp32"):
        assert torch.equal(got.cpu().double(), held64(x))


def test_ends_of_the_range(gpu):
    from dirktensor_amd import KVCache

    H = 8
    x = torch.zeros((1, 1, H, D), device="cuda")
    x[0, 0, 0] = torch.linspace(-1, 1, D) * 3.4e38
    x[0, 0, 1] = torch.linspace(-1e-35, 1e-35, D)  # (around the least scale)
    x[0, 0, 2] = torch.linspace(-1e-40, 1e-40, D)
    x[0, 0, 3, 5] = 1e-45
    x[0, 0, 4] = torch.linspace(-6, 6, D) * 2.0 ** -120
    x[0, 0, 5] = 6.0
    x[0, 0, 6] = 6.0 * (1 + 2.0 ** -22)
    x[0, 0, 7, ::32] = 2.0 ** torch.tensor([127.0, 0.0, -100.0, 126.5])  # (groups of very different size)
    c = KVCache(1, 4, H, format="fp4")
    c.append(x, x)
    for got in c.read([0], 1, mode="fp32"):
        assert torch.equal(got.cpu().double(), held64(x))


def test_appends_of_any_length_hold_the_same(gpu):
    cache.test_appends_of_any_length_hold_the_same("fp4")


@pytest.mark.parametrize("start", [0, 1, 30, 31])
@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 33])
def test_neighbouring_keys_keep_their_halves(gpu, start, T):
    """Both ways to append, from even and odd positions, behind and before other rows; written twice (cut off and appended again)."""
    from dirktensor_amd import KVCache

    H, L = 3, 80
    k, v = cache.rows((2, L, H, D), 1, torch.float32), cache.rows((2, L, H, D), 2, torch.float32)
    junk = torch.full((2, L, H, D), float("nan"), device="cuda")
    c = KVCache(2, L, H, format="fp4")
    c.append(junk, junk)
    c.truncate([0, 0])
    for a, b in ((0, start), (start, start + T), (start + T, L)):
        if b > a:
            c.append(k[:, a:b], v[:, a:b], counts=[b - a, b - a])
    for got, x in zip(c.read([0, 0], L, mode="fp32"), (k, v)):
        assert torch.equal(got.cpu().double(), held64(x))
    c.truncate([start, L])
    c.append(v[:1, start:start + T], k[:1, start:start + T], slots=[0])
    for got, x, y in zip(c.read([0, 0], start + T, mode="fp32"), (k, v), (v, k)):
        assert torch.equal(got[0, :start].cpu().double(), held64(x[0, :start]))
        assert torch.equal(got[0, start:].cpu().double(), held64(y[0, start:start + T]))
        assert torch.equal(got[1].cpu().double(), held64(x[1, :start + T]))


def test_rows_that_are_none(gpu):
    cache.test_infinities_and_nan_make_their_row_nan("fp4")
    from dirktensor_amd import KVCache

    x = torch.ones((1, 2, 2, D), device="cuda")  # (and one by one)
    x[0, 1, 0, 99] = float("inf")
    c = KVCache(1, 2, 2, format="fp4")
    for t in range(2):
        c.append(x[:, t:t + 1], x[:, t:t + 1])
    for got in c.read([0], 2, mode="fp32"):
        assert torch.isnan(got[0, 1, 0]).all() and int(torch.isnan(got).sum()) == D


def test_host_rows(gpu):
    cache.test_host_rows("fp4")


def test_offsets_past_32_bits(gpu):
    cache.test_offsets_past_32_bits("fp4")


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("lens", [[1], [2, 31, 32, 33], [127, 128, 129, 0, 700], [1000], [4099, 5]])
def test_one_token(gpu, tdt, lens):
    attn.test_one_token("fp4", tdt, lens)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("T,H,Hk,causal", [(2, 2, 2, True), (17, 2, 1, True), (5, 8, 2, False), (33, 3, 3, True), (70, 4, 2, True),
                                           (1, 16, 1, True), (1, 40, 1, True), (1, 70, 1, False)])
def test_several_tokens_and_shared_heads(gpu, tdt, T, H, Hk, causal):
    attn.test_several_tokens_and_shared_heads("fp4", tdt, T, H, Hk, causal)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("B,T,H,Hk,P", [(1, 1, 2, 2, 1), (3, 1, 2, 2, 333), (20, 1, 2, 2, 1000), (12, 5, 4, 1, 2777), (40, 1, 2, 2, 129)])
def test_shared_prefix(gpu, tdt, B, T, H, Hk, P):
    attn.test_shared_prefix("fp4", tdt, B, T, H, Hk, P)


@pytest.mark.parametrize("tdt", TYPES)
def test_nan_rows_reach_only_the_queries_that_see_them(gpu, tdt):
    attn.test_nan_rows_reach_only_the_queries_that_see_them("fp4", tdt)


@pytest.mark.parametrize("tdt", TYPES)
def test_nan_rows_and_shared_heads(gpu, tdt):
    """Several query tiles a wave, of which some see a row that is none and others do not."""
    from dirktensor_amd import KVCache, cached_attention

    T, L, H, Hk = 20, 150, 8, 2
    k, v, q = attn.randn((1, L, Hk, D), 1), attn.randn((1, L, Hk, D), 2), attn.randn((1, T, H, D), 3, tdt)
    clean, c = (KVCache(1, L + 40, Hk, format="fp4") for _ in range(2))
    clean.append(k, v)
    want = cached_attention(q, clean, attn.SCALE)
    k, v = k.clone(), v.clone()
    v[0, L - 7, 0, 5] = float("nan")   # seen by the last seven tokens, of the first four query heads
    k[0, L - 12, 1, 7] = float("inf")  # by the last twelve, of the others
    c.append(k, v)
    junk = torch.full((1, 40, Hk, D), float("nan"), device="cuda")
    c.append(junk, junk)
    c.truncate([L])
    r = cached_attention(q, c, attn.SCALE)
    hit = torch.zeros((1, T, H), dtype=torch.bool, device="cuda")
    hit[0, T - 7:, :4] = True
    hit[0, T - 12:, 4:] = True
    assert bool(torch.isnan(r.output[hit]).all())
    assert torch.equal(r.output[~hit], want.output[~hit]) and torch.equal(r.softmax_l[~hit], want.softmax_l[~hit])


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("B,T,H,Hk,longest,P", [(64, 1, 16, 16, 500, 0), (64, 1, 16, 16, 100, 300), (33, 3, 16, 16, 120, 0)])
def test_more_sequences_and_heads_than_workgroups(gpu, tdt, B, T, H, Hk, longest, P):
    attn.test_more_sequences_and_heads_than_workgroups("fp4", tdt, B, T, H, Hk, longest, P)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("B,L,T,H,Hk,P", [(1, 5, 1, 2, 2, 0), (1, 1000, 1, 2, 2, 0), (2, 3000, 3, 4, 2, 0), (20, 100, 1, 2, 2, 300),
                                          (64, 100, 1, 16, 16, 0), (3, 400, 40, 4, 2, 1500)])
def test_large_values_everywhere(gpu, tdt, B, L, T, H, Hk, P):
    ends.test_large_values_everywhere("fp4", tdt, B, L, T, H, Hk, P)


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("at", ["first", "last", "one_head", "prefix", "one_column"])
def test_large_values_in_one_place(gpu, tdt, at):
    ends.test_large_values_in_one_place("fp4", tdt, at)


@pytest.mark.parametrize("tdt", TYPES)
def test_scales_far_apart(gpu, tdt):
    """Groups of one row and rows of one block whose scales differ by many powers of two, in keys and in values."""
    from dirktensor_amd import KVCache

    L, H = 300, 2
    k, v = attn.randn((1, L, H, D), 1), attn.randn((1, L, H, D), 2)
    k = k * torch.exp2(torch.randint(-12, 1, (1, L, H, 4), device="cuda").float()).repeat_interleave(32, -1)
    v = v * torch.exp2(torch.randint(-60, 20, (1, L, H, 4), device="cuda").float()).repeat_interleave(32, -1)
    c = KVCache(1, L, H, format="fp4")
    c.append(k, v)
    attn.run(attn.randn((1, 3, H, D), 3, tdt), c)


def test_formats_do_not_mix(gpu):
    from dirktensor_amd import DTError, KVCache, cached_attention

    a, b = KVCache(1, 8, 2, format="fp4"), KVCache(1, 8, 2, format="int8")
    x = torch.ones((1, 4, 2, D), device="cuda")
    a.append(x, x)
    b.append(x, x)
    with pytest.raises(DTError, match="format"):
        cached_attention(x[:, :1], a, 0.1, prefix=b)


def test_graph_replays(gpu):
    from dirktensor_amd import KVCache, cached_attention

    L, H = 1500, 4
    k, v, q = attn.randn((1, L, H, D), 1), attn.randn((1, L, H, D), 2), attn.randn((1, 1, H, D), 3)
    c = KVCache(1, L + 1, H, format="fp4")
    c.append(k, v)
    kn, vn = attn.randn((1, 1, H, D), 4), attn.randn((1, 1, H, D), 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            c.append(kn, vn)
            r = cached_attention(q, c, attn.SCALE)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        for t in (kn, vn, q):
            t.copy_(attn.randn(tuple(t.shape), 50 + i))
        g.replay()
        torch.cuda.synchronize()
        eager = KVCache(1, L + 1, H, format="fp4")
        eager.append(k, v)
        eager.append(kn, vn)
        want = cached_attention(q, eager, attn.SCALE)
        assert torch.equal(r.output, want.output) and torch.equal(r.softmax_l, want.softmax_l)
