"""Attention over the cache against 64 bits on the values the cache holds: one and several query tokens, ragged lengths
with empty ones, shared heads, a shared prefix, masks that leave rows empty, NaN rows, strides, streams, graphs."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 128
SCALE = 1.0 / math.sqrt(D)
FORMATS = ["int8", "fp8", "bf16"]


def randn(shape, seed, tdt=torch.float32, scale=1.0):
    return (scale * torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(tdt)


def fill(cache, lens, seed, slots=None, vscale=1.0):
    """Random rows of the given lengths in the cache's slots."""
    slots = list(range(len(lens))) if slots is None else slots
    for i, (s, n) in enumerate(zip(slots, lens)):
        if n:
            cache.append(randn((1, n, cache.n_heads, D), seed + 2 * i), randn((1, n, cache.n_heads, D), seed + 2 * i + 1, scale=vscale),
                         slots=[s])


def held(cache, slot):
    n = int(cache.lengths[slot])
    if n == 0:
        return [torch.zeros((0, cache.n_heads, D), dtype=torch.float64, device="cuda")] * 2
    return [x[0].double() for x in cache.read([0], n, slots=[slot], mode="fp32")]


def reference(q, cache, causal, slots, counts, prefix, prefix_slot, scale=SCALE):
    """o, m, l in 64 bits, sum p |v| / l, and the largest sum |q_d k_d| scale a query has."""
    B, T, H, _ = q.shape
    G = H // cache.n_heads
    o = torch.zeros((B, T, H, D), dtype=torch.float64, device="cuda")
    a = torch.zeros_like(o)
    m = torch.full((B, T, H), float("-inf"), dtype=torch.float64, device="cuda")
    l, big = torch.zeros_like(m), torch.zeros_like(m)
    pk, pv = held(prefix, prefix_slot) if prefix is not None else (None, None)
    for b in range(B):
        k, v = held(cache, slots[b])
        n, c = len(k), counts[b]
        for t in range(c):
            vis = max(0, min(n, n - c + t + 1)) if causal else n
            kk, vv = k[:vis], v[:vis]
            if pk is not None:
                kk, vv = torch.cat([pk, kk]), torch.cat([pv, vv])
            if len(kk) == 0:
                continue
            for h in range(H):
                x = q[b, t, h].double()
                s = kk[:, h // G] @ x * scale
                m[b, t, h] = s.max()
                p = (s - s.max()).exp()
                l[b, t, h] = p.sum()
                o[b, t, h] = p @ vv[:, h // G].contiguous() / p.sum()
                a[b, t, h] = p @ vv[:, h // G].abs().contiguous() / p.sum()
                big[b, t, h] = (kk[:, h // G].abs() @ x.abs()).max() * scale
    return o, m, l, a, big


def check(r, ref, tdt):
    """Scores: sums of 128 products in 32 bits, at most 44 roundings one after another (12 of the accumulator, 32 within the
    instruction), and two more by the scales: d <= 46 2^-24 sum|q k| scale. A probability is then off by 2 d relative and, by
    its exponent's and exp2's roundings, by 4 2^-24 (1 + |s - m|) where it counts (|s - m| <= 2 big); sums over the keys, in 32
    bits in runs and a tree of at most 64 + 40 additions, by 104 2^-24. In bf16 a term and the result are rounded once more
    (2^-8 each)."""
    o, m, l, a, big = ref
    e = 2.0 ** -24
    d = 46 * e * big
    rel = 2 * d + 4 * e * (1 + 2 * big) + 104 * e
    empty = l == 0
    got = r.output.double()
    assert r.output.dtype == tdt
    assert bool((r.softmax_m[empty] == float("-inf")).all()) and bool((r.softmax_l[empty] == 0).all())
    assert bool((got[empty] == 0).all())
    live = ~empty
    assert bool(((r.softmax_m.double() - m).abs()[live] <= (d + 2 * e * m.abs())[live]).all())
    # (l is relative to the m that is reported)
    assert bool(((r.softmax_l.double() - l).abs()[live] <= ((rel + 2 * d) * l)[live]).all())
    tol = 2 * rel[..., None] * a
    if tdt == torch.bfloat16:
        tol = tol + 2.0 ** -8 * a + 2.0 ** -8 * (o.abs() + 2.0 ** -8 * a)
    else:
        tol = tol + e * o.abs()
    bad = ((got - o).abs() > tol + 1e-30)
    assert not bool(bad.any()), (float(((got - o).abs() / (tol + 1e-30)).max()), bad.nonzero()[:4].tolist())


def run(q, cache, causal=True, slots=None, counts=None, prefix=None, prefix_slot=0):
    from dirktensor_amd import cached_attention

    B, T = q.shape[:2]
    r = cached_attention(q, cache, SCALE, causal, slots=slots, counts=counts, prefix=prefix, prefix_slot=prefix_slot)
    ref = reference(q, cache, causal, list(range(B)) if slots is None else list(slots),
                    [T] * B if counts is None else list(counts), prefix, prefix_slot)
    check(r, ref, q.dtype)
    return r


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[1], [2, 31, 32, 33], [127, 128, 129, 0, 700], [1000], [4099, 5]])
def test_one_token(fmt, tdt, lens):
    from dirktensor_amd import KVCache

    print(f"one token {fmt} {tdt} lens={lens}", flush=True)
    c = KVCache(len(lens), max(lens), 3, format=fmt)
    fill(c, lens, 10)
    run(randn((len(lens), 1, 3, D), 1, tdt), c)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,Hk,causal", [(2, 2, 2, True), (17, 2, 1, True), (5, 8, 2, False), (33, 3, 3, True), (70, 4, 2, True),
                                           (1, 16, 1, True), (1, 40, 1, True), (1, 70, 1, False)])
def test_several_tokens_and_shared_heads(fmt, tdt, T, H, Hk, causal):
    """Every number of query tiles a workgroup takes; a slot shorter than its query tokens (its first rows see nothing);
    padded batch rows."""
    from dirktensor_amd import KVCache

    print(f"several tokens {fmt} {tdt} T={T} H={H} Hk={Hk} causal={causal}", flush=True)
    lens = [T + 300, max(1, T // 2), T, 0]
    c = KVCache(4, T + 300, Hk, format=fmt)
    fill(c, lens, 40)
    run(randn((4, T, H, D), 2, tdt), c, causal, counts=[T, T, (T + 1) // 2, T])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H,Hk,P", [(1, 1, 2, 2, 1), (3, 1, 2, 2, 333), (20, 1, 2, 2, 1000), (12, 5, 4, 1, 2777), (40, 1, 2, 2, 129)])
def test_shared_prefix(fmt, tdt, B, T, H, Hk, P):
    from dirktensor_amd import KVCache

    print(f"shared prefix {fmt} {tdt} B={B} T={T} H={H} Hk={Hk} P={P}", flush=True)
    rng = np.random.default_rng(B)
    lens = [int(n) for n in rng.integers(0, 260, size=B)]
    c, p = KVCache(B + 1, 260, Hk, format=fmt), KVCache(3, P + 5, Hk, format=fmt)
    slots = [int(s) for s in rng.permutation(B + 1)[:B]]
    fill(c, lens, 80, slots)
    fill(p, [P], 79, [2])
    counts = [int(n) for n in rng.integers(0, T + 1, size=B)]
    counts[0] = T
    run(randn((B, T, H, D), 3, tdt), c, slots=slots, counts=counts, prefix=p, prefix_slot=2)


def test_prefix_in_the_same_cache_and_slots_twice():
    from dirktensor_amd import KVCache

    c = KVCache(4, 300, 2)
    fill(c, [50, 300, 0, 7], 200)
    q = randn((5, 1, 2, D), 4, torch.bfloat16)
    q[4] = q[0]
    r = run(q, c, slots=[0, 3, 2, 1, 0], prefix=c, prefix_slot=1)
    assert torch.equal(r.output[4], r.output[0])
    r = run(q, c, slots=[0, 0, 0, 0, 0], prefix=c, prefix_slot=2)  # (an empty prefix)
    assert torch.equal(r.output[4], r.output[0])


def test_a_prefix_and_nothing_of_their_own():
    """A full batch whose slots hold nothing yet, and one none of whose rows has a query."""
    from dirktensor_amd import KVCache

    B, H = 64, 16
    c, p = KVCache(B, 10, H), KVCache(1, 500, H)
    fill(p, [500], 700)
    q = randn((B, 1, H, D), 701, torch.bfloat16)
    run(q, c, prefix=p)
    r = run(q, c, counts=[0] * B, prefix=p)
    assert not bool(r.output.any())
    fill(c, [1] * B, 702)
    run(q, c, counts=[0] * B, prefix=p)
    run(q, c, counts=[0] * B)
    run(q, c, counts=[1] + [0] * (B - 1), prefix=p)


def test_a_whole_sequence_is_the_causal_attention():
    """All tokens appended at once, unquantised, then attended: flash_attention_forward's results."""
    from dirktensor_amd import KVCache, cached_attention, flash_attention_forward

    B, T, H = 2, 400, 4
    q, k, v = (randn((B, T, H, D), s, torch.float32).bfloat16().float() for s in (5, 6, 7))
    c = KVCache(B, T, H, format="bf16")
    c.append(k, v)
    a, b = cached_attention(q, c, SCALE), flash_attention_forward(q, k, v, SCALE)
    # both lie within 1e-5 of 64 bits on rows of unit variance
    assert float((a.output - b.output).abs().max()) < 2e-5
    assert float((a.softmax_m - b.softmax_m).abs().max()) < 2e-5
    assert float(((a.softmax_l - b.softmax_l) / b.softmax_l).abs().max()) < 2e-5


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", [torch.bfloat16, torch.float32])
def test_nan_rows_reach_only_the_queries_that_see_them(fmt, tdt):
    from dirktensor_amd import KVCache, cached_attention

    T, L, H = 6, 150, 2
    k, v = randn((1, L, H, D), 8), randn((1, L, H, D), 9)
    q = randn((1, T, H, D), 10, tdt)
    clean = KVCache(1, L + 40, H, format=fmt)
    clean.append(k, v)
    want = cached_attention(q, clean, SCALE)
    k2, v2 = k.clone(), v.clone()
    v2[0, L - 3, 0, 5] = float("nan")   # seen by the last three queries of head 0
    k2[0, L - 2, 1, 7] = float("inf")   # by the last two of head 1
    c = KVCache(1, L + 40, H, format=fmt)
    c.append(k2, v2)
    # rows behind the sequence: appended, then cut off
    junk = torch.full((1, 40, H, D), float("nan"), device="cuda")
    c.append(junk, junk)
    c.truncate([L])
    r = cached_attention(q, c, SCALE)
    hit = torch.zeros((1, T, H), dtype=torch.bool, device="cuda")
    hit[0, T - 3:, 0] = True
    hit[0, T - 2:, 1] = True
    assert bool(torch.isnan(r.output[hit]).all())
    assert torch.equal(r.output[~hit], want.output[~hit])
    assert torch.equal(r.softmax_m[~hit], want.softmax_m[~hit]) and torch.equal(r.softmax_l[~hit], want.softmax_l[~hit])
    assert bool(torch.isnan(r.softmax_m[0, T - 2:, 1]).all())


def test_large_scores():
    """Scores of hundreds and thousands: the running maximum moves often, most probabilities vanish."""
    from dirktensor_amd import KVCache

    for tdt in (torch.bfloat16, torch.float32):
        c = KVCache(1, 600, 1, format="bf16")
        k = randn((1, 600, 1, D), 11) * torch.linspace(1, 60, 600, device="cuda")[None, :, None, None]
        c.append(k, randn((1, 600, 1, D), 12))
        run(randn((1, 3, 1, D), 13, tdt, 4.0), c)


def test_small_and_large_queries_in_fp32():
    """Rows of q whose size is far from one, beside ordinary ones."""
    from dirktensor_amd import KVCache

    c = KVCache(1, 200, 4)
    fill(c, [200], 300)
    q = randn((1, 2, 4, D), 14)
    q[0, 0, 0] *= 1e-36
    q[0, 0, 1] *= 1e-10
    q[0, 0, 2] = 0
    q[0, 1, 3] *= 100
    run(q, c)


def test_strided_queries_and_host_arrays():
    from dirktensor_amd import KVCache, cached_attention

    B, T, H = 2, 3, 4
    c = KVCache(B, 90, H, format="fp8")
    fill(c, [90, 40], 400)
    wide = randn((B, T, 3 * H * D), 15, torch.bfloat16)
    q = wide[..., H * D:2 * H * D].unflatten(-1, (H, D))
    want = cached_attention(q.contiguous(), c, SCALE)
    got = cached_attention(q, c, SCALE)
    assert torch.equal(got.output, want.output)
    host = cached_attention(q.float().cpu().numpy(), c, SCALE)
    dev = cached_attention(q.float(), c, SCALE)
    assert np.array_equal(host.output, dev.output.cpu().numpy())
    assert np.array_equal(host.softmax_m, dev.softmax_m.cpu().numpy()) and np.array_equal(host.softmax_l, dev.softmax_l.cpu().numpy())
    bits = cached_attention(q.contiguous().view(torch.int16).cpu().numpy().view(np.uint16), c, SCALE)
    assert np.array_equal(bits.output, want.output.view(torch.int16).cpu().numpy().view(np.uint16))


def test_streams_at_once():
    """Calls that read one cache and one prefix on several streams at the same time, each with its own workspace."""
    from dirktensor_amd import KVCache, cached_attention

    B, H = 8, 8
    c, p = KVCache(B, 2000, H), KVCache(1, 1500, H)
    fill(c, [2000 - 100 * i for i in range(B)], 500)
    fill(p, [1500], 499)
    qs = [randn((B, 1, H, D), 20 + i, torch.bfloat16) for i in range(4)]
    want = [cached_attention(q, c, SCALE, prefix=p).output for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[] for _ in qs]
    for _ in range(5):
        for i, (s, q) in enumerate(zip(streams, qs)):
            with torch.cuda.stream(s):
                got[i].append(cached_attention(q, c, SCALE, prefix=p).output)
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for o in got[i]:
            assert torch.equal(o, w)


def test_graph_replays():
    """An append and an attention captured together, replayed with other inputs, eager work between the replays."""
    from dirktensor_amd import KVCache, cached_attention

    B, H, L = 2, 4, 700
    c, p = KVCache(B, 1000, H), KVCache(1, 900, H)
    fill(c, [L, 300], 600)
    fill(p, [900], 599)
    q, k, v = (randn((B, 1, H, D), s, torch.bfloat16) for s in (30, 31, 32))
    s = torch.cuda.Stream()
    before = c.lengths
    with torch.cuda.stream(s):  # (first calls outside the capture)
        c.append(k, v)
        cached_attention(q, c, SCALE, prefix=p)
    torch.cuda.synchronize()
    c.truncate(before)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.append(k, v)
            r = cached_attention(q, c, SCALE, prefix=p)
        graphs.append(g)
        outs.append(r)
        assert c.lengths.tolist() == (before + 1).tolist()
        c.truncate(before)
    for i in range(4):
        for x, sd in ((q, 40), (k, 41), (v, 42)):
            x.copy_(randn((B, 1, H, D), sd + 10 * i, torch.bfloat16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        c.append(k, v)
        want = cached_attention(q, c, SCALE, prefix=p)
        for r in outs:
            assert torch.equal(r.output, want.output) and torch.equal(r.softmax_l, want.softmax_l)
        c.truncate(before)
        torch.cuda.synchronize()


def test_a_generation_of_several_answers():
    """A prompt in the prefix, answers appended token by token, each attended as it is: the last step is the attention over
    the whole sequences, and the same as with the prompt copied into every slot."""
    from dirktensor_amd import KVCache, cached_attention

    B, H, P, N = 5, 2, 77, 40
    pk, pv = randn((1, P, H, D), 50, torch.bfloat16), randn((1, P, H, D), 51, torch.bfloat16)
    prompt, answers, whole = KVCache(1, P, H), KVCache(B, N, H), KVCache(B, P + N, H)
    prompt.append(pk, pv)
    whole.append(pk.expand(B, P, H, D), pv.expand(B, P, H, D))
    for i in range(N):
        q, k, v = (randn((B, 1, H, D), 60 + 3 * i + j, torch.bfloat16) for j in range(3))
        answers.append(k, v)
        whole.append(k, v)
        a = cached_attention(q, answers, SCALE, prefix=prompt)
        b = cached_attention(q, whole, SCALE)
        check(a, reference(q, answers, True, range(B), [1] * B, prompt, 0), torch.bfloat16)
        # (the two sum the same terms, each rounded to bf16, in another order)
        assert float((a.output.float() - b.output.float()).abs().max()) < 0.05
    answers.truncate([0] * B)
    assert answers.lengths.tolist() == [0] * B


def test_long_cache_past_32_bits():
    """A slot whose bytes begin past 2^32, a million tokens long."""
    from dirktensor_amd import KVCache, cached_attention

    cap, H = 1 << 20, 16
    c = KVCache(2, cap, H)
    n = 1 << 15
    kv = [randn((1, n, H, D), 70 + i, torch.bfloat16) for i in range(2)]
    for _ in range(cap // n):
        c.append(*kv, slots=[1])
    q = randn((1, 1, H, D), 72, torch.bfloat16)
    r = cached_attention(q, c, SCALE, slots=[1])
    short = KVCache(1, n, H)
    short.append(*kv)
    w = cached_attention(q, short, SCALE)
    # 32 copies of the same keys: the same output and maximum, 32 times the sum
    assert torch.equal(r.softmax_m, w.softmax_m)
    assert float((r.softmax_l / (32 * w.softmax_l) - 1).abs().max()) < 1e-5
    # both are rounded to bf16 once (2^-8 relative each, of values up to about 0.1)
    assert float((r.output.float() - w.output.float()).abs().max()) <= 2 * 2.0 ** -8 * float(w.output.float().abs().max())


@pytest.mark.parametrize("fmt,tdt", [("int8", torch.bfloat16), ("int8", torch.float32), ("fp8", torch.float32), ("bf16", torch.bfloat16)])
@pytest.mark.parametrize("B,T,H,Hk,longest,P", [(64, 1, 16, 16, 500, 0), (64, 1, 16, 16, 100, 300), (33, 3, 16, 16, 120, 0),
                                                (130, 5, 16, 4, 128, 77), (256, 1, 3, 3, 2300, 0), (256, 1, 3, 3, 1200, 200)])
def test_more_sequences_and_heads_than_workgroups(fmt, tdt, B, T, H, Hk, longest, P):
    """One (head, sequence) a wave, and shares of a list in which workgroups have several, up to the largest batch."""
    from dirktensor_amd import KVCache

    print(f"more than workgroups {fmt} {tdt} B={B} T={T} H={H} Hk={Hk} longest={longest} P={P}", flush=True)
    rng = np.random.default_rng(longest)
    lens = [int(n) for n in rng.integers(0, longest + 1, size=B)]
    lens[:4] = [longest, 0, 1, 32]
    counts = [int(n) for n in rng.integers(0, T + 1, size=B)]
    counts[:4] = [T, T, T, T]
    c = KVCache(B, longest, Hk, format=fmt)
    k, v = randn((B, longest, Hk, D), 900), randn((B, longest, Hk, D), 901)
    c.append(k, v, counts=lens)
    p = None
    if P:
        p = KVCache(1, P, Hk, format=fmt)
        fill(p, [P], 902)
    run(randn((B, T, H, D), 903, tdt), c, counts=counts, prefix=p)


def test_many_query_tiles():
    """More (head, sequence, query tile) triples than are cut: a prompt in chunks over a cache, padded, with and without a
    prefix; compared with one token at a time at sampled places (the reference's loop would take minutes)."""
    from dirktensor_amd import KVCache, cached_attention

    B, T, H, Hk = 4, 700, 8, 4
    c, p = KVCache(B, 900, Hk, format="fp8"), KVCache(1, 200, Hk, format="fp8")
    fill(c, [900, 700, 350, 701], 800)
    fill(p, [200], 790)
    q = randn((B, T, H, D), 801, torch.bfloat16)
    counts = [700, 700, 500, 1]
    for pre in (None, p):
        r = cached_attention(q, c, SCALE, counts=counts, prefix=pre)
        held_at = c.lengths.copy()
        for b in range(B):
            for t in (0, 1, 333, 499, 500, 699):
                if t >= counts[b]:
                    assert not bool(r.output[b, t].any()) and bool((r.softmax_l[b, t] == 0).all())
                    continue
                seen = max(0, int(held_at[b]) - counts[b] + t + 1)
                if seen == 0 and pre is None:
                    assert not bool(r.output[b, t].any())
                    continue
                one = KVCache(1, 900, Hk, format="fp8")
                if seen:
                    k, v = c.read([0], seen, slots=[b], mode="fp32")  # (held values are held again as they are)
                    one.append(k, v)
                w = cached_attention(q[b:b + 1, t:t + 1], one, SCALE, prefix=pre)
                # the same terms in another order, each rounded to bf16 (2^-8 of a term, values of unit size) and the result once
                assert float((w.output[0, 0].float() - r.output[b, t].float()).abs().max()) <= 0.03
                assert float((w.softmax_m[0, 0] - r.softmax_m[b, t]).abs().max()) <= 1e-5


def test_a_workspace_that_is_too_small_is_refused():
    import ctypes

    from dirktensor_amd import KVCache, _capi as C

    B, H = 2, 4
    c = KVCache(400, 3000, H)  # (more slots than a call has rows)
    fill(c, [3000, 2999], 950, slots=[399, 300])
    q = randn((B, 1, H, D), 951, torch.bfloat16)
    r = run(q, c, slots=[399, 300])
    slots = np.array([399, 300], np.int32)
    need = ctypes.c_int64()
    args = (None, None, 0, C.DT_BF16)
    C.call("dt_cached_attn_workspace", c.handle, B, 1, H, D, slots.ctypes.data, *args, ctypes.byref(need))
    assert need.value > 0
    ws = torch.full((need.value + 256,), 77, dtype=torch.uint8, device="cuda")
    o = torch.zeros_like(q)

    def call(at, n):
        return C.lib().dt_cached_attn_fwd(c.handle, q.data_ptr(), o.data_ptr(), None, None, B, 1, H, D, H * D, SCALE, 1,
                                          slots.ctypes.data, None, None, 0, at, n, C.DT_BF16, C.DT_MEM_DEVICE, None)

    for at, n, msg in ((None, need.value, "the workspace has 0"), (ws.data_ptr(), need.value - 1, "the workspace has"),
                       (ws.data_ptr() + 8, need.value, "aligned")):
        assert call(at, n) == C.DT_ERR_INVALID_ARG and msg in C.lib().dt_last_error().decode()
    assert not bool(o.any())
    assert call(ws.data_ptr(), need.value) == C.DT_OK
    torch.cuda.synchronize()
    assert torch.equal(o, r.output) and bool((ws[need.value:] == 77).all())


def test_more_rows_than_a_call_takes():
    from dirktensor_amd import DTError, KVCache, cached_attention

    c = KVCache(300, 4, 1)
    x = randn((256, 2, 1, D), 960)
    c.append(x, x)
    run(x[:, -1:], c)
    with pytest.raises(DTError, match="B=257"):
        cached_attention(randn((257, 1, 1, D), 961), c, SCALE)
    with pytest.raises(DTError, match="B=257"):
        c.append(randn((257, 1, 1, D), 962), randn((257, 1, 1, D), 963))
    assert c.lengths.tolist() == [2] * 256 + [0] * 44


def test_a_closed_context():
    from dirktensor_amd import Context, KVCache, cached_attention

    ctx = Context(0)
    c = KVCache(1, 40, 2, ctx=ctx)
    x = randn((1, 4, 2, D), 1)
    c.append(x, x)
    ctx.close()
    with pytest.raises(RuntimeError, match="context"):
        cached_attention(x, c, SCALE)
    with pytest.raises(RuntimeError, match="context"):
        c.append(x, x)
    c.close()


def test_refusals():
    from dirktensor_amd import DTError, KVCache, cached_attention

    c, p = KVCache(2, 10, 2), KVCache(1, 10, 2, format="fp8")
    q = torch.zeros((2, 1, 2, D), device="cuda")
    for kw, msg in ((dict(slots=[0, 2]), "outside"), (dict(counts=[2, 0]), "outside"), (dict(prefix=p), "another"),
                    (dict(prefix=c, prefix_slot=2), "prefix_slot")):
        with pytest.raises(DTError, match=msg):
            cached_attention(q, c, SCALE, **kw)
    with pytest.raises(DTError, match="multiple"):
        cached_attention(torch.zeros((2, 1, 3, D), device="cuda"), c, SCALE)
    with pytest.raises(DTError, match="head_dim"):
        cached_attention(torch.zeros((2, 1, 2, 64), device="cuda"), c, SCALE)
    with pytest.raises(DTError, match="slots"):
        cached_attention(torch.zeros((3, 1, 2, D), device="cuda"), c, SCALE)
    with pytest.raises(DTError, match="scale"):
        cached_attention(q, c, 0.0)
    with pytest.raises(ValueError):
        cached_attention(q.cpu(), c, SCALE)
    with pytest.raises(ValueError):
        cached_attention(q[0], c, SCALE)
    with pytest.raises(TypeError):
        cached_attention(q.half(), c, SCALE)
    r = cached_attention(q, c, SCALE)  # nothing held: empty rows
    assert not bool(r.output.any()) and bool((r.softmax_m == float("-inf")).all())
