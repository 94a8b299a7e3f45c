"""Token scores and their gradient against 64 bits: row lengths and alignments around every form, masked and degenerate rows,
ties, few rows (cut into segments) and many, strided views, refusals, streams and graphs; the gradient against the formula and
against differences."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def logits_of(rows, V, seed, tdt, scale=3.0, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = (scale * torch.randn(rows * V + offset, generator=g, device="cuda")).to(tdt)
    return buf[offset:].view(rows, V)


def tokens_of(rows, V, seed, dtype=torch.int32):
    return torch.randint(0, V, (rows,), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda").to(dtype)


def reference(x, tok, k):
    """64 bits: logprob, entropy, m, l, indices, their log probabilities."""
    z = x.double()
    m = z.amax(-1, keepdim=True)
    d = z - m
    e = d.exp()
    l = e.sum(-1, keepdim=True)
    logl = l.log()
    t = torch.where(torch.isinf(d), torch.zeros_like(d), d)
    ent = (logl - (e * t).sum(-1, keepdim=True) / l)[:, 0]
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    return (d - logl).gather(1, tok.long()[:, None])[:, 0], ent, m[:, 0], l[:, 0], order.to(torch.int32), (d - logl).gather(1, order)


def check(r, x, tok, k):
    """32-bit arithmetic: x - m is rounded once (2^-24 |x - m|) and scaled once before exp2 (2 2^-24 |x - m| relative with it),
    exp2 is good to 2 2^-24 relative; a thread adds up to V / 256 + 1 values one after another, with a rounding at most at each
    (2^-24 of the sum), and rescales it seldom (counted with the adds); the tree adds 10. Terms with |x - m| > 30 do not count
    (e < 1e-13), so the sums are good to rel = (3 30 + V / 256 + 20) 2^-24, and log l to that absolutely (with log's own
    roundings, 2 2^-24 |log l|)."""
    lp, ent, m, l, order, top = reference(x, tok, k)
    V = x.shape[-1]
    rel = (110 + V / 256) * E
    assert torch.equal(r.softmax_m.double(), m)
    assert bool(((r.softmax_l.double() - l).abs() <= rel * l).all())
    tol = rel + 3 * E * l.log()
    fin = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(r.logprob), fin)
    assert bool(((r.logprob.double() - lp).abs() <= tol + 2 * E * lp.abs())[fin].all())
    # (the weighted sum's terms carry the same relative error; each addition's rounding is relative to the whole of it)
    assert bool(((r.entropy.double() - ent).abs() <= 2 * rel * (ent.abs() + 1) + tol).all())
    if k:
        assert torch.equal(r.top_index, order)
        fin = torch.isfinite(top)
        assert torch.equal(torch.isfinite(r.top_logprob), fin)
        assert bool(((r.top_logprob.double() - top).abs() <= tol[:, None] + 2 * E * top.abs())[fin].all())


def check_grad(got, x, tok, g, h, keep=None):
    """p from (x - m) - log l in 32 bits: relative error rel + 4 2^-24 (1 + |log p|); the bracket's terms are rounded and
    carry it too; |log p| <= 110 where p counts."""
    z, V = x.double(), x.shape[-1]
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    lp = torch.where(p == 0, torch.zeros_like(logp), logp)
    ent = -(p * lp).sum(-1, keepdim=True)
    g, h = g.double()[:, None], h.double()[:, None]
    if keep is not None:
        g = g * keep[:, None]
    want = -p * (g + h * (lp + ent))
    size = p * (g.abs() + h.abs() * (lp.abs() + ent.abs()))
    want.scatter_add_(1, tok.long().clamp_min(0)[:, None], g)
    size.scatter_add_(1, tok.long().clamp_min(0)[:, None], g.abs())
    rel = (110 + V / 256) * E
    tol = (4 * rel + 8 * E * (1 + lp.abs())) * size + 4 * rel * p * h.abs() + E * want.abs() + 1e-38
    if x.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 257, 1023, 2047, 2048, 2049, 4095, 4099, 8192, 8195, 16391, 50277, 100352, 131077])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_row_lengths_and_alignments(tdt, V, offset):
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    rows, k = 3, min(V, 20)
    print(f"rows of {V} {tdt} offset {offset}", flush=True)
    x, tok = logits_of(rows, V, V, tdt, offset=offset), tokens_of(rows, V, V)
    r = token_logprobs(x, tok, top_k=k)
    check(r, x, tok, k)
    none = token_logprobs(x, tok.long())
    assert none.top_index is None and torch.equal(none.logprob, r.logprob) and torch.equal(none.entropy, r.entropy)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    check_grad(token_logprobs_backward(g, x, tok, r, d_entropy=h), x, tok, g, h)
    check_grad(token_logprobs_backward(g, x, tok, r), x, tok, g, torch.zeros_like(h))


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(1, 100352, 64), (1, 100352, 0), (17, 30011, 33), (200, 4099, 64), (700, 5000, 1),
                                      (2100, 2500, 7), (2500, 61, 61), (5000, 33, 0)])
def test_few_and_many_rows(tdt, rows, V, k):
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    print(f"{rows} rows of {V} {tdt} top {k}", flush=True)
    x, tok = logits_of(rows, V, rows, tdt), tokens_of(rows, V, rows)
    r = token_logprobs(x, tok, top_k=k)
    check(r, x, tok, k)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    check_grad(token_logprobs_backward(g, x, tok, r, d_entropy=h), x, tok, g, h)


@pytest.mark.parametrize("rows", [2, 2100])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two_values", "one_thread", "zeros", "peak"])
def test_orders_and_ties(rows, kind):
    """Rows whose largest values lie anywhere: all equal, sorted, many ties, all in one thread's share, signed zeros."""
    from dirktensor_amd import token_logprobs

    V, k = 9001, 64
    print(f"{kind}, {rows} rows", flush=True)
    i = torch.arange(V, device="cuda")
    x = {"equal": torch.full((V,), 2.5, device="cuda"), "rising": i * 1e-3, "falling": -i * 1e-3,
         "two_values": (i % 7 == 3).float(), "one_thread": torch.where(i // 4 % 256 == 77, 5.0 + i * 1e-4, torch.zeros_like(i * 1.0)),
         "zeros": torch.where(i % 2 == 0, torch.tensor(0.0, device="cuda"), torch.tensor(-0.0, device="cuda")),
         "peak": torch.where(i == 8999, 80.0, 0.0)}[kind].float()
    x = x[None].expand(rows, V) if rows > 100 else x[None].repeat(rows, 1)
    tok = tokens_of(rows, V, 3)
    check(token_logprobs(x, tok, top_k=k), x, tok, k)
    b = x.bfloat16()
    check(token_logprobs(b, tok, top_k=k), b, tok, k)


def test_more_values_at_the_bound_than_the_list_holds():
    """k threads hold all of the large values, thousands of them: the selection goes one by one."""
    from dirktensor_amd import token_logprobs

    V, k = 120000, 64
    i = torch.arange(V, device="cuda")
    noise = torch.randn(V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    share = i // 4 % 256
    x = torch.where(share < 63, 60.0 + noise, torch.where(share == 63, 30.0 + noise, noise))
    # one thread's share (a piece of 4 in 256) of the whole row: rows enough that none is cut
    rows = 2048
    x = x[None].expand(rows, V)
    tok = tokens_of(rows, V, 5)
    r = token_logprobs(x, tok, top_k=k)
    want = torch.sort(x[0], descending=True, stable=True).indices[:k].to(torch.int32)
    assert torch.equal(r.top_index, want[None].expand(rows, k))
    check(token_logprobs(x[:2], tok[:2], top_k=k), x[:2], tok[:2], k)


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2049])
@pytest.mark.parametrize("kind", ["first_masked", "few_left", "rising_first_masked", "ties_first_masked", "equal_last"])
@pytest.mark.parametrize("V,k", [(40007, 64), (40007, 5), (1021, 64), (1030, 64), (2900, 33)])
def test_alternatives_behind_masked_values(tdt, rows, kind, V, k):
    """Rows that begin with masked values, or have fewer than k others: the bound of the row's beginning lets all values through."""
    from dirktensor_amd import token_logprobs

    print(f"{kind}, {rows} rows of {V} {tdt}", flush=True)
    i = torch.arange(V, device="cuda")
    x = logits_of(1, V, 11, torch.float32)[0]
    lowest = torch.full_like(x, float("-inf"))
    x = {"first_masked": torch.where(i < V // 2, lowest, x),
         "few_left": torch.where((i * 7919 % V) % 1000 == 3, x, lowest),
         "rising_first_masked": torch.where(i < V // 4, lowest, i * (40.0 / V)),
         "ties_first_masked": torch.where(i < V // 3, lowest, (i % 5).float()),
         "equal_last": torch.where(i < V - 1500, lowest, torch.ones_like(x))}[kind]
    x = x.to(tdt)[None].expand(rows, V)
    tok = torch.full((rows,), int(x[0].argmax()), dtype=torch.int32, device="cuda")
    r = token_logprobs(x, tok, top_k=k)
    check(r, x, tok, k)


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
def test_masked_and_degenerate_rows(tdt):
    """-inf and the type's lowest value in most places, rows with one token left, without any, with NaN and +inf."""
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    V, k = 5003, 30
    x = logits_of(8, V, 1, tdt).clone()
    tok = tokens_of(8, V, 1)
    low = torch.finfo(tdt).min
    x[0, 10:] = float("-inf")          # ten tokens left: the alternatives go on with the masked ones, by index
    x[1] = float("-inf")
    x[1, 4000] = 1.5                   # one left
    x[2, 20:] = low
    x[3] = low
    tok[0], tok[1], tok[2] = 4, 4000, 3
    for part in (x[:4], x[:4].repeat(600, 1)):
        t = tok[:4].repeat(len(part) // 4)
        r = token_logprobs(part, t, top_k=k)
        check(r, part, t, k)
        g, h = torch.randn(len(t), device="cuda"), torch.randn(len(t), device="cuda")
        check_grad(token_logprobs_backward(g, part, t, r, d_entropy=h), part, t, g, h)
    assert float(r.logprob[1]) == 0.0 and float(r.entropy[1]) == 0.0
    tok[0] = 11                        # a masked token
    r = token_logprobs(x[:1], tok[:1])
    assert float(r.logprob[0]) == float("-inf")
    x[4] = float("-inf")
    x[5, 2222] = float("nan")
    x[6, 5002] = float("inf")
    r = token_logprobs(x, tok, top_k=k)
    for name in ("logprob", "entropy", "softmax_m", "softmax_l"):
        assert torch.isnan(getattr(r, name)).tolist() == [False] * 4 + [True] * 3 + [False], name
    assert bool(torch.isnan(r.top_logprob[4:7]).all())
    assert r.top_index[4].tolist() == list(range(k))
    z = x[5].float().nan_to_num(nan=float("-inf"))
    assert torch.equal(r.top_index[5].long(), torch.sort(z, descending=True, stable=True).indices[:k])
    assert int(r.top_index[6, 0]) == 5002
    d = token_logprobs_backward(torch.ones(8, device="cuda"), x, tok, r, d_entropy=torch.ones(8, device="cuda"))
    assert torch.isnan(d).all(-1).tolist() == [False] * 4 + [True] * 3 + [False]
    assert bool(torch.isfinite(d[[0, 1, 2, 3, 7]]).all())


def test_all_nan_row_has_alternatives_in_range():
    from dirktensor_amd import token_logprobs

    x = torch.full((1, 300), float("nan"), device="cuda")
    r = token_logprobs(x, torch.zeros(1, dtype=torch.int32, device="cuda"), top_k=40)
    assert r.top_index[0].tolist() == list(range(40)) and bool(torch.isnan(r.top_logprob).all())


def test_ignored_and_foreign_tokens():
    from dirktensor_amd import DTError, token_logprobs, token_logprobs_backward

    V = 700
    x = logits_of(6, V, 2, torch.float32)
    tok = torch.tensor([5, -100, 699, 700, -1, 2 ** 32 + 5], dtype=torch.int64, device="cuda")
    r = token_logprobs(x, tok, ignore_index=-100)
    ok = torch.tensor([0, 2], device="cuda")
    want = reference(x[ok], tok[ok], 0)[0]
    assert float((r.logprob[ok].double() - want).abs().max()) < 1e-5
    assert float(r.logprob[1]) == 0.0 and torch.isnan(r.logprob).tolist() == [False] * 3 + [True] * 3
    assert bool(torch.isfinite(r.entropy).all())
    g, h = torch.randn(6, device="cuda"), torch.randn(6, device="cuda")
    d = token_logprobs_backward(g, x, tok, r, d_entropy=h)
    assert bool(torch.isnan(d[3:]).all())
    check_grad(d[:3], x[:3], tok[:3], g[:3], h[:3], keep=torch.tensor([1.0, 0.0, 1.0], dtype=torch.float64, device="cuda"))
    with pytest.raises(DTError, match="token 700"):
        token_logprobs(x.cpu().numpy(), tok.cpu().numpy(), ignore_index=-100)


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
def test_next_token_views_and_outputs(tdt):
    """logits[:, :-1] is taken as it is, the gradient lands in a view of a larger buffer or on the logits themselves."""
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    B, T, V = 3, 6, 1003
    full = logits_of(B * T, V, 3, tdt).view(B, T, V)
    tok = tokens_of(B * T, V, 3).view(B, T)
    x, y = full[:, :-1], tok[:, 1:]
    dense = x.contiguous()
    r, w = token_logprobs(x, y, top_k=3), token_logprobs(dense, y.contiguous(), top_k=3)
    for name in ("logprob", "entropy", "softmax_m", "softmax_l", "top_index", "top_logprob"):
        assert torch.equal(getattr(r, name), getattr(w, name)), name
    check(token_logprobs(dense.view(-1, V), y.reshape(-1), top_k=3), dense.view(-1, V), y.reshape(-1), 3)
    g, h = torch.randn((B, T - 1), device="cuda"), torch.randn((B, T - 1), device="cuda")
    want = token_logprobs_backward(g, dense, y, w, d_entropy=h)
    assert torch.equal(token_logprobs_backward(g, x, y, r, d_entropy=h), want)
    buf = torch.full_like(full, 7.0)
    out = token_logprobs_backward(g, x, y, r, d_entropy=h, out=buf[:, :-1])
    assert torch.equal(out, want) and bool((buf[:, -1] == 7.0).all())
    out = token_logprobs_backward(g, dense, y, r, d_entropy=h, out=buf.fill_(7.0)[:, :-1])
    assert torch.equal(out, want) and bool((buf[:, -1] == 7.0).all())
    wide = torch.full((B, T - 1, V + 5), 7.0, dtype=tdt, device="cuda")
    out = token_logprobs_backward(g, x, y, r, d_entropy=h, out=wide[..., 2:V + 2])
    assert torch.equal(out, want) and bool((wide[..., :2] == 7.0).all()) and bool((wide[..., V + 2:] == 7.0).all())
    last = full[:, -1].clone()
    assert torch.equal(token_logprobs_backward(g, x, y, r, d_entropy=h, out=x), want)
    assert torch.equal(full[:, -1], last)
    # other orders of the leading dimensions, one row, a vocabulary that is not contiguous
    p = dense.transpose(0, 1)
    assert torch.equal(token_logprobs(p, y.transpose(0, 1)).logprob, r.logprob.transpose(0, 1))
    p2 = p.clone(memory_format=torch.preserve_format)
    assert p2.stride() == p.stride()
    got = token_logprobs_backward(g.T, p2, y.T, token_logprobs(p2, y.T), d_entropy=h.T, out=p2)
    assert got is p2 and torch.equal(got, want.transpose(0, 1))
    one = token_logprobs(dense[0, 0], y[0, 0], top_k=2)
    assert one.logprob.shape == () and torch.equal(one.top_index, r.top_index[0, 0, :2])
    q = dense.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(token_logprobs(q, y).logprob, r.logprob)
    assert torch.equal(token_logprobs_backward(g, q, y, r, d_entropy=h), want)


def test_host_arrays():
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    B, T, V = 2, 3, 2111
    x, tok = logits_of(B * T, V, 4, torch.float32).view(B, T, V), tokens_of(B * T, V, 4).view(B, T)
    g, h = torch.randn((B, T), device="cuda"), torch.randn((B, T), device="cuda")
    for dev in (x, x.bfloat16()):
        r = token_logprobs(dev, tok, top_k=5)
        hx = dev.cpu().numpy() if dev.dtype == torch.float32 else dev.view(torch.int16).cpu().numpy().view(np.uint16)
        n = token_logprobs(hx, tok.cpu().numpy(), top_k=5)
        for name in ("logprob", "entropy", "softmax_m", "softmax_l", "top_index", "top_logprob"):
            assert np.array_equal(getattr(n, name), getattr(r, name).cpu().numpy()), name
        d = token_logprobs_backward(g, dev, tok, r, d_entropy=h)
        hd = token_logprobs_backward(g.cpu().numpy(), hx, tok.cpu().numpy(), n, d_entropy=h.cpu().numpy())
        assert np.array_equal(hd, d.cpu().numpy() if d.dtype == torch.float32 else d.view(torch.int16).cpu().numpy().view(np.uint16))


def test_gradient_against_differences():
    """d_logits of sum(g logprob + h entropy) against central differences of the forward's 64-bit formula, and of the
    forward itself: with steps of 2^-5 an fp32 forward good to 2e-6 gives the slope to 2 2e-6 / 2^-4 sum|g| + |h|, and the third
    derivative (at most 2 |g| + 8 |h|) adds 2^-10 / 6 of itself."""
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    V = 24
    x, tok = logits_of(4, V, 6, torch.float32, scale=1.0), tokens_of(4, V, 6)
    g, h = torch.randn(4, device="cuda"), torch.randn(4, device="cuda")
    d = token_logprobs_backward(g, x, tok, token_logprobs(x, tok), d_entropy=h).double()

    def value(z):
        r = token_logprobs(z, tok)
        return g.double() * r.logprob.double() + h.double() * r.entropy.double()

    step = 2.0 ** -5
    for j in range(V):
        e = torch.zeros_like(x)
        e[:, j] = step
        slope = (value(x + e) - value(x - e)) / (2 * step)
        tol = (g.abs() + h.abs()).double() * (2 * 2e-6 / (2 * step)) + step ** 2 / 6 * (2 * g.abs() + 8 * h.abs()).double()
        assert bool(((slope - d[:, j]).abs() <= tol).all()), (j, slope, d[:, j])


def test_streams_and_graph_replays():
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    rows, V = 5, 20011
    xs = [logits_of(rows, V, 10 + i, torch.float32) for i in range(4)]
    tok = tokens_of(rows, V, 10)
    want = [token_logprobs(x, tok, top_k=9) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], []
    for s, x in zip(streams * 3, xs * 3):
        with torch.cuda.stream(s):
            got.append(token_logprobs(x, tok, top_k=9))
    torch.cuda.synchronize()
    for r, w in zip(got, want * 3):
        assert torch.equal(r.top_index, w.top_index) and torch.equal(r.entropy, w.entropy)
    x, g = xs[0].clone(), torch.randn(rows, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        r = token_logprobs(x, tok, top_k=9)
        d = token_logprobs_backward(g, x, tok, r, d_entropy=g)
    for i in (1, 2, 3, 0):
        x.copy_(xs[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        w = token_logprobs(xs[i], tok, top_k=9)
        assert torch.equal(r.logprob, w.logprob) and torch.equal(r.top_index, w.top_index) and torch.equal(r.top_logprob, w.top_logprob)
        assert torch.equal(d, token_logprobs_backward(g, xs[i], tok, w, d_entropy=g))


def test_rows_past_32_bits():
    """Rows that begin past 2^31 elements."""
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    V, rows = 1 << 20, 2100
    x = torch.zeros((rows, V), dtype=torch.bfloat16, device="cuda")
    x[-1] = logits_of(1, V, 7, torch.bfloat16)[0]
    tok = torch.full((rows,), 3, dtype=torch.int32, device="cuda")
    r = token_logprobs(x, tok, top_k=4)
    check(type(r)(*(getattr(r, n)[-1:] for n in ("logprob", "entropy", "softmax_m", "softmax_l", "top_index", "top_logprob"))), x[-1:],
          tok[-1:], 4)
    assert r.top_index[0].tolist() == [0, 1, 2, 3] and abs(float(r.logprob[0]) + 20 * math.log(2)) < 1e-5
    g = torch.ones(rows, device="cuda")
    d = token_logprobs_backward(g, x, tok, r, out=x)
    assert float(d[-2, 3]) == 1.0 and float(d[-2, 4]) == -2.0 ** -20
    assert float(d[-1, 3]) > 0.9


def test_refusals():
    from dirktensor_amd import DTError, token_logprobs, token_logprobs_backward

    x, tok = logits_of(3, 50, 1, torch.float32), tokens_of(3, 50, 1)
    for k in (-1, 51, 65):
        with pytest.raises(DTError, match="top_k"):
            token_logprobs(x, tok, top_k=k)
    with pytest.raises(ValueError):
        token_logprobs(x, tok[:2])
    with pytest.raises(ValueError):
        token_logprobs(x, tok.cpu())
    with pytest.raises(ValueError):
        token_logprobs(x.cpu(), tok.cpu())
    with pytest.raises(TypeError):
        token_logprobs(x, tok.float())
    with pytest.raises(TypeError):
        token_logprobs(x.half(), tok)
    with pytest.raises(DTError):
        token_logprobs(x[:0], tok[:0])
    r = token_logprobs(x, tok)
    g = torch.ones(3, device="cuda")
    for out in (x.bfloat16(), x[:2], torch.empty((50, 3), device="cuda").t(), torch.empty((1, 50), device="cuda").expand(3, 50)):
        with pytest.raises((ValueError, DTError)):
            token_logprobs_backward(g, x, tok, r, out=out)
    buf = torch.empty(4 * 50, device="cuda")
    y = buf[:150].view(3, 50)
    y.copy_(x)
    with pytest.raises(ValueError, match="overlaps"):
        token_logprobs_backward(g, y, tok, r, out=buf[50:].view(3, 50))
    with pytest.raises(ValueError):
        token_logprobs_backward(g[:2], x, tok, r)
