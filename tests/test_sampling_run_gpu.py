"""The cache, its attention and the scores as they are used together: answers to one prompt are sampled token by token, scored as they
are sampled, attended and scored again in one pass, and a gradient is taken; each step against 64 bits."""

import math

import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn
import test_token_logprobs_gpu as scores

pytestmark = pytest.mark.gpu

D, E = 128, 2.0 ** -24


def randn(shape, seed, scale=1.0):
    return scale * torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def logits_bound(w, ref):
    """How far logits may be from W o in 64 bits: the exact mode's bound on o, through W, and a product of d terms in 32 bits
    (d + 1 roundings at most)."""
    o, _, l, a, big = ref
    rel = 2 * 46 * E * big + 4 * E * (1 + 2 * big) + 104 * E
    off = 2 * rel[..., None] * a + E * o.abs()
    flat = lambda x: x.flatten(-2)
    d = w.shape[0]
    wd = w.double().abs().contiguous()
    return flat(off) @ wd + (d + 1) * E * ((flat(o.abs()) + flat(off)) @ wd)


@pytest.mark.parametrize("fmt", ["int8", "fp8", "bf16"])
def test_answers_to_one_prompt(fmt):
    from dirktensor_amd import KVCache, cached_attention, token_logprobs, token_logprobs_backward

    N, S, P, H, Hk, V, k = 6, 20, 101, 4, 2, 1003, 5
    scale = 1.0 / math.sqrt(D)
    emb, w = randn((V, H * D), 1), randn((H * D, V), 2, 0.1)
    wq, wk, wv = (randn((H * D, n * D), 3 + i, 1.0 / math.sqrt(H * D)) for i, n in enumerate((H, Hk, Hk)))
    prompt = torch.randint(0, V, (P,), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    shared, own = KVCache(1, P, Hk, format=fmt), KVCache(N, S, Hk, format=fmt)
    x = emb[prompt]
    shared.append((x @ wk).view(1, P, Hk, D), (x @ wv).view(1, P, Hk, D))

    gen = torch.Generator(device="cuda").manual_seed(10)
    tok = prompt[-1].expand(N)
    qs, logits, chosen, each = [], [], [], []
    for i in range(S):
        x = emb[tok]
        q, key, val = (x @ wq).view(N, 1, H, D), (x @ wk).view(N, 1, Hk, D), (x @ wv).view(N, 1, Hk, D)
        own.append(key, val)
        r = cached_attention(q, own, scale, prefix=shared)
        y = r.output.view(N, H * D) @ w
        tok = torch.multinomial(torch.softmax(y, -1), 1, generator=gen)[:, 0]
        s = token_logprobs(y, tok, top_k=k)
        scores.check(s, y, tok, k)
        # from the held values to the scores, in 64 bits
        ref = attn.reference(q, own, True, range(N), [1] * N, shared, 0, scale)
        attn.check(r, ref, torch.float32)
        exact = ref[0].view(N, H * D) @ w.double()
        bound = logits_bound(w, ref)[:, 0].amax(-1)
        want = torch.log_softmax(exact, -1).gather(1, tok[:, None])[:, 0]
        # (log sum exp moves by no more than the logits do)
        tol = 2 * bound + (110 + V / 256) * E + 3 * E * math.log(V) + 2 * E * want.abs()
        assert bool(((s.logprob.double() - want).abs() <= tol).all())
        qs.append(q)
        logits.append(y)
        chosen.append(tok)
        each.append(s)

    # the answers in one pass: every query at once, and all scores
    assert own.lengths.tolist() == [S] * N
    q = torch.cat(qs, 1)
    r = cached_attention(q, own, scale, prefix=shared)
    attn.check(r, attn.reference(q, own, True, range(N), [S] * N, shared, 0, scale), torch.float32)
    y, toks = torch.stack(logits, 1), torch.stack(chosen, 1)
    s = token_logprobs(y, toks, top_k=k)
    flat = lambda t: t.reshape(N * S, *t.shape[2:])
    tol = 2 * ((110 + V / 256) * E + 3 * E * math.log(V))
    for name in ("logprob", "entropy", "top_logprob"):
        a, b = getattr(s, name), torch.stack([getattr(e, name) for e in each], 1)
        assert a.shape == b.shape and bool(((a - b).abs() <= tol * (2 + b.abs())).all()), name
    assert torch.equal(s.top_index, torch.stack([e.top_index for e in each], 1))

    # the gradient that a policy's training begins with, through the last product by autograd
    advantage, h = randn((N, S), 20), randn((N, S), 21, 0.01)
    dy = token_logprobs_backward(advantage, y, toks, s, d_entropy=h)
    assert dy.shape == y.shape
    scores.check_grad(flat(dy), flat(y), flat(toks), flat(advantage), flat(h))
    z = y.double().requires_grad_()
    lp = torch.log_softmax(z, -1)
    loss = (advantage.double() * lp.gather(2, toks[..., None])[..., 0]).sum() - (h.double()[..., None] * lp.exp() * lp).sum()
    loss.backward()
    # (the same bound as above, at its largest: |log p| <= 110, terms of size |g| + |h| 120)
    size = (advantage.abs() + 120 * h.abs()).double().amax()
    assert float((dy.double() - z.grad).abs().max()) <= float(4 * (110 + V / 256 + 2 * 111) * E * size)

    # taken back to the first half, the cache goes on from there with the same results
    own.truncate([S // 2] * N)
    again = []
    for i in range(S // 2, S):
        xk = emb[toks[:, i - 1]]
        own.append((xk @ wk).view(N, 1, Hk, D), (xk @ wv).view(N, 1, Hk, D))
        again.append(cached_attention(qs[i], own, scale, prefix=shared).output)
    attn.check(cached_attention(q, own, scale, prefix=shared), attn.reference(q, own, True, range(N), [S] * N, shared, 0, scale), torch.float32)
    for o, y0 in zip(again, logits[S // 2:]):
        assert torch.equal(o.view(N, H * D) @ w, y0)


def test_threads_streams_and_graphs_beside_each_other():
    """Attention and scores that need workspaces, from several threads on one stream, on streams of their own, and replayed from
    graphs beside them: each gets its own result."""
    import threading

    from dirktensor_amd import KVCache, cached_attention, token_logprobs

    B, H, L, V = 3, 4, 3000, 50021
    c = KVCache(B, L, H)
    c.append(randn((B, L, H, D), 30), randn((B, L, H, D), 31))
    qs = [randn((B, 1, H, D), 32 + i) for i in range(4)]
    xs = [randn((2 + i, V), 40 + i, 3.0) for i in range(4)]
    toks = [torch.arange(len(x), device="cuda") for x in xs]
    call = lambda i: (cached_attention(qs[i], c, 0.09).output, token_logprobs(xs[i], toks[i], top_k=9))
    want = [call(i) for i in range(4)]
    torch.cuda.synchronize()

    def same(got, i):
        assert torch.equal(got[0], want[i][0]) and torch.equal(got[1].top_index, want[i][1].top_index)
        assert torch.equal(got[1].logprob, want[i][1].logprob) and torch.equal(got[1].top_logprob, want[i][1].top_logprob)

    side = torch.cuda.Stream()
    graphs = []
    for i in (0, 1):  # (captured on one stream: they may not share a workspace with each other or with eager calls there)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            r = call(i)
        graphs.append((g, r))
    replayers = [torch.cuda.Stream() for _ in graphs]
    got, errors = [[] for _ in range(4)], []

    def work(i, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(40):
                    got[i].append(call(i))
        except Exception as e:  # (shown below)
            errors.append(e)

    streams = [torch.cuda.default_stream()] * 2 + [side, torch.cuda.Stream()]
    threads = [threading.Thread(target=work, args=(i, streams[i])) for i in range(4)]
    for t in threads:
        t.start()
    for _ in range(10):
        for (g, _), s in zip(graphs, replayers):
            with torch.cuda.stream(s):
                g.replay()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(4):
        assert len(got[i]) == 40
        for r in got[i]:
            same(r, i)
    for i, (_, r) in enumerate(graphs):
        same(r, i)


def test_workspaces_grow_with_the_call():
    from dirktensor_amd import KVCache, cached_attention

    c = KVCache(64, 6000, 8)
    x = randn((64, 6000, 8, D), 60).bfloat16()
    c.append(x, x)
    torch.cuda.synchronize()  # (calls on one cache are ordered by their caller)
    stream = torch.cuda.Stream()  # (nothing kept for it yet)
    with torch.cuda.stream(stream):
        for B, T in ((1, 1), (16, 2), (64, 1), (2, 1), (5, 40), (64, 9)):
            q = randn((B, T, 32, D), 61).bfloat16()
            r, again = cached_attention(q, c, 0.09), cached_attention(q, c, 0.09)
            assert torch.equal(r.output, again.output) and bool(torch.isfinite(r.output.float()).all())
            for b in (0, B - 1):
                attn.check(type(r)(r.output[b:b + 1], r.softmax_m[b:b + 1], r.softmax_l[b:b + 1]),
                           attn.reference(q[b:b + 1], c, True, [b], [T], None, 0, 0.09), torch.bfloat16)
