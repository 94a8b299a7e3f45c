"""Verified drafts against the definition in 64 bits: tokens and counts are the same, log probabilities are off by their rounding to
32 bits (2^-24 of them), what is left of 64, and the error of the row's sum: its largest term is exact, another 2^t (t <= 0, the
difference of the logits times log2 e / T) is off by 2^-24 (2 |t| ln 2) for the difference and the product and by 2^-23 for the power:
the logarithm of the sum by sum p (1.4 |t| + 2) 2^-24 over all but the largest.

A token next to a border: the kernel's powers are off by 1.1e-12, so a row's sum is too, and an exponent x / T log2 e of at most 1500
by 2^-52 of it, 4e-13: a probability by less than 5e-12 of itself (in the reference by 1e-12). Sums over p and q, which are 1 each,
are off by 1e-11, and the border, a share of their total, by as much. So another token is right as well if the border lies within
BORDER of its weight's place in the sum: where p and q are that close (0.01 as temperature of rows that both hold one token), or
with a probability of about the vocabulary times 2e-11."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
BORDER = 2e-11


def dt():
    import dirktensor_amd

    return dirktensor_amd


def inputs(B, K, V, seed, tdt, draft=True, peak=6.0, masked=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2 * torch.randn((B, K + 1, V), generator=g, device="cuda")
    x[torch.rand((B, K + 1, V), generator=g, device="cuda") < 2.0 / V] += peak
    if masked:
        hide = torch.rand((B, 1, V), generator=g, device="cuda") < 0.6
        hide[..., seed % V] = False
        x = x.masked_fill(hide, float("-inf"))
    y = (x[:, :K] + 0.7 * torch.randn((B, K, V), generator=g, device="cuda")).to(tdt) if draft else None
    u = torch.rand((B, K + 1), generator=g, device="cuda")
    if draft and K:
        p = torch.softmax(y.double(), -1).reshape(B * K, V)
        drafts = (p.cumsum(-1) < torch.rand((B * K, 1), generator=g, device="cuda")).sum(-1).clamp_max(V - 1).reshape(B, K)
    else:
        drafts = torch.where(torch.rand((B, K), generator=g, device="cuda") < 0.7, x[:, :K].argmax(-1),
                             torch.randint(0, V, (B, K), generator=g, device="cuda"))
    return x.to(tdt), drafts.int(), u, y


def reference(x, drafts, u, y, T, counts=None):
    B, K = drafts.shape
    V = x.shape[2]
    acc, tok = np.zeros(B, np.int64), np.full((B, K + 1), -1)
    score, slack = np.zeros((B, K + 1)), np.zeros((B, K + 1))
    others = {}  # tokens as right as the one named, with their scores
    for b in range(B):
        n = K if counts is None else int(counts[b])
        z = x[b].double()
        lp = torch.log_softmax(z / T if T else z, -1)
        for i in range(n + 1):
            d = int(drafts[b, i]) if i < n else -1
            known = 0 <= d < V
            valid = not bool(torch.isnan(lp[i]).any()) and bool(torch.isfinite(z[i].max()))
            taken, token = False, -1
            if T == 0:
                token = int((z[i] == z[i].max()).nonzero()[0]) if valid else -1
                taken = i < n and valid and d == token
            elif valid:
                p = lp[i].exp()
                q = None
                if i < n:
                    if y is not None:
                        q = torch.log_softmax(y[b, i].double() / T, -1).exp()  # (as p is: equal rows give equal numbers)
                        q = q if bool(torch.isfinite(q).all()) else torch.full_like(q, float("nan"))
                    else:
                        q = torch.zeros_like(p)
                        if known:
                            q[d] = 1.0
                    taken = known and float(u[b, i]) * float(q[d]) < float(p[d])
                if not taken:
                    w = p if q is None else (p - q).clamp_min(0) if y is not None else torch.where(q > 0, torch.zeros_like(p), p)
                    c = w.cumsum(0)
                    if float(c[-1]) == 0:
                        c = p.cumsum(0)
                    if bool(torch.isnan(c[-1])):
                        token = -1
                    else:
                        over = c > float(u[b, K]) * c[-1]
                        near = (c - float(u[b, K]) * c[-1]).abs()
                        near = torch.minimum(near, torch.cat([near.new_zeros(1) + float(u[b, K]) * c[-1], near[:-1]])) <= BORDER
                        others[b] = {int(j): float(lp[i, j]) for j in near.nonzero()[:, 0]} if int(near.sum()) <= 4096 else {}
                        token = int(over.nonzero()[0]) if bool(over.any()) else int((w > 0).nonzero()[-1])
            if taken:
                token = d
            tok[b, i] = token
            t = (lp[i].max() - lp[i]) / np.log(2)
            p = lp[i].exp()
            slack[b, i] = 2.0 ** -24 * float(torch.where(p > 0, p * (1.4 * t + 2), p).sum() - 2 * p.max())
            score[b, i] = float(lp[i, token]) if token >= 0 else np.nan
            if not taken:
                break
            acc[b] += 1
    return acc, tok, score, slack, others


def check(r, ref):
    acc, tok, score, slack, others = ref
    tok, score = tok.copy(), score.copy()
    for b, n in enumerate(acc):
        got = int(r.tokens[b, n])
        if got != tok[b, n] and got in others.get(b, {}):
            tok[b, n], score[b, n] = got, others[b][got]
    np.testing.assert_array_equal(np.asarray(r.accepted.cpu() if torch.is_tensor(r.accepted) else r.accepted), acc)
    np.testing.assert_array_equal(np.asarray(r.tokens.cpu() if torch.is_tensor(r.tokens) else r.tokens), tok)
    got = np.asarray(r.logprob.cpu() if torch.is_tensor(r.logprob) else r.logprob).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(score))
    ok = ~np.isnan(score)
    assert (np.abs(got - score)[ok] <= 2.0 ** -24 * np.abs(score)[ok] + slack[ok] + 1e-10).all()


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("T", [1.0, 0.6, 0.0])
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (2, 1, 2), (3, 2, 7), (5, 3, 8), (4, 3, 9), (3, 4, 2047), (2, 3, 2048), (3, 2, 2049), (33, 2, 4097),
                                   (2, 64, 301), (3, 5, 50277)])
def test_tokens(gpu, tdt, draft, T, B, K, V):
    x, d, u, y = inputs(B, K, V, B + K + V, tdt, draft)
    check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T), reference(x, d, u, y, T))


@pytest.mark.parametrize("draft", [True, False])
def test_a_large_vocabulary(gpu, draft):
    """More chunks than threads: a thread's chunk has several runs."""
    x, d, u, y = inputs(2, 1, 600011, 6, torch.bfloat16, draft)
    check(dt().verify_drafts(x, d, u, draft_logits=y), reference(x, d, u, y, 1.0))
    x[:, :, :500000] = float("-inf")
    u[:] = 1.0 - 2.0 ** -24
    check(dt().verify_drafts(x, d, u, draft_logits=y), reference(x, d, u, y, 1.0))


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("T", [0.01, 30.0])
def test_temperatures(gpu, draft, T):
    x, d, u, y = inputs(6, 3, 1001, 5, torch.float32, draft)
    check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T), reference(x, d, u, y, T))


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("T", [1.0, 0.0])
def test_ragged_counts_masks_and_int64(gpu, draft, T):
    B, K, V = 40, 4, 3001
    x, d, u, y = inputs(B, K, V, 7, torch.bfloat16, draft, masked=True)
    counts = np.arange(B) % (K + 1)
    want = reference(x, d, u, y, T, counts)
    for b in range(B):  # (the rows behind the counts are not read)
        x[b, counts[b] + 1:] = float("nan")
        if y is not None:
            y[b, counts[b]:] = float("nan")
    r = dt().verify_drafts(x, d.long(), u, draft_logits=y, temperature=T, counts=counts)
    check(r, want)
    check(dt().verify_drafts(x, d, u, draft_logits=y, temperature=T, counts=torch.as_tensor(counts)), want)


def test_ends_of_the_uniforms(gpu):
    """0 takes the first token that has a weight, the number below 1 the last region; a draft at u = 0 is taken if p > 0."""
    B, K, V = 6, 2, 5000
    x, d, u, y = inputs(B, K, V, 3, torch.float32, masked=True)
    for v in (0.0, 1.0 - 2.0 ** -24):
        for w in (0.0, 1.0 - 2.0 ** -24):
            u[:, :K], u[:, K] = v, w
            check(dt().verify_drafts(x, d, u, draft_logits=y), reference(x, d, u, y, 1.0))
            check(dt().verify_drafts(x, d, u), reference(x, d, u, None, 1.0))


def test_equal_rows_leave_nothing(gpu):
    """p = q and a draft that neither allows: the token comes from p."""
    B, V = 3, 2500
    x, _, u, _ = inputs(B, 1, V, 9, torch.float32)
    x[:, 0, 77] = float("-inf")
    d = torch.full((B, 1), 77, dtype=torch.int32, device="cuda")
    y = x[:, :1].clone()
    r = dt().verify_drafts(x, d, u, draft_logits=y)
    check(r, reference(x, d, u, y, 1.0))
    assert bool((r.accepted == 0).all()) and bool((r.tokens[:, 0] >= 0).all())
    # a draft of probability one is taken, whatever is drawn
    x[:, 0] = float("-inf")
    x[:, 0, 77] = -3e38
    check(dt().verify_drafts(x, d, u), reference(x, d, u, None, 1.0))


@pytest.mark.parametrize("T", [1.0, 0.0])
def test_ties_take_the_lowest_index(gpu, T):
    B, K, V = 4, 1, 9000
    x = torch.zeros((B, K + 1, V), device="cuda")
    x[1, :, 4000:] = 3.0
    x[2, 0, [8191, 8192, 300]] = 50.0
    x[3] = torch.finfo(torch.float32).min  # (a mask of the type's lowest value: all equal)
    d = torch.tensor([[0], [4000], [300], [1]], dtype=torch.int32, device="cuda")
    u = torch.full((B, K + 1), 0.25, device="cuda")
    check(dt().verify_drafts(x, d, u, temperature=T), reference(x, d, u, None, T))


@pytest.mark.parametrize("T", [1.0, 0.0])
@pytest.mark.parametrize("what", ["nan", "inf", "empty"])
@pytest.mark.parametrize("where", ["target", "draft", "last"])
def test_rows_that_are_none(gpu, T, what, where):
    B, K, V = 4, 3, 5000
    x, d, u, y = inputs(B, K, V, 11, torch.float32)
    u[:] = 0.0  # (what can be accepted is)
    if T == 0:
        d = x[:, :K].argmax(-1).int()
    rows = {"target": x[:, 1], "draft": y[:, 1], "last": x[:, K]}[where]
    if what == "empty":
        rows[:] = float("-inf")
    else:
        rows[:, 1234] = float(what)
    r = dt().verify_drafts(x, d, u, draft_logits=y, temperature=T)
    if T == 0 and where == "draft":
        assert bool((r.accepted == K).all())
        return
    assert bool((r.accepted == (K if where == "last" else 1)).all())
    at = K if where == "last" else 1
    assert bool((r.tokens[:, at] == -1).all()) and bool((r.tokens[:, :at] == d[:, :at]).all())
    if where != "draft":
        assert bool(torch.isnan(r.logprob[:, at]).all())
    assert not bool(torch.isnan(r.logprob[:, :at]).any())


def test_drafts_outside_the_vocabulary(gpu):
    B, K, V = 3, 2, 700
    x, d, u, y = inputs(B, K, V, 13, torch.float32)
    d[0, 0], d[1, 1], d[2, 0] = -1, V, 2**31 - 1
    for yy in (y, None):
        for T in (1.0, 0.0):
            want = reference(x, d, u, yy, T)
            check(dt().verify_drafts(x, d, u, draft_logits=yy, temperature=T), want)
            far = d.long()
            far[2, 0] = 2**40 + 5
            check(dt().verify_drafts(x, far, u, draft_logits=yy, temperature=T), want)


def test_strided_rows(gpu):
    B, K, V = 3, 2, 1003
    for tdt in TYPES:
        x, d, u, y = inputs(B, K, V, 15, tdt)
        want = reference(x, d, u, y, 1.0)
        wide = torch.full((B, K + 3, V + 5), float("nan"), dtype=tdt, device="cuda")
        wide[:, 1:K + 2, 3:V + 3] = x
        wide_y = torch.full((K, B, V + 1), float("nan"), dtype=tdt, device="cuda")
        wide_y[..., :V] = y.transpose(0, 1)
        check(dt().verify_drafts(wide[:, 1:K + 2, 3:V + 3], d.t().contiguous().t(), u, draft_logits=wide_y[..., :V].transpose(0, 1)), want)
        shared = x[:1].expand(B, -1, -1)  # (one row of logits for the whole batch)
        check(dt().verify_drafts(shared, d, u, draft_logits=y), reference(shared, d, u, y, 1.0))


def test_host_arrays(gpu):
    B, K, V = 3, 2, 1003
    for tdt in TYPES:
        for draft in (True, False):
            x, d, u, y = inputs(B, K, V, 17, tdt, draft)
            host = lambda t: (t.view(torch.int16).cpu().numpy().view(np.uint16) if t.dtype == torch.bfloat16 else t.cpu().numpy())
            r = dt().verify_drafts(host(x), host(d), host(u), draft_logits=host(y) if draft else None, temperature=0.9)
            check(r, reference(x, d, u, y, 0.9))
    r = dt().verify_drafts(host(x)[:, :1], np.zeros((B, 0), np.int32), host(u)[:, :1])
    check(r, reference(x[:, :1], d[:, :0], u[:, :1], None, 1.0))
    r = dt().verify_drafts(host(x), host(d), None, temperature=0)
    check(r, reference(x, d, u, None, 0))


def test_what_is_emitted_is_distributed_as_p(gpu):
    """Over a grid of the two random numbers and all drafts, each as often as q draws it. A grid of 16 places in the middles of
    its cells is off by at most 1/32 for each border that a token's region has: two of the drawing, one of the acceptance."""
    V, n = 5, 16
    g = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn((1, 2, V), generator=g, device="cuda").expand(n * n, 2, V)
    y = torch.randn((1, 1, V), generator=g, device="cuda").expand(n * n, 1, V)
    grid = (torch.arange(n, device="cuda") + 0.5) / n
    u = torch.stack([grid[:, None].expand(n, n), grid[None].expand(n, n)], -1).reshape(n * n, 2).float().contiguous()
    p, q = (torch.softmax(t[0, 0].double(), -1).cpu() for t in (x, y))
    seen = torch.zeros(V, dtype=torch.float64)
    for d in range(V):
        r = dt().verify_drafts(x, torch.full((n * n, 1), d, dtype=torch.int32, device="cuda"), u, draft_logits=y)
        seen += q[d] * torch.bincount(r.tokens[:, 0].cpu().long(), minlength=V).double() / (n * n)
    assert float((seen - p).abs().max()) <= 3 / 32, (seen, p)


def test_streams_and_graph_replays(gpu):
    shapes = [(2, 3, 20011), (17, 1, 5003)]
    ins = [inputs(*s, 23 + i, torch.float32) for i, s in enumerate(shapes)]
    call = lambda i: dt().verify_drafts(ins[i][0], ins[i][1], ins[i][2], draft_logits=ins[i][3])
    same = lambda a, b: torch.equal(a.accepted, b.accepted) and torch.equal(a.tokens, b.tokens) and torch.equal(a.logprob, b.logprob)
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in shapes]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same(r, want[i]) for r in got[i])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = call(0)
    for i in range(4):
        for a, b in zip(ins[0], inputs(*shapes[0], 50 + i, torch.float32)):
            a.copy_(b)
        call(1)
        g.replay()
        eager = call(0)
        torch.cuda.synchronize()
        assert same(r, eager)
        check(r, reference(*ins[0], 1.0))


def test_refusals(gpu):
    x, d, u, y = inputs(2, 3, 100, 1, torch.float32)
    bad = [dict(drafts=d[:, :2]), dict(uniforms=u[:, :2]), dict(draft_logits=y[:, :2]), dict(draft_logits=y.bfloat16()), dict(drafts=d.cpu()),
           dict(counts=[1]), dict(logits=x[0])]
    for kw in bad:
        a = dict(logits=x, drafts=d, uniforms=u)
        a.update(kw)
        with pytest.raises(ValueError):
            dt().verify_drafts(**a)
    for kw in (dict(drafts=d.float()), dict(uniforms=u.double())):
        a = dict(logits=x, drafts=d, uniforms=u)
        a.update(kw)
        with pytest.raises(TypeError):
            dt().verify_drafts(**a)
    for kw, msg in ((dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(counts=[0, 4]), "counts"),
                    (dict(uniforms=None), "uniforms")):
        a = dict(logits=x, drafts=d, uniforms=u)
        a.update(kw)
        with pytest.raises(dt().DTError, match=msg):
            dt().verify_drafts(**a)
    with pytest.raises(dt().DTError, match="K=65"):
        dt().verify_drafts(torch.zeros((1, 66, 10), device="cuda"), torch.zeros((1, 65), dtype=torch.int32, device="cuda"),
                           torch.zeros((1, 66), device="cuda"))
    with pytest.raises(dt().DTError, match="B=257"):
        dt().verify_drafts(torch.zeros((257, 1, 10), device="cuda"), torch.zeros((257, 0), dtype=torch.int32, device="cuda"),
                           torch.zeros((257, 1), device="cuda"))
    with pytest.raises(dt().DTError, match="draft 100"):
        dt().verify_drafts(x.cpu().numpy(), np.full((2, 3), 100, np.int32), u.cpu().numpy())
