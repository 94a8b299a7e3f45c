"""The operators that answer with a model and score its answers, as a program built on this package calls them.

    cache_rows   KVCache.append of new key and value rows, quantised as they are written, and KVCache.read of the
                 same rows
    attn         cached_attention of the newest tokens over the cache, with or without a prefix that the whole
                 batch shares
    logprobs     token_logprobs: log probabilities of given tokens, with the entropy and the top alternatives
    logprobs_bwd token_logprobs_backward: the logits' gradient from those of the log probabilities and entropies

``listed()`` names the measured cases, ``draw(rng)`` takes one more from the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one call (its plain form unless ``own`` is set), ``work`` counts what it
cannot do without and ``exact`` computes the result in 64 bits.

Rows are held by (token, head): 128 values with one scale.
    int8  scale = amax / 127 in 32 bits; q = x / scale to the nearest whole number, ties to even
    fp8   scale = the smallest power of two with amax / scale <= 448; q = x / scale as e4m3, ties to even
    bf16  q = x as bf16, scale 1
"""

import math

import numpy as np
import torch

own = False

D = 128                  # head size
SCALE = 1.0 / math.sqrt(D)
DEV = "cuda:0"


# ---- the cases ------------------------------------------------------------------------------------------------


def listed():
    return [
        # one token of each of eight conversations enters the cache: the launches count
        dict(name="cache_rows_int8_step_b8", kind="cache_rows", format="int8", mode="bf16", B=8, T=1, Hk=16,
             capacity=2048),
        # a long prompt's keys and values enter the cache
        dict(name="cache_rows_fp8_t4096", kind="cache_rows", format="fp8", mode="bf16", B=2, T=4096, Hk=16,
             capacity=8192),
        # the next token of one conversation of ordinary length, unquantised: latency
        dict(name="attn_bf16_b1_t1000", kind="attn", format="bf16", mode="bf16", B=1, T=1, H=16, Hk=16, prefix=0,
             length=1000, ragged=False),
        # the next tokens of sixteen conversations of different lengths
        dict(name="attn_int8_b16_ragged", kind="attn", format="int8", mode="bf16", B=16, T=1, H=16, Hk=16, prefix=0,
             length=4096, ragged=True),
        # the next tokens of a full batch at the longest context: the cache's bytes are all that counts
        dict(name="attn_fp8_b32_t8192", kind="attn", format="fp8", mode="bf16", B=32, T=1, H=16, Hk=16, prefix=0,
             length=8192, ragged=False),
        # many answers sampled to one prompt: the prompt is read once for all of them
        dict(name="attn_int8_b64_prefix4096", kind="attn", format="int8", mode="bf16", B=64, T=1, H=16, Hk=16,
             prefix=4096, length=512, ragged=True),
        # several tokens a sequence at once (a draft that is verified), behind a shared prompt of odd length
        dict(name="attn_fp8_b12_t5_prefix2777", kind="attn", format="fp8", mode="bf16", B=12, T=5, H=16, Hk=16,
             prefix=2777, length=300, ragged=True),
        # exact mode
        dict(name="attn_int8_fp32_b4_t1500", kind="attn", format="int8", mode="fp32", B=4, T=1, H=16, Hk=16, prefix=0,
             length=1500, ragged=False),
        # the sampled tokens of a step's batch are scored, with twenty alternatives each
        dict(name="logprobs_fp32_rows16_top20", kind="logprobs", mode="fp32", rows=16, V=100352, top_k=20),
        # a sequence is scored at every position, with five alternatives
        dict(name="logprobs_fp32_rows2048_top5", kind="logprobs", mode="fp32", rows=2048, V=100352, top_k=5),
        # the gradient that a policy's training starts from, short rows of an odd vocabulary
        dict(name="logprobs_bwd_bf16_rows300", kind="logprobs_bwd", mode="bf16", rows=300, V=50277),
        # and over a whole sequence and vocabulary
        dict(name="logprobs_bwd_fp32_rows2048", kind="logprobs_bwd", mode="fp32", rows=2048, V=100352),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cache_rows", "attn", "attn", "attn", "logprobs", "logprobs_bwd"])
    mode = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "cache_rows":
        B = _log_int(rng, 1, 32)
        T = _log_int(rng, 1, 8192 // B)
        return dict(kind=kind, format=rng.choice(["int8", "fp8", "bf16"]), mode=mode, B=B, T=T,
                    Hk=rng.choice([2, 4, 16, 16]), capacity=T + _log_int(rng, 1, 4096))
    if kind == "attn":
        H = rng.choice([4, 16, 16, 16])
        Hk = rng.choice([H, H, H, H // 4])
        T = rng.choice([1, 1, 1, _log_int(rng, 2, 128)])
        B = _log_int(rng, 1, 64 if T < 8 else 8)
        prefix = rng.choice([0, _log_int(rng, 33, 8192)])
        length = T + _log_int(rng, 1, min(8192, 131072 // B))
        return dict(kind=kind, format=rng.choice(["int8", "fp8", "bf16"]), mode=mode, B=B, T=T, H=H, Hk=Hk,
                    prefix=prefix, length=length, ragged=B > 1 and rng.random() < 0.6)
    V = _log_int(rng, 1000, 120000)
    rows = _log_int(rng, 1, min(2048, 200000000 // V))
    if kind == "logprobs":
        return dict(kind=kind, mode=mode, rows=rows, V=V, top_k=rng.randint(0, 32))
    return dict(kind=kind, mode=mode, rows=rows, V=V)


# ---- inputs ---------------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _tdt(case):
    return torch.bfloat16 if case["mode"] == "bf16" else torch.float32


def _randn(g, shape, tdt):
    return torch.randn(shape, generator=g, device=DEV).to(tdt)


def _rows(case, g, B, T):
    """Keys as the norm and the rotation leave them, values of token-dependent size: [B, T, Hk, D] each."""
    k = _randn(g, (B, T, case["Hk"], D), _tdt(case))
    v = torch.randn((B, T, case["Hk"], D), generator=g, device=DEV)
    v *= torch.exp(0.5 * torch.randn((B, T, 1, 1), generator=g, device=DEV))
    return k, v.to(_tdt(case))


def _lengths(case, seed):
    """Tokens of each sequence, the T newest among them; the longest has ``length``."""
    L = np.full(case["B"], case["length"], np.int32)
    if case["ragged"]:
        rng = np.random.default_rng(int(seed) + 7)
        L = rng.integers(case["T"], case["length"] + 1, size=case["B"]).astype(np.int32)
        L[int(rng.integers(case["B"]))] = case["length"]
    return L


def _starts(case, seed):
    """Tokens that the cache holds before the new rows."""
    rng = np.random.default_rng(int(seed) + 9)
    return rng.integers(0, case["capacity"] - case["T"] + 1, size=case["B"]).astype(np.int32)


def _attn_inputs(case, seed):
    """Queries [B, T, H, D] and the rows of the cache [B, length, Hk, D], of the prefix [1, prefix, Hk, D]."""
    g = _gen(seed)
    q = _randn(g, (case["B"], case["T"], case["H"], D), _tdt(case))
    k, v = _rows(case, g, case["B"], case["length"])
    pk, pv = _rows(case, g, 1, case["prefix"]) if case["prefix"] else (None, None)
    return q, k, v, pk, pv


def _logits(case, seed):
    """Logits of a trained model: broad, with one row in two sure of its token; tokens to score, half of them the
    likeliest."""
    g = _gen(seed)
    rows, V = case["rows"], case["V"]
    x = 2.5 * torch.randn((rows, V), generator=g, device=DEV)
    peak = torch.randint(0, V, (rows,), generator=g, device=DEV)
    lift = torch.where(torch.rand((rows,), generator=g, device=DEV) < 0.5, 18.0, 6.0)
    x[torch.arange(rows, device=DEV), peak] += lift
    other = torch.randint(0, V, (rows,), generator=g, device=DEV)
    tok = torch.where(torch.rand((rows,), generator=g, device=DEV) < 0.5, peak, other).to(torch.int32)
    return x.to(_tdt(case)), tok


def _grads(case, seed):
    """The advantages of the scored tokens and the weights of the entropies."""
    g = _gen(seed + 1000003)
    return (torch.randn((case["rows"],), generator=g, device=DEV) / case["rows"],
            0.01 * torch.rand((case["rows"],), generator=g, device=DEV) / case["rows"])


# ---- the plain forms ------------------------------------------------------------------------------------------


def _plain_quant(x, fmt):
    """What the cache holds of rows x [..., D]: (q, scale [..., 1])."""
    x = x.float()
    if fmt == "bf16":
        return x.bfloat16(), torch.ones_like(x[..., :1])
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        scale = (amax.double() / 127.0).float()  # (the nearest in 32 bits: a division by a number need not be)
        q = torch.round(x.double() / scale.clamp_min(1e-45).double()).clamp(-127, 127)  # (64 bits at the borders)
        return q.to(torch.int8), scale
    mant, expo = torch.frexp(amax)  # amax = mant 2^expo, mant in [0.5, 1): 448 = 0.875 2^9
    e = (expo - 9 + (mant > 0.875).int()).clamp_min(-126)
    scale = torch.ldexp(torch.ones_like(amax), e)
    return (x / scale).to(torch.float8_e4m3fn), scale


def _plain_value(q, scale):
    return q.float() * scale


def _plain_attention(q, kc, vc, lens, prefix):
    """q [B, T, H, D]; kc, vc the held rows (q, scale) of [B, L, Hk, D]; prefix None or those of [1, P, Hk, D]."""
    B, T, H, _ = q.shape
    Hk, L = kc[0].shape[2], kc[0].shape[1]
    G = H // Hk
    # [B, Hk, G T, D]: the queries that share a head's keys
    Q = q.float().reshape(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    K = _plain_value(*kc).permute(0, 2, 3, 1).contiguous()
    S = torch.matmul(Q, K) * SCALE
    pos = torch.arange(L, device=q.device)
    last = lens[:, None] - T + torch.arange(T, device=q.device)[None, :]          # [B, T]: the newest visible key
    hide = pos[None, None, :] > last[:, :, None]                                  # [B, T, L]
    S = S.reshape(B, Hk, G, T, L).masked_fill(hide[:, None, None], float("-inf")).reshape(B, Hk, G * T, L)
    m = S.amax(-1, keepdim=True)
    if prefix is not None:
        P = prefix[0][0].shape[1]
        PK = _plain_value(*prefix[0])[0].permute(1, 2, 0).contiguous()            # [Hk, D, P]
        QP = Q.permute(1, 0, 2, 3).reshape(Hk, B * G * T, D)
        SP = (torch.matmul(QP, PK) * SCALE).reshape(Hk, B, G * T, P).permute(1, 0, 2, 3)
        m = torch.maximum(m, SP.amax(-1, keepdim=True))
    E = torch.exp(S - m)
    l = E.sum(-1, keepdim=True)
    O = torch.matmul(E, _plain_value(*vc).permute(0, 2, 1, 3).contiguous())
    if prefix is not None:
        EP = torch.exp(SP - m)
        l = l + EP.sum(-1, keepdim=True)
        PV = _plain_value(*prefix[1])[0].permute(1, 0, 2).contiguous()            # [Hk, P, D]
        EPh = EP.permute(1, 0, 2, 3).reshape(Hk, B * G * T, P)
        O = O + torch.matmul(EPh, PV).reshape(Hk, B, G * T, D).permute(1, 0, 2, 3)
    O = (O / l).reshape(B, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    stat = lambda t: t[..., 0].reshape(B, Hk, G, T).permute(0, 3, 1, 2).reshape(B, T, H).contiguous()
    return O.to(q.dtype), stat(m), stat(l)


def _plain_logprobs(logits, tok, top_k):
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    l = e.sum(-1, keepdim=True)
    logl = torch.log(l)
    entropy = logl[:, 0] - (e * d).sum(-1) / l[:, 0]
    lp = d.gather(1, tok.long()[:, None])[:, 0] - logl[:, 0]
    out = [lp, entropy, m[:, 0], l[:, 0]]
    if top_k:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top_k]
        out += [order.to(torch.int32), d.gather(1, order) - logl]
    return out


def _plain_logprobs_bwd(logits, tok, m, l, entropy, g, h):
    lp = logits.float() - m[:, None] - torch.log(l)[:, None]
    p = torch.exp(lp)
    d = -p * (g[:, None] + h[:, None] * (lp + entropy[:, None]))
    d.scatter_add_(1, tok.long()[:, None], g[:, None])
    return d.to(logits.dtype)


# ---- one call -------------------------------------------------------------------------------------------------


def prepare(case, seed):
    st = dict(case=case)
    if case["kind"] == "cache_rows":
        st["k"], st["v"] = _rows(case, _gen(seed), case["B"], case["T"])
        st["starts"] = _starts(case, seed)
        if own:
            import dirktensor_amd as dt

            st["cache"] = dt.KVCache(case["B"], case["capacity"], case["Hk"], format=case["format"])
            lo = int(st["starts"].max())
            if lo:  # what the cache holds already
                z = torch.zeros((case["B"], lo, case["Hk"], D), dtype=_tdt(case), device=DEV)
                st["cache"].append(z, z)
        else:
            shape = (case["B"], case["capacity"], case["Hk"])
            qdt = dict(int8=torch.int8, fp8=torch.float8_e4m3fn, bf16=torch.bfloat16)[case["format"]]
            st["held"] = [(torch.zeros((*shape, D), device=DEV).to(qdt), torch.zeros((*shape, 1), device=DEV))
                          for _ in range(2)]
            pos = torch.as_tensor(st["starts"], device=DEV).long()[:, None] + torch.arange(case["T"], device=DEV)
            st["at"] = (torch.arange(case["B"], device=DEV)[:, None].expand_as(pos), pos)
    elif case["kind"] == "attn":
        q, k, v, pk, pv = _attn_inputs(case, seed)
        lens = _lengths(case, seed)
        st["q"] = q
        if own:
            import dirktensor_amd as dt

            st["cache"] = dt.KVCache(case["B"], case["length"], case["Hk"], format=case["format"])
            st["cache"].append(k, v, counts=lens)
            st["prefix"] = None
            if pk is not None:
                st["prefix"] = dt.KVCache(1, case["prefix"], case["Hk"], format=case["format"])
                st["prefix"].append(pk, pv)
        else:
            st["kc"], st["vc"] = _plain_quant(k, case["format"]), _plain_quant(v, case["format"])
            st["prefix"] = None
            if pk is not None:
                st["prefix"] = (_plain_quant(pk, case["format"]), _plain_quant(pv, case["format"]))
            st["lens"] = torch.as_tensor(lens, device=DEV).long()
    else:
        st["x"], st["tok"] = _logits(case, seed)
        if case["kind"] == "logprobs_bwd":
            st["g"], st["h"] = _grads(case, seed)
            if own:
                import dirktensor_amd as dt

                st["fwd"] = dt.token_logprobs(st["x"], st["tok"])
            else:
                _, st["ent"], st["m"], st["l"] = _plain_logprobs(st["x"], st["tok"], 0)
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    case = st["case"]
    if case["kind"] == "cache_rows":
        out = []
        for x, (hq, hs) in zip((st["k"], st["v"]), st["held"]):
            q, scale = _plain_quant(x, case["format"])
            # (indexed writes go by bytes where a type of 8 bits has none of its own)
            hb, qb = (hq.view(torch.int8), q.view(torch.int8)) if q.element_size() == 1 else (hq, q)
            hb[st["at"]] = qb
            hs[st["at"]] = scale
            out.append(_plain_value(hb[st["at"]].view(q.dtype), hs[st["at"]]).to(x.dtype))
        return out
    if case["kind"] == "attn":
        return _plain_attention(st["q"], st["kc"], st["vc"], st["lens"], st["prefix"])
    if case["kind"] == "logprobs":
        return _plain_logprobs(st["x"], st["tok"], case["top_k"])
    return _plain_logprobs_bwd(st["x"], st["tok"], st["m"], st["l"], st["ent"], st["g"], st["h"])


def _run_own(st):
    import dirktensor_amd as dt

    case = st["case"]
    if case["kind"] == "cache_rows":
        cache = st["cache"]
        cache.truncate(st["starts"])
        cache.append(st["k"], st["v"])
        return list(cache.read(st["starts"], case["T"], mode=case["mode"]))
    if case["kind"] == "attn":
        r = dt.cached_attention(st["q"], st["cache"], SCALE, prefix=st["prefix"])
        return r.output, r.softmax_m, r.softmax_l
    if case["kind"] == "logprobs":
        r = dt.token_logprobs(st["x"], st["tok"], top_k=case["top_k"])
        out = [r.logprob, r.entropy, r.softmax_m, r.softmax_l]
        return out + [r.top_index, r.top_logprob] if case["top_k"] else out
    return dt.token_logprobs_backward(st["g"], st["x"], st["tok"], st["fwd"], d_entropy=st["h"])


# ---- what a call cannot do without ----------------------------------------------------------------------------


def work(case):
    es = 2 if case["mode"] == "bf16" else 4
    held = lambda n: n * (D * 2 if case["format"] == "bf16" else D + 4)  # (int8 and fp8 with a scale of 32 bits)
    if case["kind"] == "cache_rows":
        n = case["B"] * case["T"] * case["Hk"]
        return dict(bytes=2 * (2 * n * D * es + 2 * held(n)), flops=2 * n * D * 4)
    if case["kind"] == "attn":
        lens = _lengths(case, 0)  # (of one seed; the others' are alike)
        keys = int(lens.sum())
        rows = case["B"] * case["T"] * case["H"]
        pairs = keys * case["T"] * case["H"] + rows * case["prefix"]
        return dict(bytes=2 * held((keys + case["prefix"]) * case["Hk"]) + 2 * rows * D * es + 8 * rows,
                    flops=4 * pairs * D)
    n = case["rows"] * case["V"]
    if case["kind"] == "logprobs":
        return dict(bytes=n * es + case["rows"] * (20 + 8 * case["top_k"]), flops=6 * n)
    return dict(bytes=2 * n * es + case["rows"] * 24, flops=8 * n)


# ---- 64 bits --------------------------------------------------------------------------------------------------


def _held64(x, fmt):
    """The values that the cache stands for, row by row, from their definition."""
    x = x.double()
    if fmt == "bf16":
        return x.to(torch.float32).to(torch.bfloat16).double()
    top = x.abs().max(dim=-1, keepdim=True).values
    if fmt == "int8":
        step = (top / 127).float().double()
        near = torch.where(step > 0, x / step, torch.zeros_like(x)).round()
        return near.clamp(-127, 127) * step
    # fp8: to a multiple of the row's power of two times e4m3's step at that size (3 bits behind the leading one,
    # 2^-9 at the least)
    step = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -120) / 448)).clamp_min(-126))
    step = torch.where(top > 448 * step, 2 * step, step)
    step = torch.where(top <= 448 * (step / 2), step / 2, step).clamp_min(2.0 ** -126)
    y = x / step
    ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (y / ulp).round() * ulp * step


def exact(case, seed):
    if case["kind"] == "cache_rows":
        return [_held64(x, case["format"]) for x in _rows(case, _gen(seed), case["B"], case["T"])]
    if case["kind"] == "attn":
        return _exact_attn(case, seed)
    x, tok = _logits(case, seed)
    g, h = _grads(case, seed)
    parts = []
    for lo in range(0, case["rows"], 64):  # (64 rows of 64-bit values at a time)
        z, t = x[lo:lo + 64].double(), tok[lo:lo + 64].long()
        r = torch.arange(len(t), device=z.device)
        top = z.max(-1).values
        lse = torch.logsumexp(z, -1)
        lp = z - lse[:, None]
        p = lp.exp()
        ent = -(p * lp).sum(-1)
        if case["kind"] == "logprobs":
            part = [lp[r, t], ent, top, (lse - top).exp()]
            if case["top_k"]:
                # the largest left, the first of equals, one after another
                idx, left = [], z.clone()
                for _ in range(case["top_k"]):
                    best = left.max(-1, keepdim=True).values
                    at = (left == best).to(torch.int8).argmax(-1)
                    idx.append(at)
                    left[r, at] = float("-inf")
                idx = torch.stack(idx, -1)
                part += [idx.to(torch.int32), lp.gather(1, idx)]
        else:
            gr, hr = g[lo:lo + 64].double(), h[lo:lo + 64].double()
            dz = -p * gr[:, None] - hr[:, None] * p * (lp + ent[:, None])
            dz[r, t] += gr
            part = [dz]
        parts.append(part)
    out = [torch.cat(c) for c in zip(*parts)]
    return out if case["kind"] == "logprobs" else out[0]


def _exact_attn(case, seed):
    q, k, v, pk, pv = _attn_inputs(case, seed)
    lens = _lengths(case, seed)
    B, T, H, G = case["B"], case["T"], case["H"], case["H"] // case["Hk"]
    O = torch.empty((B, T, H, D), dtype=torch.float64, device=DEV)
    m = torch.empty((B, T, H), dtype=torch.float64, device=DEV)
    l = torch.empty_like(m)
    if pk is not None:
        pk, pv = _held64(pk, case["format"])[0], _held64(pv, case["format"])[0]
    for b in range(B):
        n = int(lens[b])
        kb, vb = _held64(k[b, :n], case["format"]), _held64(v[b, :n], case["format"])
        first = torch.arange(n, device=DEV)
        if pk is not None:
            kb, vb = torch.cat([pk, kb]), torch.cat([pv, vb])
            first = torch.cat([torch.full((len(pk),), -1, device=DEV), first])
        seen = first[None, :] <= n - T + torch.arange(T, device=DEV)[:, None]
        for h in range(H):
            s = q[b, :, h].double() @ kb[:, h // G].t().contiguous() * SCALE
            s = torch.where(seen, s, torch.full_like(s, float("-inf")))
            m[b, :, h] = s.max(-1).values
            w = (s - m[b, :, h, None]).exp()
            l[b, :, h] = w.sum(-1)
            O[b, :, h] = w @ vb[:, h // G].contiguous() / l[b, :, h, None]
    return O, m, l
