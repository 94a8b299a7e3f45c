"""The operators of a generation step with drafted tokens, as a program built on this package calls them.

    rotary          queries and keys rotated to their positions (rotary, and rotary_backward for its gradient)
    head_norm       head_norm_rotary: each head's norm and the rotation in one pass
    head_norm_bwd   head_norm_rotary_backward: the gradients of rows and norm weights
    verify          verify_drafts: drafted tokens against the model's logits, from given random numbers
    cache_rows      KVCache.append and KVCache.read of rows in 4 bits
    attn            cached_attention over a cache in 4 bits

``listed()`` names the measured cases, ``draw(rng)`` takes one more from the same ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one call (its plain form unless ``own`` is set), ``work`` counts what it
cannot do without and ``exact`` computes the result in 64 bits.

Rows of 128 values in 4 bits: four groups of 32, each with a scale, the smallest power of two (at least 2^-120) with
amax / scale <= 6; a value is x / scale as e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), ties to even.
"""

import math

import numpy as np
import torch

own = False

D = 128                  # head size
SCALE = 1.0 / math.sqrt(D)
EPS = 1e-6
DEV = "cuda:0"


# ---- the cases ------------------------------------------------------------------------------------------------


def _rope(dims=128, layout="half", theta=500000.0, scaling="none", factor=1.0, original=8192, low=1.0, high=32.0,
          magnitude=1.0):
    return dict(dims=dims, layout=layout, theta=theta, scaling=scaling, factor=factor, original=original, low=low,
                high=high, magnitude=magnitude)


def listed():
    return [
        # the new token of each of eight conversations, a quarter of the head rotated: the launch counts
        dict(name="rotary_step_b8", kind="rotary", mode="bf16", backward=False, B=8, T=1, H=16, Hk=16, far=8192,
             positions="starts", **_rope(dims=32, layout="interleaved")),
        # the gradient of a long sequence's rotation, scaled for a context of a million positions, in exact mode
        dict(name="rotary_bwd_fp32_t8192", kind="rotary", mode="fp32", backward=True, B=2, T=8192, H=16, Hk=16,
             far=1 << 20, positions="given",
             **_rope(layout="interleaved", scaling="ramp", factor=16.0, magnitude=1.25)),
        # five tokens (a draft and the one before it) of twelve conversations, shared key heads
        dict(name="head_norm_b12_t5", kind="head_norm", mode="bf16", B=12, T=5, H=16, Hk=4, far=8192,
             positions="starts", **_rope()),
        # long prompts
        dict(name="head_norm_t4096", kind="head_norm", mode="bf16", B=4, T=4096, H=16, Hk=16, far=4096,
             positions="given", **_rope()),
        # a training step's gradients, odd length, part of the head rotated, in exact mode
        dict(name="head_norm_bwd_fp32_t777", kind="head_norm_bwd", mode="fp32", B=1, T=777, H=16, Hk=16, far=777,
             positions="none", **_rope(dims=96)),
        # and of a large batch with shared key heads
        dict(name="head_norm_bwd_t8192", kind="head_norm_bwd", mode="bf16", B=4, T=8192, H=16, Hk=4, far=8192,
             positions="none", **_rope()),
        # one conversation's four drafted tokens: latency
        dict(name="verify_fp32_b1_k4", kind="verify", mode="fp32", B=1, K=4, V=100352, draft=True, temperature=1.0,
             masked=False, ragged=False),
        # a full batch's drafts, of different numbers
        dict(name="verify_b64_k5", kind="verify", mode="bf16", B=64, K=5, V=100352, draft=True, temperature=0.8,
             masked=False, ragged=True),
        # five tokens of each of twelve conversations enter the cache
        dict(name="cache_rows_fp4_b12_t5", kind="cache_rows", mode="bf16", B=12, T=5, Hk=16, capacity=2048),
        # a long prompt's keys and values enter the cache
        dict(name="cache_rows_fp4_t4096", kind="cache_rows", mode="bf16", B=2, T=4096, Hk=16, capacity=8192),
        # five tokens of twelve conversations of different lengths, shared key heads, behind a shared prompt
        dict(name="attn_fp4_b12_t5_prefix2777", kind="attn", mode="bf16", B=12, T=5, H=16, Hk=4, prefix=2777,
             length=1500, ragged=True),
        # the next tokens of a full batch at the longest context: the cache's bytes are all that counts
        dict(name="attn_fp4_b32_t8192", kind="attn", mode="bf16", B=32, T=1, H=16, Hk=16, prefix=0, length=8192,
             ragged=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "head_norm", "head_norm_bwd", "verify", "verify", "cache_rows", "attn", "attn"])
    mode = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("rotary", "head_norm", "head_norm_bwd"):
        H = rng.choice([4, 16, 16, 12])
        B = _log_int(rng, 1, 32)
        T = _log_int(rng, 1, 16384 // B)
        scaling = rng.choice(["none", "none", "linear", "theta", "ramp"])
        far = max(T, _log_int(rng, 64, 1 << 20))
        case = dict(kind=kind, mode=mode, B=B, T=T, H=H, Hk=rng.choice([H, H, H // 4, 1]), far=far,
                    positions=rng.choice(["none", "starts", "given"]),
                    **_rope(dims=rng.choice([128, 128, 96, 64, 32, 16]), layout=rng.choice(["half", "interleaved"]),
                            scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 40.0]),
                            magnitude=rng.choice([1.0, 1.0, 1.2])))
        if kind == "rotary":
            case["backward"] = rng.random() < 0.4
        return case
    if kind == "verify":
        V = _log_int(rng, 1000, 120000)
        K = rng.choice([0, 1, 2, 3, 4, 5, 7, 8])
        B = _log_int(rng, 1, min(64, max(1, 60000000 // (V * (2 * K + 1)))))
        return dict(kind=kind, mode=mode, B=B, K=K, V=V, draft=rng.random() < 0.7,
                    temperature=rng.choice([1.0, 0.7, 1.3, 0.0]), masked=rng.random() < 0.3,
                    ragged=B > 1 and rng.random() < 0.5)
    if kind == "cache_rows":
        B = _log_int(rng, 1, 32)
        T = _log_int(rng, 1, 8192 // B)
        return dict(kind=kind, mode=mode, B=B, T=T, Hk=rng.choice([2, 4, 16, 16]),
                    capacity=T + _log_int(rng, 1, 4096))
    H = rng.choice([4, 16, 16, 16])
    T = rng.choice([1, 1, 1, _log_int(rng, 2, 128)])
    B = _log_int(rng, 1, 64 if T < 8 else 8)
    prefix = rng.choice([0, _log_int(rng, 33, 8192)])
    length = T + _log_int(rng, 1, min(8192, 131072 // B))
    return dict(kind=kind, mode=mode, B=B, T=T, H=H, Hk=rng.choice([H, H, H // 4]), prefix=prefix, length=length,
                ragged=B > 1 and rng.random() < 0.6)


# ---- inputs ---------------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _tdt(case):
    return torch.bfloat16 if case["mode"] == "bf16" else torch.float32


def _randn(g, shape, tdt=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(tdt)


def _starts(case, seed):
    """The positions of the rows' first tokens, on the host; a sequence that begins has 0."""
    if case["positions"] == "none":
        return np.zeros(case["B"], np.int32)
    rng = np.random.default_rng(int(seed) + 5)
    return rng.integers(0, case["far"] - case["T"] + 1, size=case["B"]).astype(np.int32)


def _position_tensor(case, seed):
    """[B, T] positions; given ones jump now and then, as in sequences packed into one row."""
    pos = torch.as_tensor(_starts(case, seed), device=DEV)[:, None] + torch.arange(case["T"], device=DEV, dtype=torch.int32)
    if case["positions"] == "given":
        jump = torch.randint(0, case["T"] + 1, (case["B"], 1), generator=_gen(seed + 11), device=DEV)
        at = torch.arange(case["T"], device=DEV)[None]
        pos = torch.where(at >= jump, (at - jump).to(torch.int32), pos)
    return pos.to(torch.int32).contiguous()


def _heads(case, seed):
    """Projected queries and keys, [B, T, heads, D]: of token-dependent size, as projections are."""
    g = _gen(seed)
    size = torch.exp(0.3 * _randn(g, (case["B"], case["T"], 1, 1)))
    q = (1.5 * size * _randn(g, (case["B"], case["T"], case["H"], D))).to(_tdt(case))
    k = (1.5 * size * _randn(g, (case["B"], case["T"], case["Hk"], D))).to(_tdt(case))
    return q, k


def _head_grads(case, seed):
    g = _gen(seed + 1000003)
    return tuple((0.01 * _randn(g, (case["B"], case["T"], n, D))).to(_tdt(case)) for n in (case["H"], case["Hk"]))


def _norm_weights(seed):
    g = _gen(seed + 2000003)
    return 1.0 + 0.1 * _randn(g, (D,)), 1.0 + 0.1 * _randn(g, (D,))


def _drafting(case, seed):
    """Logits of a model and of a smaller one that follows it, the tokens that the smaller one drafted, the random
    numbers, and how many drafts each row has."""
    g = _gen(seed)
    B, K, V = case["B"], case["K"], case["V"]
    x = 2.5 * _randn(g, (B, K + 1, V))
    peak = torch.randint(0, V, (B, K + 1, 1), generator=g, device=DEV)
    lift = torch.where(torch.rand((B, K + 1, 1), generator=g, device=DEV) < 0.5, 18.0, 9.0)
    x.scatter_add_(2, peak, lift)
    hide = None
    if case["masked"]:  # tokens that an answer's form does not allow, in half of the vocabulary
        hide = torch.rand((B, 1, V), generator=g, device=DEV) < 0.5
        hide.scatter_(2, peak[:, :1], False)
    y = None
    if case["draft"]:
        y = x[:, :K] + 0.7 * _randn(g, (B, K, V))
        if hide is not None:
            y.masked_fill_(hide, float("-inf"))
        u = torch.rand((B, K, V), generator=g, device=DEV).clamp_min(1e-9)
        drafts = (y / max(case["temperature"], 0.05) - torch.log(-torch.log(u))).argmax(-1)
        y = y.to(_tdt(case))
    else:
        other = torch.randint(0, V, (B, K), generator=g, device=DEV)
        drafts = torch.where(torch.rand((B, K), generator=g, device=DEV) < 0.7, peak[:, :K, 0], other)
    if hide is not None:
        x.masked_fill_(hide, float("-inf"))
    uniforms = torch.rand((B, K + 1), generator=g, device=DEV)
    counts = None
    if case["ragged"]:
        counts = np.random.default_rng(int(seed) + 3).integers(0, K + 1, size=B).astype(np.int32)
        counts[-1] = K
    return x.to(_tdt(case)), drafts.to(torch.int32), uniforms, y, counts


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


def _held_before(case, seed):
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


# ---- the plain forms ------------------------------------------------------------------------------------------


def _plain_frequencies(case):
    """Angle of a position's step for each pair, in 64 bits."""
    n = case["dims"]
    theta = case["theta"]
    if case["scaling"] == "theta":
        theta = theta * case["factor"] ** (n / (n - 2))
    f = torch.tensor(theta, dtype=torch.float64) ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "ramp":
        turns = f * case["original"] / (2 * math.pi)
        keep = ((turns - case["low"]) / (case["high"] - case["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / case["factor"])
    return f.to(DEV)


def _plain_rotate(x, pos, freq, case, sign=1.0):
    """x [B, T, heads, D] in 32 bits, rotated."""
    n = case["dims"]
    angle = pos[..., None].double() * freq  # (far positions: 64 bits)
    c = (torch.cos(angle) * case["magnitude"]).float()[:, :, None]
    s = (torch.sin(angle) * (sign * case["magnitude"])).float()[:, :, None]
    if case["layout"] == "half":
        a, b = x[..., : n // 2], x[..., n // 2 : n]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1) if n < D else turned


def _plain_norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_head_norm_bwd(d, x, w, pos, freq, case):
    g = _plain_rotate(d.float(), pos, freq, case, -1.0)
    x = x.float()
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * inv
    gw = g * w
    dx = inv * (gw - n * (gw * n).mean(-1, keepdim=True))
    return dx.to(d.dtype), (g * n).sum((0, 1, 2), dtype=torch.float64).float()


def _plain_verify(logits, drafts, uniforms, draft_logits, temperature, counts):
    """Accepted drafts of each row, its tokens (the accepted, one more, then -1) and their log probabilities."""
    B, K1, V = logits.shape
    K = K1 - 1
    rows = torch.arange(B, device=logits.device)
    n_drafts = torch.full((B,), K, device=logits.device) if counts is None else counts
    z = logits.double()  # (64 bits: a token is one side of a border or the other)
    z = z / temperature if temperature else z
    lp = z - z.amax(-1, keepdim=True)
    lp = lp - torch.log(torch.exp(lp).sum(-1, keepdim=True))
    at = drafts.long()[..., None]
    use = torch.arange(K, device=logits.device)[None] < n_drafts[:, None]
    if temperature == 0:
        best = logits.argmax(-1)
        ok = (best[:, :K] == drafts) & use
        accepted = ok.long().cumprod(-1).sum(-1)
        token = best[rows, accepted]
    else:
        p_x = torch.exp(lp[:, :K].gather(2, at))[..., 0]
        if draft_logits is not None:
            q = draft_logits.double() / temperature
            q = torch.exp(q - q.amax(-1, keepdim=True))
            q = q / q.sum(-1, keepdim=True)
            q_x = q.gather(2, at)[..., 0]
        else:
            q_x = torch.ones_like(p_x)
        ok = (uniforms[:, :K].double() * q_x < p_x) & use
        accepted = ok.long().cumprod(-1).sum(-1)
        w = torch.exp(lp[rows, accepted])
        refused = accepted < n_drafts
        if K:
            i = accepted.clamp_max(K - 1)
            if draft_logits is not None:
                w = torch.where(refused[:, None], (w - q[rows, i]).clamp_min(0), w)
            else:
                x = drafts.long()[rows, i][:, None]
                w = w.scatter(1, x, torch.where(refused[:, None], torch.zeros_like(w[:, :1]), w.gather(1, x)))
        total = w.cumsum(-1)
        bound = uniforms[:, K:].double() * total[:, -1:]
        token = (total <= bound).sum(-1)
    place = torch.arange(K1, device=logits.device)[None]
    tokens = torch.cat([drafts.long(), token[:, None]], 1)
    tokens = torch.where(place < accepted[:, None], tokens, token[:, None])
    score = lp.gather(2, tokens[..., None])[..., 0]
    past = place > accepted[:, None]
    tokens = tokens.masked_fill(past, -1).to(torch.int32)
    return accepted.to(torch.int32), tokens, score.masked_fill(past, 0).float()


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _plain_quant(x):
    """Rows x [..., D] in 4 bits: codes two to a byte [..., D / 2] and scales [..., 4, 1]."""
    g = x.float().unflatten(-1, (4, 32))
    amax = g.abs().amax(-1, keepdim=True)
    mant, expo = torch.frexp(amax)  # amax = mant 2^expo, mant in [0.5, 1): 6 = 0.75 2^3
    e = (expo - 3 + (mant > 0.75).int()).clamp_min(-120)
    scale = torch.ldexp(torch.ones_like(amax), e)
    y = (g / scale).abs()
    code = torch.zeros_like(y, dtype=torch.uint8)
    for i in range(7):  # past the middle of two levels; at it, where the lower one is odd
        mid = 0.5 * (_LEVELS[i] + _LEVELS[i + 1])
        code += ((y > mid) if i % 2 == 0 else (y >= mid)).to(torch.uint8)
    code += (g < 0).to(torch.uint8) * 8
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _plain_value(codes, scale):
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    table = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)
    return (table[code].unflatten(-1, (4, 32)) * scale).flatten(-2)


def _plain_attention(q, kc, vc, lens, prefix):
    """q [B, T, H, D]; kc, vc the held rows of [B, L, Hk, D]; prefix None or those of [1, P, Hk, D]."""
    B, T, H, _ = q.shape
    Hk, L = kc[0].shape[2], kc[0].shape[1]
    G = H // Hk
    # [B, Hk, G T, D]: the queries that share a head's keys
    Q = q.float().reshape(B, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * T, D)
    K = _plain_value(*kc).permute(0, 2, 3, 1).contiguous()
    S = torch.matmul(Q, K) * SCALE
    del K
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


# ---- one call -------------------------------------------------------------------------------------------------


def prepare(case, seed):
    st = dict(case=case)
    if own:
        import dirktensor_amd as dt
    if case["kind"] in ("rotary", "head_norm", "head_norm_bwd"):
        if case["kind"] != "rotary" or not case["backward"]:
            st["q"], st["k"] = _heads(case, seed)
        if case["kind"] == "head_norm_bwd" or case.get("backward"):
            st["dq"], st["dk"] = _head_grads(case, seed)
        if case["kind"] != "rotary":
            st["wq"], st["wk"] = _norm_weights(seed)
        if own:
            st["rot"] = dt.Rotary(dims=case["dims"], layout=case["layout"], theta=case["theta"],
                                  scaling=None if case["scaling"] == "none" else case["scaling"],
                                  factor=case["factor"], original_length=case["original"], low=case["low"],
                                  high=case["high"], magnitude=case["magnitude"])
            st["at"] = dict()
            if case["positions"] == "starts":
                st["at"] = dict(starts=_starts(case, seed))
            elif case["positions"] == "given":
                st["at"] = dict(positions=_position_tensor(case, seed))
        else:
            st["freq"] = _plain_frequencies(case)
            st["pos"] = _position_tensor(case, seed)
    elif case["kind"] == "verify":
        st["x"], st["drafts"], st["u"], st["y"], counts = _drafting(case, seed)
        st["counts"] = counts if own or counts is None else torch.as_tensor(counts, device=DEV).long()
    elif case["kind"] == "cache_rows":
        st["k"], st["v"] = _rows(case, _gen(seed), case["B"], case["T"])
        st["starts"] = _held_before(case, seed)
        if own:
            st["cache"] = dt.KVCache(case["B"], case["capacity"], case["Hk"], format="fp4")
            lo = int(st["starts"].max())
            if lo:  # what the cache holds already
                z = torch.zeros((case["B"], lo, case["Hk"], D), dtype=_tdt(case), device=DEV)
                st["cache"].append(z, z)
        else:
            shape = (case["B"], case["capacity"], case["Hk"])
            st["held"] = [(torch.zeros((*shape, D // 2), dtype=torch.uint8, device=DEV),
                           torch.zeros((*shape, 4, 1), device=DEV)) for _ in range(2)]
            pos = torch.as_tensor(st["starts"], device=DEV).long()[:, None] + torch.arange(case["T"], device=DEV)
            st["at"] = (torch.arange(case["B"], device=DEV)[:, None].expand_as(pos), pos)
    else:
        q, k, v, pk, pv = _attn_inputs(case, seed)
        lens = _lengths(case, seed)
        st["q"] = q
        st["prefix"] = None
        if own:
            st["cache"] = dt.KVCache(case["B"], case["length"], case["Hk"], format="fp4")
            st["cache"].append(k, v, counts=lens)
            if pk is not None:
                st["prefix"] = dt.KVCache(1, case["prefix"], case["Hk"], format="fp4")
                st["prefix"].append(pk, pv)
        else:
            # (a few sequences at a time: the steps' temporaries are large)
            parts = [[_plain_quant(c) for c in x.split(4)] for x in (k, v)]
            st["kc"], st["vc"] = (tuple(torch.cat(t) for t in zip(*p)) for p in parts)
            if pk is not None:
                st["prefix"] = (_plain_quant(pk), _plain_quant(pv))
            st["lens"] = torch.as_tensor(lens, device=DEV).long()
    return st


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "rotary":
        xs, sign = ((st["dq"], st["dk"]), -1.0) if case["backward"] else ((st["q"], st["k"]), 1.0)
        return [_plain_rotate(x.float(), st["pos"], st["freq"], case, sign).to(x.dtype) for x in xs]
    if kind == "head_norm":
        return [_plain_rotate(_plain_norm(x.float(), w), st["pos"], st["freq"], case).to(x.dtype)
                for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"]))]
    if kind == "head_norm_bwd":
        dq, dwq = _plain_head_norm_bwd(st["dq"], st["q"], st["wq"], st["pos"], st["freq"], case)
        dk, dwk = _plain_head_norm_bwd(st["dk"], st["k"], st["wk"], st["pos"], st["freq"], case)
        return dq, dk, dwq, dwk
    if kind == "verify":
        return _plain_verify(st["x"], st["drafts"], st["u"], st["y"], case["temperature"], st["counts"])
    if kind == "cache_rows":
        out = []
        for x, (hc, hs) in zip((st["k"], st["v"]), st["held"]):
            hc[st["at"]], hs[st["at"]] = _plain_quant(x)
            out.append(_plain_value(hc[st["at"]], hs[st["at"]]).to(x.dtype))
        return out
    return _plain_attention(st["q"], st["kc"], st["vc"], st["lens"], st["prefix"])


def _run_own(st):
    import dirktensor_amd as dt

    case = st["case"]
    kind = case["kind"]
    if kind == "rotary":
        if case["backward"]:
            return dt.rotary_backward(st["dq"], st["dk"], st["rot"], **st["at"])
        return dt.rotary(st["q"], st["k"], st["rot"], **st["at"])
    if kind == "head_norm":
        return dt.head_norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["rot"], eps=EPS, **st["at"])
    if kind == "head_norm_bwd":
        r = dt.head_norm_rotary_backward(st["dq"], st["dk"], st["q"], st["k"], st["wq"], st["wk"], st["rot"], eps=EPS,
                                         **st["at"])
        return r.d_Q, r.d_K, r.d_q_weight, r.d_k_weight
    if kind == "verify":
        r = dt.verify_drafts(st["x"], st["drafts"], st["u"], draft_logits=st["y"], temperature=case["temperature"],
                             counts=st["counts"])
        return r.accepted, r.tokens, r.logprob
    if kind == "cache_rows":
        st["cache"].truncate(st["starts"])
        st["cache"].append(st["k"], st["v"])
        return list(st["cache"].read(st["starts"], case["T"], mode=case["mode"]))
    r = dt.cached_attention(st["q"], st["cache"], SCALE, prefix=st["prefix"])
    return r.output, r.softmax_m, r.softmax_l


# ---- what a call cannot do without ----------------------------------------------------------------------------


def work(case):
    es = 2 if case["mode"] == "bf16" else 4
    kind = case["kind"]
    held = lambda n: n * (D // 2 + 4)
    if kind in ("rotary", "head_norm", "head_norm_bwd"):
        n = case["B"] * case["T"] * (case["H"] + case["Hk"]) * D
        if kind == "rotary":  # (values past the rotated ones move too: results are tensors of their own)
            return dict(bytes=2 * n * es, flops=3 * n)
        if kind == "head_norm":
            return dict(bytes=2 * n * es + 8 * D, flops=7 * n)
        return dict(bytes=3 * n * es + 16 * D, flops=14 * n)
    if kind == "verify":
        B, K, V = case["B"], case["K"], case["V"]
        drafts = B * K if not case["ragged"] else int(_ragged_counts(case, 0).sum())
        read = (drafts + B) + (drafts if case["draft"] and case["temperature"] else 0)
        return dict(bytes=read * V * es + 4 * B * (K + (K + 1) + 1 + 2 * (K + 1)), flops=4 * read * V)
    if kind == "cache_rows":
        n = case["B"] * case["T"] * case["Hk"]
        return dict(bytes=2 * (2 * n * D * es + 2 * held(n)), flops=2 * n * D * 4)
    lens = _lengths(case, 0)  # (of one seed; the others' are alike)
    keys = int(lens.sum())
    rows = case["B"] * case["T"] * case["H"]
    pairs = keys * case["T"] * case["H"] + rows * case["prefix"]
    return dict(bytes=2 * held((keys + case["prefix"]) * case["Hk"]) + 2 * rows * D * es + 8 * rows,
                flops=4 * pairs * D)


def _ragged_counts(case, seed):
    counts = np.random.default_rng(int(seed) + 3).integers(0, case["K"] + 1, size=case["B"])
    counts[-1] = case["K"]
    return counts


# ---- 64 bits --------------------------------------------------------------------------------------------------


def _turn64(x, pos, case, back=False):
    """Rotation as a product with e^(i angle), in 64 bits."""
    n, theta = case["dims"], case["theta"]
    i = torch.arange(n // 2, dtype=torch.float64, device=DEV)
    if case["scaling"] == "theta":
        theta *= case["factor"] ** (n / (n - 2))
    f = torch.exp(-(2 * i / n) * math.log(theta))
    if case["scaling"] == "linear":
        f /= case["factor"]
    if case["scaling"] == "ramp":
        whole = case["original"] * f / (2 * math.pi)
        share = torch.clip((whole - case["low"]) / (case["high"] - case["low"]), 0.0, 1.0)
        f = share * f + (1 - share) * f / case["factor"]
    angle = pos.double()[:, :, None] * f
    unit = torch.polar(torch.full_like(angle, case["magnitude"]), -angle if back else angle)[:, :, None]
    first, second = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _held64(x):
    """The values that the cache stands for, from their definition."""
    x = x.double().unflatten(-1, (4, 32))
    top = x.abs().max(dim=-1, keepdim=True).values
    step = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -119) / 6)).clamp_min(-120))
    step = torch.where(top > 6 * step, 2 * step, step)
    step = torch.where(top <= 6 * (step / 2), step / 2, step).clamp_min(2.0 ** -120)
    y = x / step
    ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1.0))) - 1)  # (one bit behind the leading one, 0.5 at least)
    return ((y / ulp).round() * ulp * step).flatten(-2)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("rotary", "head_norm", "head_norm_bwd"):
        pos = _position_tensor(case, seed)
        if kind == "rotary":
            xs = _head_grads(case, seed) if case["backward"] else _heads(case, seed)
            return [_turn64(x.double(), pos, case, case["backward"]) for x in xs]
        out, weight_grads = [], []
        for i in range(2):
            x, w = _heads(case, seed)[i].double(), _norm_weights(seed)[i].double()
            size = torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
            if kind == "head_norm":
                out.append(_turn64(x / size * w, pos, case))
                continue
            g = _turn64(_head_grads(case, seed)[i].double(), pos, case, True)
            # d(x / size): the part of g w along x is taken out
            along = (g * w * x).mean(-1, keepdim=True) / size ** 2
            out.append((g * w - x * along) / size)
            weight_grads.append((g * x / size).reshape(-1, D).sum(0))
        return (*out, *weight_grads) if weight_grads else out
    if kind == "verify":
        return _exact_verify(case, seed)
    if kind == "cache_rows":
        return [_held64(x) for x in _rows(case, _gen(seed), case["B"], case["T"])]
    return _exact_attn(case, seed)


def _exact_verify(case, seed):
    x, drafts, uniforms, y, counts = _drafting(case, seed)
    B, K, T = case["B"], case["K"], case["temperature"]
    accepted = torch.zeros(B, dtype=torch.int32)
    tokens = torch.full((B, K + 1), -1, dtype=torch.int32)
    score = torch.zeros((B, K + 1), dtype=torch.float64)
    for b in range(B):
        n = K if counts is None else int(counts[b])
        u = uniforms[b].double().cpu()
        z = x[b].double()
        lp = torch.log_softmax(z / T if T else z, -1)
        for i in range(n + 1):
            left = None  # what the next token is drawn from, where this draft is not taken
            if T == 0:
                token = int((z[i] == z[i].max()).nonzero()[0])
                if i < n and token == int(drafts[b, i]):
                    left = None
                else:
                    left = token
            else:
                p = lp[i].exp()
                q = None
                if i < n:
                    d = int(drafts[b, i])
                    if y is not None:
                        q = torch.softmax(y[b, i].double() / T, -1)
                    else:
                        q = torch.zeros_like(p)
                        q[d] = 1.0
                if q is None or not float(u[i]) * float(q[d]) < float(p[d]):
                    w = p if q is None else (p - q).clamp_min(0) if y is not None else p * (1 - q)
                    c = w.cumsum(0)
                    left = int(torch.searchsorted(c, u[K].to(DEV) * c[-1], right=True))
            t = left if left is not None else int(drafts[b, i])
            tokens[b, i] = t
            score[b, i] = lp[i, t].cpu()
            if left is not None:
                break
            accepted[b] += 1
    return accepted.to(DEV), tokens.to(DEV), score.to(DEV)


def _exact_attn(case, seed):
    q, k, v, pk, pv = _attn_inputs(case, seed)
    lens = _lengths(case, seed)
    B, T, H, G = case["B"], case["T"], case["H"], case["H"] // case["Hk"]
    O = torch.empty((B, T, H, D), dtype=torch.float64, device=DEV)
    m = torch.empty((B, T, H), dtype=torch.float64, device=DEV)
    l = torch.empty_like(m)
    if pk is not None:
        pk, pv = _held64(pk)[0], _held64(pv)[0]
    for b in range(B):
        n = int(lens[b])
        kb, vb = _held64(k[b, :n]), _held64(v[b, :n])
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
