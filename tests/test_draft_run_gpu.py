"""The operators of a generation step used together: queries and keys normed and rotated where the cache continues, appended in 4 bits,
attended to behind a shared prompt, drafts verified, the cache cut to what was accepted; and the norm and rotation around the
attention of a training step, forwards and backwards."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_rotary_gpu import norm64, turn64
from test_verify_drafts_gpu import check as check_verified
from test_verify_drafts_gpu import reference as verified64

pytestmark = pytest.mark.gpu

D, H, HK, DM, V = 128, 4, 2, 64, 501
SCALE = 1 / np.sqrt(D)


def randn(shape, seed, scale=1.0):
    return scale * torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


class Layer:
    """One attention layer between an embedding and a head, of random weights."""

    def __init__(self):
        import dirktensor_amd as dt

        self.dt = dt
        self.embed = randn((V, DM), 1)
        self.wqkv = randn((DM, (H + 2 * HK) * D), 2, DM ** -0.5)
        self.wo = randn((H * D, V), 3, 2.5 * (H * D) ** -0.5)
        self.nq, self.nk = 1 + 0.1 * randn((D,), 4), 1 + 0.1 * randn((D,), 5)
        self.rot = dt.Rotary(dims=96, scaling="ramp", factor=4.0, original_length=512)

    def logits(self, tokens, cache, prefix, before):
        """tokens [B, T] behind what the cache holds, `before` tokens of a shared prompt before that"""
        qkv = self.embed[tokens] @ self.wqkv
        q = qkv[..., :H * D].unflatten(-1, (H, D))
        k = qkv[..., H * D:(H + HK) * D].unflatten(-1, (HK, D))
        v = qkv[..., (H + HK) * D:].unflatten(-1, (HK, D))
        B = tokens.shape[0]
        self.dt.head_norm_rotary(q, k, self.nq, self.nk, self.rot, starts=cache.lengths[:B] + before, inplace=True)
        cache.append(k, v)
        r = self.dt.cached_attention(q, cache, SCALE, prefix=prefix)
        return r.output.flatten(2) @ self.wo


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_generation_with_drafts(gpu, temperature):
    import dirktensor_amd as dt

    layer = Layer()
    B, K, steps, P = 3, 4, 8, 45
    g = torch.Generator(device="cuda").manual_seed(7)
    prompt = torch.randint(0, V, (1, P), generator=g, device="cuda")
    prefix = dt.KVCache(1, P, HK, format="fp4")
    layer.logits(prompt, prefix, None, 0)
    cache = dt.KVCache(B, 200, HK, format="fp4")
    answers = [[int(t)] for t in torch.randint(0, V, (B,), generator=g, device="cuda")]
    accepted = 0
    for step in range(steps):
        # the newest token of each answer and K drafts behind it: what the model itself finds likely behind random ones, one of them off
        newest = torch.tensor([[a[-1]] for a in answers], device="cuda")
        held = cache.lengths[:B].copy()
        assert held.tolist() == [len(a) - 1 for a in answers]
        drafts = layer.logits(torch.cat([newest, torch.randint(0, V, (B, K), generator=g, device="cuda")], 1), cache, prefix, P)[:, :K].argmax(-1)
        cache.truncate(held)
        drafts[0, step % K] = (drafts[0, step % K] + 1) % V
        x = layer.logits(torch.cat([newest, drafts], 1), cache, prefix, P)
        u = torch.rand((B, K + 1), generator=g, device="cuda")
        y = x[:, :K] + 0.3 * torch.randn((B, K, V), generator=g, device="cuda")
        r = dt.verify_drafts(x, drafts, u, draft_logits=y, temperature=temperature)
        check_verified(r, verified64(x, drafts, u, y, temperature))
        n = r.accepted.cpu().numpy()
        accepted += int(n.sum())
        for b in range(B):
            answers[b] += r.tokens[b, :n[b] + 1].tolist()
        cache.truncate(held + 1 + n)  # what was verified: the newest token and the accepted drafts
    assert accepted > 0
    # the cache holds what one run over the accepted tokens holds, and answers the same
    for b in range(B):
        fresh = dt.KVCache(1, 200, HK, format="fp4")
        tokens = torch.tensor([answers[b][:-1]], device="cuda")
        x = layer.logits(tokens, fresh, prefix, P)
        n = len(answers[b]) - 1
        assert cache.lengths[b] == n
        # (rows of one length and another go through the matrix product in another order: codes may differ by a step where a value lies
        # next to a border, 2^-20 of them near enough)
        for a, c in zip(cache.read([0], n, slots=[b], mode="fp32"), fresh.read([0], n, mode="fp32")):
            assert int((a != c).sum()) <= 3, int((a != c).sum())
        q = randn((1, 1, H, D), 50 + b)
        a, c = dt.cached_attention(q, cache, SCALE, slots=[b], prefix=prefix), dt.cached_attention(q, fresh, SCALE, prefix=prefix)
        # one code of one key in n is half its size off at most: 1 / n of the weights times that
        assert float((a.output - c.output).abs().max()) <= 3 * 6.0 / n


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
def test_a_training_step_through_the_attention(gpu, tdt):
    """Norm and rotation, attention, its backward, the norm's and rotation's backward, against the chain in 64 bits by automatic
    differentiation on the CPU. The bound is that of the attention's parity, over the chain: 1e-4 and 2e-2 of the largest value,
    for each of the three operators that round to the type."""
    import dirktensor_amd as dt

    B, T, Hn = 2, 70, 2
    rot = dt.Rotary(dims=64, layout="interleaved")
    q, k, v, d = (randn((B, T, Hn, D), 10 + i).to(tdt) for i in range(4))
    w, u = 1 + 0.1 * randn((D,), 20), 1 + 0.1 * randn((D,), 21)
    qr, kr = dt.head_norm_rotary(q, k, w, u, rot)
    r = dt.flash_attention_forward(qr, kr, v, SCALE)
    gr = dt.flash_attention_backward(d, r.output, r.softmax_m, r.softmax_l, qr, kr, v, SCALE)
    h = dt.head_norm_rotary_backward(gr.d_Q, gr.d_K, q, k, w, u, rot)

    leaves = [t.detach().cpu().double().requires_grad_() for t in (q, k, v, w, u)]
    pos = torch.arange(T)[None].expand(B, T)

    def turned(x):  # (turn64 writes in place: the same by a mask of pairs)
        f = torch.from_numpy(rot.frequencies)
        c, s = (fn(pos[..., None].double() * f)[:, :, None] for fn in (torch.cos, torch.sin))
        a, b = x[..., 0:64:2], x[..., 1:64:2]
        return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., 64:]], -1)

    x = turned(norm64(leaves[0], leaves[3]))
    y = turned(norm64(leaves[1], leaves[4]))
    assert torch.allclose(x.detach(), turn64(norm64(leaves[0], leaves[3]).detach(), pos, rot), atol=1e-12)
    s = torch.einsum("bthd,bshd->bhts", x, y) * SCALE
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), float("-inf"))
    o = torch.einsum("bhts,bshd->bthd", torch.softmax(s, -1), leaves[2])
    o.backward(d.cpu().double())
    tol = 3 * (1e-4 if tdt == torch.float32 else 2e-2)
    for got, leaf in zip((h.d_Q, h.d_K, gr.d_V, h.d_q_weight, h.d_k_weight), leaves):
        ref = leaf.grad
        assert float((got.cpu().double() - ref).abs().max()) <= tol * float(ref.abs().max())


def test_threads_streams_and_graphs_beside_each_other(gpu):
    """A captured step replayed while other streams run the same operators with workspaces of their own."""
    import dirktensor_amd as dt

    x, y = randn((4, 4, 5003), 1, 3.0), randn((4, 3, 5003), 2, 3.0)
    d = y.argmax(-1).int()
    u = torch.rand((4, 4), device="cuda")
    q, dq = randn((1, 300, 4, D), 3), randn((1, 300, 4, D), 4)
    w, rot = torch.ones(D, device="cuda"), dt.Rotary()

    def both():
        r = dt.verify_drafts(x, d, u, draft_logits=y)
        h = dt.head_norm_rotary_backward(dq, None, q, None, w, None, rot)
        return r.tokens, r.logprob, h.d_Q, h.d_q_weight

    want = [t.clone() for t in both()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        g.replay()
        for s in streams:
            with torch.cuda.stream(s):
                got.append(both())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
