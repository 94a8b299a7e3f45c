"""A generation with drafts whose cache is looked at after every step: it holds what was verified and no more, and a query over it gets
what the definition in 64 bits gives on the rows it reads back (with the bounds of test_cached_attn_gpu)."""

import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn
from test_draft_run_gpu import D, H, HK, SCALE, V, Layer, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1.0, 0.0])
@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
def test_the_cache_of_a_generation_with_drafts(gpu, temperature, tdt):
    import dirktensor_amd as dt

    layer = Layer()
    B, K, steps, P = 3, 4, 9, 45
    g = torch.Generator(device="cuda").manual_seed(11)
    prefix, cache = dt.KVCache(1, P, HK, format="fp4"), dt.KVCache(B, 100, HK, format="fp4")
    layer.logits(torch.randint(0, V, (1, P), generator=g, device="cuda"), prefix, None, 0)
    answers = [[int(t)] for t in torch.randint(0, V, (B,), generator=g, device="cuda")]
    for step in range(steps):
        held = cache.lengths[:B].copy()
        newest = torch.tensor([[a[-1]] for a in answers], device="cuda")
        guess = torch.cat([newest, torch.randint(0, V, (B, K), generator=g, device="cuda")], 1)
        drafts = layer.logits(guess, cache, prefix, P)[:, :K].argmax(-1)
        cache.truncate(held)
        x = layer.logits(torch.cat([newest, drafts], 1), cache, prefix, P)
        u = torch.rand((B, K + 1), generator=g, device="cuda")
        r = dt.verify_drafts(x, drafts, u, draft_logits=x[:, :K].flip(0), temperature=temperature)
        n = r.accepted.cpu().numpy()
        for b in range(B):
            answers[b] += r.tokens[b, :n[b] + 1].tolist()
        before = [t.clone() for t in cache.read([0] * B, int(held.min()) + 1, mode="fp32")]
        cache.truncate(held + 1 + n)
        assert cache.lengths[:B].tolist() == [len(a) - 1 for a in answers]
        for a, c in zip(before, cache.read([0] * B, int(held.min()) + 1, mode="fp32")):
            assert torch.equal(a, c)
        q = randn((B, 2, H, D), 100 + step).to(tdt)
        attn.run(q, cache, prefix=prefix)
        attn.run(q, cache, causal=False)
    for b in range(B):
        # one run over the accepted tokens holds the same, but for codes of values next to a border (the matrix product adds in another
        # order for rows of another number); with the same codes the same comes out, bit for bit
        fresh = dt.KVCache(1, 100, HK, format="fp4")
        layer.logits(torch.tensor([answers[b][:-1]], device="cuda"), fresh, prefix, P)
        n = len(answers[b]) - 1
        rows = [c.read([0], n, slots=[s], mode="fp32") for c, s in ((cache, b), (fresh, 0))]
        off = [int((x != y).sum()) for x, y in zip(*rows)]
        assert max(off) <= 3, off
        q = randn((1, 1, H, D), 50 + b).to(tdt)
        one = attn.run(q, cache, slots=[b], prefix=prefix)
        other = attn.run(q, fresh, prefix=prefix)
        if off == [0, 0]:
            assert torch.equal(one.output, other.output) and torch.equal(one.softmax_l, other.softmax_l)
        assert torch.equal(one.output, dt.cached_attention(q, cache, SCALE, slots=[b], prefix=prefix).output)
