"""The tests of cached attention and of the scores' gradient once more, with checks that a NaN cannot pass. (A comparison `error > bound`
is false for NaN: an output that was never written, or a product of 0 and infinity, would pass a test that asks for no such place.)"""

import inspect
import itertools

import pytest

torch = pytest.importorskip("torch")

import test_cached_attn_gpu as attn
import test_sampling_run_gpu as sampling
import test_token_logprobs_gpu as scores

_attn_check, _check_grad = attn.check, scores.check_grad


def check(r, ref, tdt):
    assert not any(bool(torch.isnan(x).any()) for x in (r.output, r.softmax_m, r.softmax_l, *ref))
    _attn_check(r, ref, tdt)


def check_grad(got, *args, **kw):
    assert not bool(torch.isnan(got).any())
    _check_grad(got, *args, **kw)


def _cases(*tests):
    for f in tests:
        marks = [m for m in getattr(f, "pytestmark", []) if m.name == "parametrize"]
        names = [m.args[0].replace(" ", "").split(",") for m in marks]
        for values in itertools.product(*(m.args[1] for m in marks)):
            kw = {}
            for n, v in zip(names, values):
                kw.update(zip(n, v) if len(n) > 1 else [(n[0], v)])
            assert set(kw) == set(inspect.signature(f).parameters)
            yield pytest.param(f, kw, id="-".join([f.__name__, *(str(v).replace("torch.", "") for v in kw.values())]))


@pytest.mark.gpu
@pytest.mark.parametrize("test,kw", _cases(
    attn.test_one_token, attn.test_several_tokens_and_shared_heads, attn.test_shared_prefix, attn.test_prefix_in_the_same_cache_and_slots_twice,
    attn.test_a_prefix_and_nothing_of_their_own, attn.test_large_scores, attn.test_small_and_large_queries_in_fp32,
    attn.test_a_generation_of_several_answers, attn.test_more_sequences_and_heads_than_workgroups, attn.test_more_rows_than_a_call_takes,
    scores.test_row_lengths_and_alignments, scores.test_few_and_many_rows, scores.test_masked_and_degenerate_rows,
    scores.test_ignored_and_foreign_tokens, sampling.test_answers_to_one_prompt, sampling.test_workspaces_grow_with_the_call))
def test_again(test, kw, monkeypatch):
    monkeypatch.setattr(attn, "check", check)
    monkeypatch.setattr(scores, "check_grad", check_grad)
    test(**kw)


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["nowhere", "everywhere", "one_place"])
def test_the_attention_check_refuses_nan(tdt, where):
    from dirktensor_amd import FlashAttentionResult

    shape = (2, 3, 4)
    m, l = torch.zeros(shape, dtype=torch.float64), torch.full(shape, 2.0, dtype=torch.float64)
    o = torch.ones((*shape, 128), dtype=torch.float64)
    out = o.to(tdt)
    if where == "everywhere":
        out.fill_(float("nan"))
    elif where == "one_place":
        out[1, 2, 3, 77] = float("nan")
    r, ref = FlashAttentionResult(out, m.float(), l.float()), (o, m, l, o.abs(), torch.ones_like(m))
    if where == "nowhere":
        check(r, ref, tdt)
    else:
        with pytest.raises(AssertionError):
            check(r, ref, tdt)
    r.output = o.to(tdt)
    r.output[0, 0, 0, 0] = 1.1  # (and what the bounds refuse)
    with pytest.raises(AssertionError):
        check(r, ref, tdt)


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["nowhere", "everywhere", "one_place"])
def test_the_gradient_check_refuses_nan(tdt, where):
    x = torch.linspace(-2, 2, 2 * 50).view(2, 50).to(tdt)
    tok, g, h = torch.tensor([3, 7], dtype=torch.int32), torch.tensor([1.0, -0.5]), torch.tensor([0.25, 0.5])
    z = x.double().requires_grad_()
    lp = torch.log_softmax(z, -1)
    ((g.double() * lp.gather(1, tok.long()[:, None])[:, 0]).sum() - (h.double()[:, None] * lp.exp() * lp).sum()).backward()
    got = z.grad.to(tdt)
    if where == "nowhere":
        check_grad(got, x, tok, g, h)
        got[1, 7] *= 1.1
    elif where == "everywhere":
        got.fill_(float("nan"))
    else:
        got[0, 49] = float("nan")
    with pytest.raises(AssertionError):
        check_grad(got, x, tok, g, h)
