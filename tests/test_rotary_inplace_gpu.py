"""Rotations in place beside torch's automatic gradients: a tensor that a graph saved is known to have changed, and one that requires a
gradient is not overwritten where gradients are recorded."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 128


def calls():
    import dirktensor_amd as dt

    rot = dt.Rotary(dims=64)
    w = torch.ones(D, device="cuda")
    return [lambda q, k: dt.rotary(q, k, rot, inplace=True), lambda q, k: dt.rotary_backward(q, k, rot, inplace=True),
            lambda q, k: dt.head_norm_rotary(q, k, w, w, rot, inplace=True)]


def rows(*heads):
    return [torch.randn((2, 3, n, D), device="cuda") for n in heads]


@pytest.mark.parametrize("i", range(3))
@pytest.mark.parametrize("which", ["q", "k", "view"])
def test_a_graph_that_saved_the_tensor_raises(gpu, i, which):
    call = calls()[i]
    qkv = torch.randn((2, 3, 6 * D), device="cuda")
    q, k = (qkv[..., a * D:b * D].unflatten(-1, (b - a, D)) for a, b in ((0, 4), (4, 6)))
    saved = {"q": q, "k": k, "view": qkv}[which]
    w = torch.ones((), device="cuda", requires_grad=True)
    loss = (w * saved).sum()  # (saves what w is multiplied by)
    before = saved.clone()
    call(q, k)
    assert not torch.equal(saved, before)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()


@pytest.mark.parametrize("i", range(3))
def test_without_k_and_out_of_place(gpu, i):
    import dirktensor_amd as dt

    q, k = rows(4, 2)
    at = q._version
    calls()[i](q, None)
    assert q._version > at
    at = q._version, k._version
    dt.rotary(q, k, dt.Rotary())
    assert (q._version, k._version) == at
    with torch.inference_mode():
        calls()[i](*rows(4, 2))


@pytest.mark.parametrize("i", range(3))
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("leaf", [True, False])
def test_tensors_that_require_a_gradient(gpu, i, which, leaf):
    x = rows(4, 2)
    x[which].requires_grad_()
    if not leaf:
        x[which] = x[which] * 2
    before = [t.detach().clone() for t in x]
    with pytest.raises(ValueError, match="requires a gradient"):
        calls()[i](*x)
    assert all(torch.equal(t.detach(), b) for t, b in zip(x, before))
    with torch.no_grad():
        y = calls()[i](*x)
    assert y[0] is x[0] and y[1] is x[1] and not torch.equal(x[0].detach(), before[0])
