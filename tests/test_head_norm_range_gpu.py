"""Each head's norm at the ends of fp32's range and beside infinities, forwards and backwards, against the formulas in 64 bits (with the
bounds of test_rotary_gpu)."""

import pytest

torch = pytest.importorskip("torch")

from test_rotary_gpu import EPS, check, default_positions, grads64, norm64, randn, turn64

pytestmark = pytest.mark.gpu

D, DIMS = 128, 64
TYPES = [torch.float32, torch.bfloat16]


def dt():
    import dirktensor_amd

    return dirktensor_amd


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
@pytest.mark.parametrize("at", [3, 40, 100])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_an_infinity_leaves_zeros_beside_it(gpu, tdt, value, at, layout):
    """x / sqrt(mean x^2 + eps) of a head with an infinity: 0 for its finite values, NaN for the infinity, and for the value that turns
    with it."""
    rot = dt().Rotary(dims=DIMS, layout=layout)
    q, k = randn((2, 3, 9, D), 1, tdt), randn((2, 3, 2, D), 2, tdt)
    w, u = 1 + 0.1 * randn((D,), 3), 1 + 0.1 * randn((D,), 4)
    want = dt().head_norm_rotary(q, k, w, u, rot)
    x, y = q.clone(), k.clone()
    x[1, 2, 8, at], y[0, 1, 1, at] = value, value
    got = dt().head_norm_rotary(x, y, w, u, rot)
    hit = torch.zeros(D, dtype=torch.bool, device="cuda")
    hit[at] = True
    if at < DIMS:
        hit[(at + DIMS // 2) % DIMS if layout == "half" else at ^ 1] = True
    for g, e, head in zip(got, want, ((1, 2, 8), (0, 1, 1))):
        assert bool(torch.isnan(g[head][hit]).all()) and bool((g[head][~hit] == 0).all())
        e = e.clone()
        e[head] = g[head]
        assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(e))  # (the other heads are as they were)


@pytest.mark.parametrize("tdt", TYPES)
def test_gradients_beside_an_infinity(gpu, tdt):
    """Its head's gradients are NaN (the mean of w g n is), and of the weights' the one of its column; the other columns are sums
    without that head, whose n is 0 there."""
    rot = dt().Rotary(dims=DIMS)
    q, d = randn((1, 5, 9, D), 1, tdt), randn((1, 5, 9, D), 2, tdt)
    w = 1 + 0.1 * randn((D,), 3)
    x, without = q.clone(), d.clone()
    x[0, 3, 4, 77] = float("inf")
    without[0, 3, 4] = 0  # (no gradient: its terms are 0 too)
    r, e = (dt().head_norm_rotary_backward(g, None, v, None, w, None, rot) for g, v in ((d, x), (without, q)))
    assert bool(torch.isnan(r.d_Q[0, 3, 4]).all()) and int(torch.isnan(r.d_Q).sum()) == D
    assert torch.isnan(r.d_q_weight[77]) and int(torch.isnan(r.d_q_weight).sum()) == 1
    keep = torch.arange(D, device="cuda") != 77
    assert torch.equal(r.d_q_weight[keep], e.d_q_weight[keep])


def test_a_nan_beside_an_infinity(gpu):
    rot = dt().Rotary(dims=DIMS)
    q = randn((1, 2, 2, D), 1)
    q[0, 0, 0, 5], q[0, 0, 0, 90] = float("inf"), float("nan")
    y = dt().head_norm_rotary(q, None, torch.ones(D, device="cuda"), None, rot)[0]
    assert bool(torch.isnan(y[0, 0, 0]).all()) and int(torch.isnan(y).sum()) == D


@pytest.mark.parametrize("size", [1e18, 1.4e19, 1e30, 8e37, 3e38])
def test_large_rows(gpu, size):
    """To the end of the range. From a root mean square of 2^126 on the factor, 2^-128 at least, is no normal number, and its rounding is up
    to 2^-150 / 2^-128 = 4 h; the gradient has it in front and in n, twice beside the mean: (61 + 12) / 61 of what is there without."""
    rot = dt().Rotary(dims=DIMS)
    q = randn((1, 4, 3, D), 1).clamp(-1, 1) * size
    q[0, 1] = size * torch.sign(q[0, 1])
    w = 1 + 0.1 * randn((D,), 2)
    pos = default_positions(1, 4)
    ref = norm64(q.double(), w.double())
    y = dt().head_norm_rotary(q, None, w, None, rot, eps=EPS)[0]
    check(y, turn64(ref, pos, rot), turn64(ref, pos, rot, size=True), 21 + 4, torch.float32)
    if size > 1e19:  # (smaller: sums of 32 bits, as elsewhere)
        d = randn((1, 4, 3, D), 3) * 1e20
        r = dt().head_norm_rotary_backward(d, None, q, None, w, None, rot, eps=EPS)
        dx, dw, dx_size, dw_size = grads64(d, q, w, pos, rot)
        err = (r.d_Q.double() - dx).abs()
        assert bool((err <= 1.2 * 2.0 ** -24 * dx_size + 2.0 ** -149).all())
        check(r.d_q_weight, dw, dw_size, 21 + 4 + 2 + 55, torch.float32)
