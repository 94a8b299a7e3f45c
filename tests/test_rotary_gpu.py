"""Rotations of queries and keys, with and without each head's norm, and their gradients, against the formulas in 64 bits.

Tolerances, in units h = 2^-24 (half a step of fp32, relative): a cosine or sine is off by at most 2 h from the function, 1 h
from the rounding of its argument and 1 h from the magnitude; a product and a sum add 1 h each. So a rotated value is off by
6 h mag (|a| + |b|) of its pair. The norm's factor: a sum of 128 squares in chains of 16 and 3 (20 h), the mean and eps 2 h, of which
the root takes half, root and quotient 2 h: 13 h, and 2 h for the products with it and the weight. bf16 adds half a step, 2^-8."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 128
H24 = 2.0 ** -24
EPS = 1e-6
TYPES = [torch.float32, torch.bfloat16]


def dt():
    import dirktensor_amd

    return dirktensor_amd


def randn(shape, seed, tdt=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(tdt)


def pairs(rot):
    n = rot.dims
    i = torch.arange(n // 2)
    return (i, i + n // 2) if rot.layout == "half" else (2 * i, 2 * i + 1)


def turn64(x, pos, rot, sign=1.0, size=False):
    """x [B, T, heads, 128] in 64 bits, rotated; or the sizes mag (|a| + |b|) that bound its error."""
    a, b = pairs(rot)
    out = x.abs() if size else x.clone()
    if size:
        out[..., a] = out[..., b] = rot.magnitude * (x[..., a].abs() + x[..., b].abs())
        return out
    f = rot.frequencies.astype(np.longdouble)
    t = pos.cpu().numpy().astype(np.longdouble)[..., None] * f
    c = torch.from_numpy(np.cos(t).astype(np.float64)).to(x.device)[:, :, None] * rot.magnitude
    s = torch.from_numpy(np.sin(t).astype(np.float64)).to(x.device)[:, :, None] * (sign * rot.magnitude)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def check(got, ref, size, units, tdt):
    tol = units * H24 * size + (2.0 ** -8 * ref.abs() if tdt == torch.bfloat16 else 0) + 1e-37
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), got.shape)


def default_positions(B, T, starts=None):
    pos = torch.arange(T, device="cuda")[None].expand(B, T)
    return pos if starts is None else pos + torch.as_tensor(np.asarray(starts), device="cuda")[:, None]


LAYOUTS = ["half", "interleaved"]


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dims", [16, 32, 48, 64, 96, 112, 128])
@pytest.mark.parametrize("B,T,H,Hk", [(1, 1, 1, 1), (2, 7, 5, 3), (3, 50, 16, 16)])
def test_rotation_and_gradient(gpu, tdt, layout, dims, B, T, H, Hk):
    rot = dt().Rotary(dims=dims, layout=layout, magnitude=1.25)
    q, k = randn((B, T, H, D), 1, tdt), randn((B, T, Hk, D), 2, tdt)
    pos = default_positions(B, T)
    for f, sign in ((dt().rotary, 1.0), (dt().rotary_backward, -1.0)):
        out = f(q, k, rot)
        for x, y in zip((q, k), out):
            assert y.dtype == x.dtype and y.shape == x.shape
            check(y, turn64(x.double(), pos, rot, sign), turn64(x.double(), pos, rot, size=True), 6, tdt)
            assert torch.equal(y[..., dims:], x[..., dims:])


@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 4.0), ("theta", 8.0), ("ramp", 16.0)])
@pytest.mark.parametrize("kind", ["starts", "int32", "int64"])
def test_scaled_frequencies_at_far_positions(gpu, scaling, factor, kind):
    B, T, H = 5, 9, 2
    rot = dt().Rotary(dims=128, scaling=scaling, factor=factor, original_length=4096, low=1.0, high=32.0)
    i = np.arange(64)
    f = 500000.0 ** (-2.0 * i / 128)
    if scaling == "linear":
        f = f / factor
    if scaling == "theta":
        f = (500000.0 * factor ** (128 / 126)) ** (-2.0 * i / 128)
        assert np.isclose(f[-1] * factor, 500000.0 ** (-126 / 128), rtol=1e-12) and f[0] == 1.0
    if scaling == "ramp":
        turns = f * 4096 / (2 * np.pi)
        keep = np.clip((turns - 1) / 31, 0, 1)
        f = f * (keep + (1 - keep) / factor)
    np.testing.assert_allclose(rot.frequencies, f, rtol=1e-12)
    q = randn((B, T, H, D), 3)
    starts = np.array([0, 8191, 1 << 20, -77, 12345678])
    pos = default_positions(B, T, starts)
    at = dict(starts=starts) if kind == "starts" else dict(positions=pos.to(torch.int32 if kind == "int32" else torch.int64))
    out, none = dt().rotary(q, None, rot, **at)
    assert none is None
    # (an angle in 64 bits: two roundings of up to 2^25 turns' fraction of their 2^-53, far below h)
    check(out, turn64(q.double(), pos, rot), turn64(q.double(), pos, rot, size=True), 6, torch.float32)


def test_the_last_positions(gpu):
    """The angle at the end of 32 bits: position and frequency in turns are each off by 2^-53 of the angle, the product too."""
    rot = dt().Rotary()
    pos = torch.tensor([[2**31 - 1, 2**31 - 2, -2**31, 2**30 + 1]], dtype=torch.int32, device="cuda")
    q = randn((1, 4, 3, D), 4)
    out, _ = dt().rotary(q, None, rot, positions=pos)
    angle = 3 * 2.0 ** 31 * 2.0 ** -53
    check(out, turn64(q.double(), pos, rot), turn64(q.double(), pos, rot, size=True), 6 + angle / H24, torch.float32)
    assert torch.equal(out, dt().rotary(q, None, rot, positions=pos.long())[0])


@pytest.mark.parametrize("B", [32, 33, 256])
def test_starts_of_many_rows(gpu, B):
    rot = dt().Rotary(dims=64)
    starts = np.arange(B) * 31 % 977
    q, k = randn((B, 2, 4, D), 5), randn((B, 2, 1, D), 6)
    pos = default_positions(B, 2, starts)
    a = dt().rotary(q, k, rot, starts=starts)
    b = dt().rotary(q, k, rot, positions=pos.int())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(a[0], turn64(q.double(), pos, rot), turn64(q.double(), pos, rot, size=True), 6, torch.float32)
    many = randn((300, 1, 2, D), 7)  # (more rows than starts can name: position 0)
    assert torch.equal(dt().rotary(many, None, rot)[0], many)


def norm64(x, w):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dims,B,T,H,Hk", [(128, 1, 1, 1, 1), (96, 2, 7, 5, 3), (16, 1, 33, 16, 4), (128, 3, 50, 16, 16), (64, 2, 9, 12, 0)])
def test_head_norm(gpu, tdt, layout, dims, B, T, H, Hk):
    rot = dt().Rotary(dims=dims, layout=layout, magnitude=0.75)
    q, k = randn((B, T, H, D), 1, tdt, 2.0), (randn((B, T, Hk, D), 2, tdt, 0.5) if Hk else None)
    wq, wk = 1 + 0.1 * randn((D,), 3), 1 + 0.1 * randn((D,), 4)
    starts = np.arange(B) * 100
    pos = default_positions(B, T, starts)
    out = dt().head_norm_rotary(q, k, wq, wk, rot, starts=starts, eps=EPS)
    for x, w, y in zip((q, k), (wq, wk), out):
        if x is None:
            assert y is None
            continue
        n = norm64(x.double(), w.double())
        check(y, turn64(n, pos, rot), turn64(n, pos, rot, size=True), 21, tdt)


def grads64(d, x, w, pos, rot):
    """dx, dw and the sizes that bound their errors."""
    g = turn64(d.double(), pos, rot, -1.0)
    size = turn64(d.double(), pos, rot, size=True)  # of g: off by 6 h of it
    x, w = x.double(), w.double()
    inv = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    n = x * inv
    dx = inv * (w * g - n * (w * g * n).mean(-1, keepdim=True))
    A = w.abs() * size
    # w g: 6 h of the rotation, 1 h, 13 h of the factor in front, 3 h of products and the difference; the mean's terms 6 + 1 + 14 h,
    # their sum 20 h, the n and inv in front 13 h each and 4 h
    dx_size = inv * (23 * A + n.abs() * 61 * (A * n.abs()).mean(-1, keepdim=True))
    return dx, (g * n).sum((0, 1, 2)), dx_size, (size * n.abs()).sum((0, 1, 2))


@pytest.mark.parametrize("tdt", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dims,B,T,H,Hk", [(128, 1, 1, 1, 1), (96, 2, 7, 5, 3), (16, 1, 33, 16, 4), (128, 3, 50, 16, 16), (64, 2, 9, 12, 0),
                                           (128, 1, 3001, 16, 2)])
def test_head_norm_gradients(gpu, tdt, layout, dims, B, T, H, Hk):
    rot = dt().Rotary(dims=dims, layout=layout, magnitude=0.75)
    q, k = randn((B, T, H, D), 1, tdt, 2.0), (randn((B, T, Hk, D), 2, tdt, 0.5) if Hk else None)
    dq, dk = randn((B, T, H, D), 5, tdt), (randn((B, T, Hk, D), 6, tdt) if Hk else None)
    wq, wk = 1 + 0.1 * randn((D,), 3), 1 + 0.1 * randn((D,), 4)
    pos = default_positions(B, T)
    r = dt().head_norm_rotary_backward(dq, dk, q, k, wq, wk, rot, eps=EPS)
    again = dt().head_norm_rotary_backward(dq, dk, q, k, wq, wk, rot, positions=pos.int(), eps=EPS)
    for d, x, w, dx, dw, dx2, dw2 in ((dq, q, wq, r.d_Q, r.d_q_weight, again.d_Q, again.d_q_weight),
                                      (dk, k, wk, r.d_K, r.d_k_weight, again.d_K, again.d_k_weight)):
        if x is None:
            assert dx is None and dw is None
            continue
        ref, ref_w, size, size_w = grads64(d, x, w, pos, rot)
        check(dx, ref, size, 1, tdt)
        # a term: 6 h of the rotation, 13 + 2 h; sums of all tokens and heads in chains: a lane's (items over 2048 waves), 3 and 4
        # of a workgroup, 32 and 16 of the workgroups
        items = B * T * ((x.shape[2] + 7) // 8)
        check(dw, ref_w, size_w, 21 + items / 2048 + 1 + 55, torch.float32)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_heads_that_are_none_do_not_reach_the_other_heads_weights(gpu):
    """9 heads: the last group of eight has one. A NaN in a head of q makes q's weights' gradient NaN, not k's."""
    rot = dt().Rotary()
    q, k, dq, dk = randn((1, 3, 9, D), 1), randn((1, 3, 9, D), 2), randn((1, 3, 9, D), 3), randn((1, 3, 9, D), 4)
    w = torch.ones(D, device="cuda")
    want = dt().head_norm_rotary_backward(dq, dk, q, k, w, w, rot)
    q[0, 1, 8, 5] = float("nan")
    r = dt().head_norm_rotary_backward(dq, dk, q, k, w, w, rot)
    assert torch.equal(r.d_K, want.d_K) and torch.equal(r.d_k_weight, want.d_k_weight)
    assert torch.isnan(r.d_Q[0, 1, 8]).all() and int(torch.isnan(r.d_Q).sum()) == D
    assert torch.isnan(r.d_q_weight).all()


def test_gradients_against_differences(gpu):
    """<d, f(x + e v) - f(x - e v)> / 2e of the 64-bit formula against the kernel's gradients along v."""
    rot = dt().Rotary(dims=96, layout="interleaved")
    q, d, v = randn((1, 5, 3, D), 1), randn((1, 5, 3, D), 2), randn((1, 5, 3, D), 3)
    w, u = 1 + 0.1 * randn((D,), 4), randn((D,), 5)
    pos = default_positions(1, 5)
    r = dt().head_norm_rotary_backward(d, None, q, None, w, None, rot, eps=EPS)
    f = lambda x, y: (d.double() * turn64(norm64(x, y), pos, rot)).sum()
    e = 1e-4
    x, y = q.double(), w.double()
    along_x = (f(x + e * v, y) - f(x - e * v, y)) / (2 * e)
    along_w = (f(x, y + e * u) - f(x, y - e * u)) / (2 * e)
    # the difference is off by e^2 times the third derivative (of the order of the sizes' sum: 2000), the kernel by fp32
    assert abs(float((r.d_Q.double() * v).sum() - along_x)) < 2e-5 * 2000
    assert abs(float((r.d_q_weight.double() * u).sum() - along_w)) < 2e-5 * 2000


@pytest.mark.parametrize("tdt", TYPES)
def test_views_of_a_projection_and_in_place(gpu, tdt):
    B, T, H, Hk = 2, 6, 5, 2
    qkv = randn((B, T, (H + 2 * Hk) * D), 1, tdt)
    before = qkv.clone()
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
    w = 1 + 0.1 * randn((D,), 2)
    rot = dt().Rotary(dims=64)
    dense = dt().head_norm_rotary(q.contiguous(), k.contiguous(), w, w, rot)
    strided = dt().head_norm_rotary(q, k, w, w, rot)
    assert torch.equal(qkv, before)
    rq, rk = dt().head_norm_rotary(q, k, w, w, rot, inplace=True)
    assert rq is q and rk is k
    for a, b, c in zip(dense, strided, (q, k)):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert torch.equal(qkv[..., (H + Hk) * D:], before[..., (H + Hk) * D:])  # (the values beside them stay)
    # strides and alignments that no row of 16-byte pieces has are copied, and refused in place
    odd = randn((B, T, H, D + 1), 3, tdt)[..., :D]
    assert torch.equal(dt().rotary(odd, None, rot)[0], dt().rotary(odd.contiguous(), None, rot)[0])
    swapped = randn((B, H, T, D), 4, tdt).transpose(1, 2)
    assert torch.equal(dt().rotary(swapped, None, rot)[0], dt().rotary(swapped.contiguous(), None, rot)[0])
    for x in (odd, swapped):
        with pytest.raises(ValueError, match="in place"):
            dt().rotary(x, None, rot, inplace=True)


def test_infinities_large_and_zero_rows(gpu):
    rot = dt().Rotary(dims=64)
    q = randn((1, 5, 2, D), 1)
    q[0, 0, 0, 100] = float("inf")  # (a value that does not turn)
    q[0, 1, 0, 3] = float("nan")
    q[0, 2] *= 1e25                 # squares past fp32's range
    q[0, 3] = 0
    q[0, 4] *= 1e-30
    y = dt().rotary(q, None, rot)[0]
    assert torch.equal(y[0, 0, 0, 64:], q[0, 0, 0, 64:]) and torch.isfinite(y[0, 0, 0, :64]).all()
    assert torch.isnan(y[0, 1, 0, [3, 35]]).all() and int(torch.isnan(y).sum()) == 2
    w = torch.ones(D, device="cuda")
    n = dt().head_norm_rotary(q, None, w, None, rot)[0]
    assert torch.isfinite(n[0, 0, 1]).all() and torch.isnan(n[0, 1, 0]).all() and torch.isfinite(n[0, 1, 1]).all()
    pos = default_positions(1, 5)
    ref = norm64(q.double(), w.double())
    check(n[:, 2:], turn64(ref, pos, rot)[:, 2:], turn64(ref, pos, rot, size=True)[:, 2:], 21, torch.float32)
    assert bool((n[0, 3] == 0).all())
    d = randn((1, 5, 2, D), 2)
    r = dt().head_norm_rotary_backward(d, None, q, None, w, None, rot)
    ref, _, size, _ = grads64(d, q, w, pos, rot)
    check(r.d_Q[:, 2:], ref[:, 2:], size[:, 2:], 1, torch.float32)


@pytest.mark.parametrize("tdt", TYPES)
def test_host_arrays(gpu, tdt):
    B, T, H, Hk = 2, 5, 4, 2
    q, k, d, e = (randn((B, T, n, D), i, tdt) for i, n in ((1, H), (2, Hk), (3, H), (4, Hk)))
    w, v = 1 + 0.1 * randn((D,), 5), 1 + 0.1 * randn((D,), 6)
    host = lambda t: (t.view(torch.int16).cpu().numpy().view(np.uint16) if t.dtype == torch.bfloat16 else t.cpu().numpy())
    same = lambda a, t: np.array_equal(a.view(np.uint8), np.ascontiguousarray(host(t)).view(np.uint8))
    rot = dt().Rotary(dims=96, layout="interleaved")
    pos = torch.randint(0, 5000, (B, T), device="cuda")
    p = pos.cpu().numpy()
    for a, b in zip(dt().rotary(host(q), host(k), rot, positions=p), dt().rotary(q, k, rot, positions=pos)):
        assert same(a, b)
    for a, b in zip(dt().head_norm_rotary(host(q), host(k), host(w), host(v), rot, starts=[3, 9]),
                    dt().head_norm_rotary(q, k, w, v, rot, starts=[3, 9])):
        assert same(a, b)
    hr = dt().head_norm_rotary_backward(host(d), host(e), host(q), host(k), host(w), host(v), rot, positions=p.astype(np.int32))
    dr = dt().head_norm_rotary_backward(d, e, q, k, w, v, rot, positions=pos)
    for a, b in zip((hr.d_Q, hr.d_K, hr.d_q_weight, hr.d_k_weight), (dr.d_Q, dr.d_K, dr.d_q_weight, dr.d_k_weight)):
        assert same(a, b)
    x = host(q).copy()
    y, _ = dt().rotary(x, None, rot, inplace=True)
    assert y is x and same(x, dt().rotary(q, None, rot)[0])


def test_streams_and_graph_replays(gpu):
    """The gradients' workspace: calls on two streams at once, and a captured call between eager ones."""
    rot = dt().Rotary()
    n = [(1, 400, 16, D), (3, 77, 16, D)]
    q = [randn(s, i) for i, s in enumerate(n)]
    d = [randn(s, 10 + i) for i, s in enumerate(n)]
    w = 1 + 0.1 * randn((D,), 5)
    call = lambda i: dt().head_norm_rotary_backward(d[i], None, q[i], None, w, None, rot)
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in n]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r.d_Q, want[i].d_Q) and torch.equal(r.d_q_weight, want[i].d_q_weight)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = call(0)
        y = dt().head_norm_rotary(q[1], None, w, None, rot, starts=[5, 6, 7])[0]
    for i in range(4):
        q[0].copy_(randn(n[0], 100 + i))
        q[1].copy_(randn(n[1], 200 + i))
        call(1)
        g.replay()
        after = call(0)
        torch.cuda.synchronize()
        assert torch.equal(r.d_Q, after.d_Q) and torch.equal(r.d_q_weight, after.d_q_weight)
        assert torch.equal(y, dt().head_norm_rotary(q[1], None, w, None, rot, starts=[5, 6, 7])[0])


def test_offsets_past_32_bits(gpu):
    """Rows whose last token lies more than 2^32 bytes behind the first."""
    T, H = 70000, 256
    x = torch.zeros((1, T, H, D), dtype=torch.bfloat16, device="cuda")
    x[:, -3:] = randn((1, 3, H, D), 1, torch.bfloat16)
    rot = dt().Rotary()
    pos = torch.arange(T, device="cuda", dtype=torch.int32)[None]
    y = dt().rotary(x, None, rot)[0]
    z = dt().rotary(x[:, -3:], None, rot, positions=pos[:, -3:])[0]
    assert torch.equal(y[:, -3:], z)
    assert bool((y[:, 5:-3:999] == 0).all())


def test_refusals(gpu):
    rot = dt().Rotary()
    q, k = randn((2, 3, 4, D), 1), randn((2, 3, 2, D), 2)
    w = torch.ones(D, device="cuda")
    for bad in (dict(layout="other"), dict(scaling="other"), dict(frequencies=[1.0])):
        with pytest.raises(ValueError):
            dt().Rotary(**bad)
    with pytest.raises(ValueError, match="128"):
        dt().rotary(q[..., :64], None, rot)
    with pytest.raises(ValueError):
        dt().rotary(q, k[:1], rot)
    with pytest.raises(TypeError):
        dt().rotary(q, k.bfloat16(), rot)
    with pytest.raises(TypeError):
        dt().rotary(q.half(), None, rot)
    with pytest.raises(ValueError, match="ROCm"):
        dt().rotary(q.cpu(), None, rot)
    with pytest.raises(ValueError, match="exclude"):
        dt().rotary(q, k, rot, positions=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), starts=[0, 0])
    with pytest.raises(ValueError, match="shape"):
        dt().rotary(q, k, rot, positions=torch.zeros((2, 2), dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        dt().rotary(q, k, rot, positions=torch.zeros((2, 3), device="cuda"))
    with pytest.raises(ValueError):
        dt().rotary(q, k, rot, starts=[1])
    with pytest.raises(dt().DTError, match="T=0"):
        dt().rotary(q[:, :0], None, rot)
    with pytest.raises(dt().DTError, match="other"):
        dt().rotary(q, q, rot, inplace=True)
    with pytest.raises(ValueError, match="q_weight"):
        dt().head_norm_rotary(q, None, w[:64], None, rot)
    with pytest.raises(ValueError, match="k_weight"):
        dt().head_norm_rotary(q, k, w, w.bfloat16(), rot)
    with pytest.raises(dt().DTError, match="eps"):
        dt().head_norm_rotary(q, k, w, w, rot, eps=0.0)
    with pytest.raises(ValueError):
        dt().head_norm_rotary_backward(q, None, q, k, w, w, rot)
    with pytest.raises(ValueError):
        dt().head_norm_rotary_backward(q, k, q, randn((2, 3, 1, D), 3), w, w, rot)
