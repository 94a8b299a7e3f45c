"""Rows in the key/value cache: what is held against the formats' definitions in 64 bits, at lengths around the cache's
blocks of 32, by many small appends as by one, with rows of infinities and NaN, from strided views and from the host."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 128
FORMATS = ["int8", "fp8", "bf16"]


def held64(x, fmt):
    """What the cache stands for, in 64 bits, of finite rows x [..., D]."""
    x = x.detach().cpu().double()
    if fmt == "bf16":
        return x.float().bfloat16().double()
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        s = (amax / 127).float().double()
        q = torch.where(s > 0, x / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(x)).round()
        return q.clamp(-127, 127) * s
    e = torch.full_like(amax, -126.0)
    for cand in range(-126, 121):  # the smallest power of two that brings the row within 448
        e = torch.where(amax > 448 * 2.0 ** (cand - 1), torch.full_like(e, float(cand)), e) if cand > -126 else e
    s = 2.0 ** e
    y = x / s
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    q = (y / step).round() * step
    return torch.where((q * s).abs() < 2.0 ** 128, q, 240 * torch.sign(q)) * s  # (256 2^120 is past fp32's range)


def rows(shape, seed, tdt, wide=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if wide:  # rows of very different size, halves and ends of the int8 range hit exactly, zeros
        x = x * torch.exp(8 * torch.randn(shape[:-1], generator=g, device="cuda"))[..., None]
        x[..., 0, :] = torch.arange(D, device="cuda") * 0.5 - 0.5
        x[..., 0, 5] = 127.0
        x[..., 0, 0, :, :] = 0.0
    return x.to(tdt)


def check(got, x, fmt):
    """The values come back in the mode they went in: one rounding of the held value (none is left in 32 bits but that of
    the product with the scale)."""
    want = held64(x, fmt)
    eps = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    err = (got.cpu().double() - want).abs()
    # (bf16: the 32-bit product is rounded before; below the normal range a step is 2^-149 or bf16's 2^-133)
    tiny = 2.0 ** -134 if got.dtype == torch.bfloat16 else 2.0 ** -150
    assert bool((err <= want.abs() * (eps + 2.0 ** -24) + 2 * tiny).all()), float((err / want.abs().clamp_min(1e-30)).max())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (2, 31, 3), (3, 32, 2), (1, 33, 16), (2, 200, 5)])
def test_held_values(fmt, tdt, B, T, H):
    from dirktensor_amd import KVCache

    print(f"held values {fmt} {tdt} B={B} T={T} H={H}", flush=True)
    c = KVCache(B, T + 3, H, format=fmt)
    k, v = rows((B, T, H, D), 1, tdt, wide=True), rows((B, T, H, D), 2, tdt, wide=True)
    c.append(k, v)
    assert c.lengths.tolist() == [T] * B
    mode = "fp32" if tdt == torch.float32 else "bf16"
    gk, gv = c.read([0] * B, T, mode=mode)
    check(gk, k, fmt)
    check(gv, v, fmt)
    # the other mode rounds the same held values
    ok, ov = c.read([0] * B, T, mode="bf16" if mode == "fp32" else "fp32")
    for other, x in ((ok, k), (ov, v)):
        check(other, x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_appends_of_any_length_hold_the_same(fmt):
    """Runs of 1, 5, 32, 26, 64, 70 tokens, ragged over the slots in any order, hold what one append holds; the other
    slots and the bytes behind the sequences stay as they were."""
    from dirktensor_amd import KVCache

    B, T, H = 3, 198, 4
    k, v = rows((B, T, H, D), 3, torch.float32), rows((B, T, H, D), 4, torch.float32)
    one, many = KVCache(B, T, H, format=fmt), KVCache(5, 256, H, format=fmt)
    one.append(k, v)
    other = rows((1, 256, H, D), 5, torch.float32)
    many.append(other, other, slots=[2])
    slots = [4, 0, 3]
    at = np.zeros(B, int)
    rng = np.random.default_rng(0)
    for run in (1, 5, 32, 26, 64, 70) * 4:
        cnt = np.minimum(rng.integers(0, run + 1, size=B), T - at)
        pick = lambda x: torch.stack([torch.cat([x[b, at[b]:at[b] + cnt[b]], x.new_full((run - cnt[b], H, D), 7.0)])
                                      for b in range(B)])
        many.append(pick(k), pick(v), slots=slots, counts=cnt)
        at += cnt
        assert many.lengths[slots].tolist() == at.tolist()
    n = int(at.min())
    assert n > 64
    for b in range(B):
        for x, y in zip(one.read([0], int(at[b]), slots=[b], mode="fp32"), many.read([0], int(at[b]), slots=[slots[b]], mode="fp32")):
            assert torch.equal(x, y)
        a, z = one.read([n // 2], 7, slots=[b], mode="fp32"), many.read([n // 2], 7, slots=[slots[b]], mode="fp32")
        assert torch.equal(a[0], z[0]) and torch.equal(a[1], z[1])
    check(many.read([0], 256, slots=[2], mode="fp32")[0], other, fmt)
    assert many.lengths.tolist()[1] == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_infinities_and_nan_make_their_row_nan(fmt):
    from dirktensor_amd import KVCache

    T, H = 40, 2
    k, v = rows((1, T, H, D), 6, torch.float32), rows((1, T, H, D), 7, torch.float32)
    k[0, 3, 1, 100] = float("inf")
    k[0, 33, 0, 0] = float("-inf")
    v[0, 3, 0, 17] = float("nan")
    v[0, 39, 1, 127] = 3.4e38  # infinite as bf16, a number in the others
    c = KVCache(1, T, H, format=fmt)
    c.append(k, v)
    for mode in ("fp32", "bf16"):
        gk, gv = c.read([0], T, mode=mode)
        want_k, want_v = torch.zeros((1, T, H), dtype=torch.bool), torch.zeros((1, T, H), dtype=torch.bool)
        want_k[0, 3, 1] = want_k[0, 33, 0] = want_v[0, 3, 0] = True
        if fmt == "bf16":
            want_v[0, 39, 1] = True
        assert torch.equal(torch.isnan(gk).all(-1).cpu(), want_k) and torch.equal(torch.isnan(gk).any(-1).cpu(), want_k)
        assert torch.equal(torch.isnan(gv).all(-1).cpu(), want_v) and torch.equal(torch.isnan(gv).any(-1).cpu(), want_v)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_ends_of_the_range(fmt):
    """Rows at the top of fp32's range and below its normal one."""
    from dirktensor_amd import KVCache

    H = 8
    x = torch.zeros((1, 1, H, D), device="cuda")
    x[0, 0, 0] = torch.linspace(-1, 1, D) * 3.4e38
    x[0, 0, 1] = torch.linspace(-1e-37, 1e-37, D)
    x[0, 0, 2] = torch.linspace(-1e-40, 1e-40, D)
    x[0, 0, 3, 5] = 1e-45
    x[0, 0, 4] = torch.linspace(-0.4, 0.4, D) * 2.0 ** -113  # (around where int8 divides by its scale)
    x[0, 0, 5] = 448.0
    x[0, 0, 6] = 448.0 * (1 + 2.0 ** -23)
    x[0, 0, 7] = -1.0
    c = KVCache(1, 4, H, format=fmt)
    c.append(x, x)
    check(c.read([0], 1, mode="fp32")[1], x, fmt)


def test_strided_rows():
    """Column blocks of a projection's output are taken as they are, other strides are copied; both hold the same."""
    from dirktensor_amd import KVCache

    B, T, H = 2, 37, 3
    g = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn((B, T, 3 * H * D), generator=g, device="cuda").bfloat16()
    k, v = (qkv[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in (1, 2))
    want = KVCache(B, T, H)
    want.append(k.contiguous(), v.contiguous())
    ref = want.read([0, 0], T)
    for kk, vv in ((k, v), (k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), v),
                   (torch.cat([k, k], -1)[..., :D], v)):
        c = KVCache(B, T, H)
        c.append(kk, vv)
        got = c.read([0, 0], T)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    c = KVCache(B, T, H)
    same = k[:1, :1].expand(2, 5, H, D)  # one token's rows, many times
    c.append(same, same)
    assert torch.equal(c.read([0, 0], 5)[0], ref[0][:1, :1].expand(2, 5, H, D))


@pytest.mark.parametrize("fmt", FORMATS)
def test_host_rows(fmt):
    from dirktensor_amd import KVCache

    B, T, H = 2, 45, 2
    k, v = rows((B, T, H, D), 10, torch.float32), rows((B, T, H, D), 11, torch.float32)
    dev, host = KVCache(B, T, H, format=fmt), KVCache(B, T, H, format=fmt)
    dev.append(k, v)
    host.append(k.cpu().numpy(), v.cpu().numpy())
    a = dev.read([2, 4], 30, mode="fp32")
    b = host.read([2, 4], 30, mode="fp32", host=True)
    for x, y in zip(a, b):
        assert np.array_equal(x.cpu().numpy(), y)
    bits = host.read([2, 4], 30, mode="bf16", host=True)
    for x, y in zip(dev.read([2, 4], 30, mode="bf16"), bits):
        assert np.array_equal(x.view(torch.int16).cpu().numpy().view(np.uint16), y)


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(fmt):
    """Heads and slots whose bytes begin past 2^32."""
    from dirktensor_amd import KVCache

    slots, cap, H = (3, 1 << 20, 16) if fmt != "bf16" else (2, 1 << 20, 16)
    c = KVCache(slots, cap, H, format=fmt)  # 4 GiB of values a slot in 8 bits
    k, v = rows((1, 70, H, D), 12, torch.bfloat16), rows((1, 70, H, D), 13, torch.bfloat16)
    zero = torch.zeros((1, 1 << 15, H, D), dtype=torch.bfloat16, device="cuda")
    for _ in range(31):
        c.append(zero, zero, slots=[slots - 1])
    c.append(zero, zero, slots=[slots - 1], counts=[(1 << 15) - 70])
    c.append(k, v, slots=[slots - 1])
    assert c.lengths[slots - 1] == cap
    gk, gv = c.read([cap - 70], 70, slots=[slots - 1])
    check(gk, k, fmt)
    check(gv, v, fmt)
    assert not bool(c.read([cap - 100], 30, slots=[slots - 1])[1].any())
    c.close()


def test_refusals():
    from dirktensor_amd import DTError, KVCache

    c = KVCache(2, 10, 2)
    x = torch.zeros((2, 4, 2, D), device="cuda")
    c.append(x, x)
    for kw, msg in ((dict(slots=[0, 0]), "both"), (dict(slots=[0, 2]), "outside"), (dict(counts=[5, 0]), "outside"),
                    (dict(counts=[-1, 0]), "outside")):
        with pytest.raises(DTError, match=msg):
            c.append(x, x, **kw)
    big = torch.zeros((1, 7, 2, D), device="cuda")
    with pytest.raises(DTError, match="do not fit"):
        c.append(big, big)
    c.append(big, big, counts=[6])
    assert c.lengths.tolist() == [10, 4]  # nothing moved in the refused calls
    with pytest.raises(DTError, match="holds 4"):
        c.read([0, 0], 5)
    with pytest.raises(DTError, match="outside"):
        c.truncate([11, 4])
    with pytest.raises(DTError, match="outside"):
        c.truncate([3, -1])
    c.truncate([3, 0])
    assert c.lengths.tolist() == [3, 0]
    with pytest.raises(ValueError):
        c.append(x[..., :64], x[..., :64])
    with pytest.raises(ValueError):
        c.append(x.cpu(), x.cpu())
    with pytest.raises(TypeError):
        c.append(x, x.bfloat16())
    with pytest.raises(TypeError):
        c.append(x.half(), x.half())
    with pytest.raises(ValueError):
        c.append(x, x, slots=[0.5, 1.0])
    with pytest.raises(ValueError):
        c.append(x, x, slots=[0, 1, 2])
    with pytest.raises(ValueError):
        KVCache(1, 1, 1, format="int4")
    with pytest.raises(DTError, match="cannot be had"):
        KVCache(65535, 1 << 20, 16)
    c.close()
    with pytest.raises(RuntimeError, match="closed"):
        c.append(x, x)
