"""Gradients of each head's norm and rotation over many batch rows, where a wave's next token is another row's. With the bounds of
test_rotary_gpu."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_rotary_gpu import EPS, check, default_positions, grads64, randn

pytestmark = pytest.mark.gpu

D = 128


def dt():
    import dirktensor_amd

    return dirktensor_amd


def weights():
    return 1 + 0.1 * randn((D,), 3), 1 + 0.1 * randn((D,), 4)


def units(tokens, H, Hk):
    """What a column's sum is off by (test_head_norm_gradients): a term by 21 h, then one addition after another, a lane's (3072 waves share
    the groups of eight heads of both tensors), 3 and 4 of a workgroup, 48 and 16 of the workgroups."""
    groups = (H + 7) // 8 + (Hk + 7) // 8
    return 21 + -(-tokens * groups // 3072) + 71


@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["starts", "int64"])
@pytest.mark.parametrize("B,T,H,Hk", [(5, 1501, 3, 2), (250, 37, 2, 0), (256, 16, 9, 3), (4000, 1, 4, 1), (3001, 3, 1, 1), (7, 2000, 16, 4), (2, 5000, 20, 7)])
def test_gradients_of_many_rows(gpu, tdt, kind, B, T, H, Hk):
    """More tokens than waves: their next tokens lie a step of up to 3072 further, behind the ends of rows."""
    rot = dt().Rotary(dims=96, magnitude=0.75)
    q, dq = randn((B, T, H, D), 1, tdt, 2.0), randn((B, T, H, D), 5, tdt)
    k, dk = (randn((B, T, Hk, D), 2, tdt, 0.5), randn((B, T, Hk, D), 6, tdt)) if Hk else (None, None)
    wq, wk = weights()
    starts = (np.arange(B) * 7919) % 100003
    pos = default_positions(B, T, starts)
    at = dict(starts=starts) if kind == "starts" else dict(positions=pos.contiguous())
    if kind == "starts" and B > 256:  # (more rows than starts are for)
        at = dict(positions=pos.int())
    r = dt().head_norm_rotary_backward(dq, dk, q, k, wq, wk, rot, eps=EPS, **at)
    for d, x, w, dx, dw in ((dq, q, wq, r.d_Q, r.d_q_weight), (dk, k, wk, r.d_K, r.d_k_weight)):
        if x is None:
            continue
        ref_w, size_w = 0.0, 0.0
        for i in range(0, B, max(1, B // 8)):  # (64 bits: some rows at a time)
            j = slice(i, i + max(1, B // 8))
            ref, rw, size, sw = grads64(d[j], x[j], w, pos[j], rot)
            check(dx[j], ref, size, 1, tdt)
            ref_w, size_w = ref_w + rw, size_w + sw
        check(dw, ref_w, size_w, units(B * T, H, Hk), torch.float32)


def test_rows_of_one_token_take_no_longer(gpu):
    """The same tokens as four rows and as 32768: the same work, so the same time (a quarter more is allowed, of the shortest of
    many runs), and the same bits."""
    rot = dt().Rotary()
    n, H, Hk = 32768, 16, 4
    wq, wk = weights()
    x = [randn((n, h, D), i, torch.bfloat16) for i, h in enumerate((H, Hk, H, Hk))]
    pos = torch.randint(0, 8192, (n,), device="cuda", dtype=torch.int32)

    def call(B):
        dq, dk, q, k = (t.view(B, n // B, t.shape[1], D) for t in x)
        return dt().head_norm_rotary_backward(dq, dk, q, k, wq, wk, rot, positions=pos.view(B, n // B))

    def shortest(B):
        best = float("inf")
        for _ in range(20):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(5):
                call(B)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) / 5)
        return best

    few, many = call(4), call(n)
    assert torch.equal(few.d_Q.view(-1), many.d_Q.view(-1)) and torch.equal(few.d_K.view(-1), many.d_K.view(-1))
    assert torch.equal(few.d_q_weight, many.d_q_weight) and torch.equal(few.d_k_weight, many.d_k_weight)
    times = shortest(4), shortest(n)
    print(f"4 rows {1e3 * times[0]:.1f} us, {n} rows {1e3 * times[1]:.1f} us", flush=True)
    assert times[1] <= 1.25 * times[0]
