"""Rotations, norms and their gradients of tensors that go past the caches: bit for bit what the same rows give in small calls, and the
formulas in 64 bits on some of them (with the bounds of test_rotary_gpu)."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_rotary_gpu import D, check, default_positions, grads64, norm64, randn, turn64
from test_rotary_rows_gpu import dt, units, weights

pytestmark = pytest.mark.gpu


# (results of 105 MB, which stay in the last-level cache, of 180 MB, where the gradient's rows go past it, and of 300 MB, where all do)
@pytest.mark.parametrize("tdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,Hk", [(2, 5127, 16, 4), (1, 17579, 16, 4), (3, 9767, 16, 4)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_large_tensors(gpu, tdt, B, T, H, Hk, layout):
    rot = dt().Rotary(dims=112, layout=layout)
    T = T if tdt == torch.float32 else 2 * T + 1
    q, k, dq, dk = (randn((B, T, h, D), i, tdt) for i, h in enumerate((H, Hk, H, Hk)))
    wq, wk = weights()
    starts = np.arange(B) * 500 + 3
    pos = default_positions(B, T, starts)
    at = dict(starts=starts)
    plain = dt().rotary(q, k, rot, **at)
    back = dt().rotary_backward(dq, dk, rot, **at)
    norm = dt().head_norm_rotary(q, k, wq, wk, rot, **at)
    grad = dt().head_norm_rotary_backward(dq, dk, q, k, wq, wk, rot, **at)
    whole = (*plain, *back, *norm, grad.d_Q, grad.d_K)
    for b in range(B):
        for i in range(0, T, 997):
            j = slice(i, min(i + 997, T))
            s = dict(starts=[int(starts[b]) + i])
            part = [t[b:b + 1, j].contiguous() for t in (q, k, dq, dk)]
            g = dt().head_norm_rotary_backward(part[2], part[3], part[0], part[1], wq, wk, rot, **s)
            small = (*dt().rotary(part[0], part[1], rot, **s), *dt().rotary_backward(part[2], part[3], rot, **s),
                     *dt().head_norm_rotary(part[0], part[1], wq, wk, rot, **s), g.d_Q, g.d_K)
            for big, few in zip(whole, small):
                assert torch.equal(big[b:b + 1, j], few)
    j = slice(T - 300, T)
    for x, d, w, y, z, m, g in zip((q, k), (dq, dk), (wq, wk), plain, back, norm, (grad.d_Q, grad.d_K)):
        x, d, p = x[:, j], d[:, j], pos[:, j]
        check(y[:, j], turn64(x.double(), p, rot), turn64(x.double(), p, rot, size=True), 6, tdt)
        check(z[:, j], turn64(d.double(), p, rot, -1.0), turn64(d.double(), p, rot, size=True), 6, tdt)
        e = norm64(x.double(), w.double())
        check(m[:, j], turn64(e, p, rot), turn64(e, p, rot, size=True), 21, tdt)
        ref, _, size, _ = grads64(d, x, w, p, rot)
        check(g[:, j], ref, size, 1, tdt)
    for x, d, w, dw in ((q, dq, wq, grad.d_q_weight), (k, dk, wk, grad.d_k_weight)):
        ref, size = 0.0, 0.0
        for b in range(B):
            _, rw, _, sw = grads64(d[b:b + 1], x[b:b + 1], w, pos[b:b + 1], rot)
            ref, size = ref + rw, size + sw
        check(dw, ref, size, units(B * T, H, Hk), torch.float32)
