"""Drafts drawn from nearly the model's own probabilities: p and q agree to rounding almost everywhere, so what max(p - q, 0) leaves of a
value follows from the last digits of the rows' sums. Tokens are those of the definition in 64 bits, with the border's slack that
test_verify_drafts_gpu derives: 2e-11 of the probabilities' sum."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_verify_drafts_gpu import BORDER, check, reference

pytestmark = pytest.mark.gpu


def dt():
    import dirktensor_amd

    return dirktensor_amd


def close_rows(V, T, seed, share=2e-10):
    """Logits x [V] and draft logits y, equal but for the last eight values (more likely in x, by 0.008 of the sum together), the eight before
    them (less likely) and one that brings the rows' sums to 1 - share of each other: all the others have p - q = share p."""
    rng = np.random.default_rng(seed)
    x = 2 * rng.standard_normal(V)
    total = np.exp(x / T).sum()
    x[-17:] = T * np.log(total * (3e-3 + 1e-3 * rng.random(17)))
    x[-17] = T * np.log(total * 1e-5)
    x = x.astype(np.float32)
    y = x.copy()
    e = lambda v: np.exp(v.astype(np.float64) / T)
    y[-8:] = T * np.log(e(x[-8:]) - 1e-3 * total)
    y[-16:-8] = T * np.log(e(x[-16:-8]) + 1e-3 * total)
    rest = np.arange(V) != V - 17
    y[-16] = T * np.log(e(x).sum() - e(np.delete(y, V - 16)).sum())  # (to fp32's steps of this value; then of one much smaller)
    y[-17] = T * np.log(e(x).sum() / (1 - share) - e(y[rest]).sum())
    assert abs(e(x).sum() / e(y).sum() - (1 - share)) < 0.1 * abs(share)
    return x, y


@pytest.mark.parametrize("V", [4001, 50021])
@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("share", [2e-10, -2e-10])
def test_what_is_left_of_close_rows(gpu, V, T, share):
    """The refused draft is one that y favours. What is left: 2e-10 of the sum, or nothing, in the values that agree, 0.008 at the last
    eight."""
    n, B = 12, 8
    u = torch.full((B, 2), 0.999, device="cuda")
    u[:, 1] = torch.tensor([0.0, 1e-9, 3e-9, 7e-9, 1e-8, 1.5e-8, 0.3, 0.99])
    d = torch.full((B, 1), V - 12, dtype=torch.int32, device="cuda")
    wrong = []
    for seed in range(n):
        x, y = (torch.from_numpy(v).cuda() for v in close_rows(V, T, seed, share))
        X, Y = x.expand(B, 2, V), y.expand(B, 1, V)
        r = dt().verify_drafts(X, d, u, draft_logits=Y, temperature=T)
        want = reference(X, d, u, Y, T)
        first = want[1][:, 0]
        assert (want[0] == 0).all() and (first[6:] >= V - 8).all()
        assert first[0] == 0 and len(set(first[:6].tolist())) >= 5 if share > 0 else (first >= V - 17).all()
        # (thousands of borders lie within BORDER of each other: more than the reference names)
        p, q = (np.exp((v - v.max()) / T) for v in (t.cpu().numpy().astype(np.float64) for t in (x, y)))
        p, q = p / p.sum(), q / q.sum()
        w = np.concatenate([[0.0], np.maximum(p - q, 0).cumsum()])
        got = r.tokens[:, 0].cpu().numpy()
        bound = u[:, 1].cpu().numpy().astype(np.float64) * w[-1]
        off = np.maximum(w[got] - bound, bound - w[got + 1])
        if not (off <= BORDER).all():
            wrong.append((seed, off.tolist(), got.tolist(), first.tolist()))
        want[1][:, 0], want[2][:, 0] = got, np.log(p[got])
        check(r, want)
    assert not wrong, wrong
