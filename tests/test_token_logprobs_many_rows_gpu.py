"""The gradient of as many rows as the forward takes: more workgroups than one launch has."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_gradient_of_more_rows_than_one_launch_takes():
    from dirktensor_amd import token_logprobs, token_logprobs_backward

    rows, V = (1 << 22) + 5, 4097  # two workgroups a row: 8388618
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 69 GB for the gradient")
    row = torch.randn(V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x = row.expand(rows, V)
    tok = torch.arange(rows, device="cuda") % V
    r = token_logprobs(x, tok)
    g = torch.randn(rows, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    d = token_logprobs_backward(g, x, tok, r)
    p = torch.softmax(row.double(), 0)
    # p is good to (110 + V / 256 + 4 (1 + |log p|)) 2^-24 relative, with |log p| < 20; the product and the sum are rounded once each
    tol = (110 + V / 256 + 84 + 2) * 2.0 ** -24
    step = 1 << 17
    print(f"gradient of {rows} rows of {V}", flush=True)
    for at in range(0, rows, step):
        end = min(rows, at + step)
        gs = g[at:end, None]
        want = (-gs * p.float()).scatter_add_(1, tok[at:end, None], gs)
        # (want in 32 bits: 3 roundings)
        bound = (tol + 3 * 2.0 ** -24) * (gs.abs() * p.float()).scatter_add_(1, tok[at:end, None], gs.abs()) + 1e-38
        assert bool(((d[at:end] - want).abs() <= bound).all()), at
    del d
    torch.cuda.empty_cache()
