"""SiLU * mul quantised: values close to a half between two integers, on either side, go to the nearer one.  Gates of 20 and more have
SiLU(g) = g to 2e-9, so y = g * up is a product of two 16-bit numbers, exact in 32 bits, and 127 y / max can be reckoned exactly."""
import numpy as np
import pytest
import torch

from semi_pd_b200 import ops

pytestmark = pytest.mark.gpu

# The factor 1 / (1 + e^-g) is the same number for all of them.  What is rounded on the way, 2^-24 each: g times that factor and the
# product with up, both for the value and for the maximum, and the quotient 127 / max; the last sum rounds to the integer.
ERROR = 5.1 * 2.0 ** -24


def pairs_beside_halves(dtype, rng, side):
    """(gates, ups, integers) of one row, the largest product first: 127 y / max is 1 to 2 times ERROR below a half (side -1) or above."""
    bits = 7 if dtype == torch.bfloat16 else 10
    g, u = rng.integers(2 ** bits, 2 * 2 ** bits, (2, 1_000_000))
    down = 2.0 ** -rng.integers(0, 7, g.shape)
    for _ in range(100):  # (products of 8 bits each come that close to a half for some maxima only)
        top_g, top_u = 2 * 2 ** bits - 1 - 2 * rng.integers(0, 2 ** (bits - 2), 2)
        t = 127 * (g * u * down) / float(top_g * top_u)
        away = side * (t - np.floor(t) - 0.5) / t
        hit = np.flatnonzero((away > 1.05 * ERROR) & (away < 2 * ERROR) & (t < 127))[:2047]
        if len(hit) >= 4:
            break
    assert len(hit) >= 4
    gates, ups = g[hit] * (32 / 2 ** bits), u[hit] * down[hit] / 2 ** bits  # gates of 32 to 64
    n = np.floor(t[hit] + 0.5)
    return (np.concatenate([[top_g * 32 / 2 ** bits], gates]), np.concatenate([[top_u / 2 ** bits], ups]), np.concatenate([[127], n]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("side", [-1, 1])
@pytest.mark.parametrize("rows", [6, 6000])
def test_next_to_halves(dtype, side, rows):
    rng = np.random.default_rng(7 + side)
    k, distinct = 2048, 6
    x = torch.zeros(distinct, 2 * k, dtype=torch.float64)
    want = torch.zeros(distinct, k, dtype=torch.int8)
    for r in range(distinct):
        g, u, n = pairs_beside_halves(dtype, rng, side)
        signs = rng.choice([-1.0, 1.0], len(g))
        x[r, :len(g)], x[r, k:k + len(g)] = torch.from_numpy(g), torch.from_numpy(u * signs)
        want[r, :len(g)] = torch.from_numpy(n * signs).to(torch.int8)
    assert torch.equal(x.to(dtype).double(), x)
    x, want = x.to(dtype).cuda().repeat(rows // distinct, 1), want.cuda().repeat(rows // distinct, 1)
    q, _ = ops.silu_and_mul_quant_int8(x)
    assert torch.equal(q, want)
