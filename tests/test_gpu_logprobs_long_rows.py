"""16-bit log-probabilities over long rows: a sum leaves its accumulator in the tensor cores after 16 k-blocks of 64 products, or the k-blocks
go to several accumulators in turn."""
import pytest
import torch

from semi_pd_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 32, 64, 600])  # tokens on N, 8, 8 and 4 accumulators; tokens on M, chunks of 16 k-blocks
def test_ones_beside_a_large_product(m, dtype):
    """One product of 2^24, then a single 1 in each instruction of 16 products.  Next to 2^24 a 1 is half a place of fp32: in the same
    accumulator every one of them is lost, cut or rounded to even.  Only a quarter of the k-blocks at most may be in that accumulator: the
    others' sums are exact and so are the additions of their multiples of 4 up to 2^24 + 512."""
    k, v = 8192, 2000
    x = torch.zeros(m, k, device=DEV, dtype=dtype)
    w = torch.zeros(v, k, device=DEV, dtype=dtype)
    x[:, ::16] = 1
    x[:, 0] = 4096
    row = 1234
    w[row] = x[0]
    targets = torch.full((m,), row, device=DEV)
    logprobs, lse = ops.linear_logprobs(x, w, targets)
    kept = lse.double() - 2.0 ** 24
    places = 4  # the result in units of 1, half a place: the logit times log2 e, its logarithm's sum, times ln 2, and their constants
    assert (kept >= 384 - places).all() and (kept <= 511 + places).all(), kept
    assert (logprobs.abs() <= places).all()
    assert torch.equal(lse, lse[:1].expand(m))
