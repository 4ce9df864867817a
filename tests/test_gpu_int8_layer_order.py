"""A layer's weight quantised and multiplied by right away, in memory that held another layer's integers."""
import pytest
import torch

from semi_pd_b200 import layers

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("n,k", [(4096, 4096), (28672, 4096), (264, 14336)])
def test_quantised_and_used(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m + n)
    src = [(torch.randn(n, k, generator=g, device=DEV) * k ** -0.5).bfloat16() for _ in range(2)]
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()

    def run(w, wait):
        layer = layers.ColumnParallelLinear(k, n)
        layer.weight = w
        layer.quantize_weight_int8()
        if wait:
            torch.cuda.synchronize()
        return layer(x)[0]

    want = [run(w, True) for w in src]
    assert not torch.equal(*want)
    for i in range(30):
        got = run(src[i % 2], False)
        assert torch.equal(got, want[i % 2]), i
