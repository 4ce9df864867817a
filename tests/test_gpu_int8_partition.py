"""Products of 8-bit integers on the streams of a partition of the SMs: cut by the clusters that fit there, launched and captured, and on both
sides at once.  Integer sums have no order, so the results are the same bits as on the whole device."""
import pytest
import torch

from semi_pd_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def operands(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m + n)
    a = torch.randint(-128, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(m, 1, generator=g, device=DEV) + 0.5, torch.rand(n, 1, generator=g, device=DEV) + 0.5
    return a, b.t(), sa, sb, torch.bfloat16


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (64, 4096, 14336), (160, 2304, 8192), (256, 1024, 8192), (16, 5120, 5120),
                                   (500, 1024, 8192), (300, 28672, 512)])
@pytest.mark.parametrize("sides", [(76, 72), (112, 36)])
def test_on_a_partition(m, n, k, sides):
    part = ops.get_partition(0, *sides)
    args = operands(m, n, k)
    want = ops.int8_scaled_mm(*args)
    torch.cuda.synchronize()
    got, graphs = [], []
    for stream, sms in ((part.prefill_stream, part.prefill_sms), (part.decode_stream, part.decode_sms)):
        ops.set_sm_budget(sms)
        try:
            with torch.cuda.stream(stream):
                got.append(ops.int8_scaled_mm(*args))
                stream.synchronize()
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1], stream=stream):
                    got.append(ops.int8_scaled_mm(*args))
        finally:
            ops.set_sm_budget(0)
    for _ in range(3):  # both sides at once
        for graph, stream in zip(graphs, (part.prefill_stream, part.decode_stream)):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)
    ops.check_waits()
