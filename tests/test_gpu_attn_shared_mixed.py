"""Groups and requests of no group in one batch, with the counts that the host knows: both ways give the same attention, and the
counts alone decide which one is taken."""
import pytest
import torch

from tests.test_gpu_attn_shared import D, check, device, make_case

pytestmark = pytest.mark.gpu


def _call(c, d, tokens):
    from semi_pd_b200 import ops
    return ops.attn_decode_shared(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], 0, c["hq"],
                                  c["hk"], D, c["scale"], shared_tokens=tokens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups,alone,lists", [
    ([(1000, [5, 40, 130])], [300, 1, 2000], ([0, 3], [1000])),
    ([(384, [3, 9]), (0, [5]), (0, [700]), (1000, [1, 2, 3, 4])], [33], ([0, 2, 4, 8], [384, 0, 1000])),
    ([(0, [50]), (0, [5]), (640, [7] * 20)], [], ([2, 22], [640])),
    ([(256, [1, 2])] * 3 + [(0, [9])] * 40 + [(2000, [1, 300])], [128] * 60, ([0, 2, 4, 6, 46, 48], [256, 256, 256, 0, 2000]))])
def test_mixed_batches(groups, alone, lists, dtype):
    from semi_pd_b200 import ops
    c = make_case(groups, alone, 16, 4, dtype, seed=len(groups))
    c["indptr"], c["shared"] = lists
    d = device(c)
    want = ops.attn_decode(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], 16, 4, D, c["scale"])
    shared = _call(c, d, ops.SharedTokens(1 << 20, 1 << 24, 0, 1 << 20))
    check(c, shared)
    known = ops.attn_shared_tokens(*lists, c["lens"])
    assert known.group == sum(n // 128 * 128 for n in lists[1]) and known.longest == max(c["lens"])
    check(c, _call(c, d, known))
    alone_way = _call(c, d, ops.SharedTokens(0, 0, 0, 0))
    check(c, alone_way)
    assert not torch.equal(shared, alone_way) and bool((alone_way.float() - want.float()).abs().max() < 0.05)


def test_refused_counts():
    from semi_pd_b200 import ops
    c = make_case([(300, [20, 21])], [], 8, 2)
    d = device(c)
    for bad in ((-1, 0, 0, 0), (0, -1, 0, 0), (0, 0, -1, 0), (0, 0, 0, -1)):
        with pytest.raises(RuntimeError, match="token counts"):
            _call(c, d, ops.SharedTokens(*bad))


def test_refused_workspaces():
    from semi_pd_b200 import ops
    c = make_case([(300, [20, 21])], [], 8, 2)
    d = device(c)
    need = ops.new_attn_shared_workspace(torch.device("cuda", 0), 2, 8, 2, D).numel()
    wide = torch.zeros(2 * need + 16, dtype=torch.uint8, device="cuda")
    for bad, match in ((wide[::2], "contiguous"), (wide[4:], "aligned"), (wide[:need - 16], "too small")):
        with pytest.raises(RuntimeError, match=match):
            ops.attn_decode_shared(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], 300, 8, 2, D, 0.1,
                                   workspace=bad)
    # counted in bytes
    ops.attn_decode_shared(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], 300, 8, 2, D, 0.1,
                           workspace=torch.zeros(need // 4 + 4, dtype=torch.float32, device="cuda"))
