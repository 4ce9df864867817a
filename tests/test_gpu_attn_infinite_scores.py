"""Decode attention where scores are not finite, against the formula: a key of score -inf weighs nothing, whole tiles of such keys
included; a NaN or +inf among a request's keys, or nothing but -inf, makes that request's output NaN (0 / 0) and no other's.

Column 0 of every query is 1, so that a key whose column 0 is -inf has the score -inf with every query; the bounds are those of
finite scores (test_gpu_attn_shared)."""
import pytest
import torch

from tests.test_gpu_attn_shared import D, call, device, make_case, reference

pytestmark = pytest.mark.gpu
INF = float("inf")


def _case(groups, alone, hq=8, hk=2, dtype=torch.bfloat16, seed=0):
    c = make_case(groups, alone, hq, hk, dtype, seed)
    c["q"].view(-1, hq, D)[:, :, 0] = 1
    return c


def _put(c, row, positions, value, column=0, head=None):
    slots = c["table"][c["rpi"][row]].long()[positions]
    if head is None:
        c["k"][slots, :, column] = value
    else:
        c["k"][slots, head, column] = value


def _check(c, out):
    want, tol = reference(c)
    got = out.cpu().double().view(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    assert bool((got[ok] - want[ok]).abs().le(tol[ok]).all())
    return want


def _both_ways(c):
    """With the shared keys read once, and by request."""
    from semi_pd_b200 import ops
    d = device(c)
    want = _check(c, call(c, d))
    _check(c, ops.attn_decode(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], c["hq"], c["hk"], D, c["scale"]))
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("first,last", [(512, 640), (512, 700), (600, 640), (512, 513), (640, 800), (0, 128), (0, 512), (64, 192), (0, 640)])
def test_tiles_of_minus_infinity(first, last, dtype):
    """Positions [first, last) of one member (shared ones: of all) weigh nothing; 512 are shared."""
    c = _case([(512, [300, 290, 1])], [400], dtype=dtype, seed=first + last)
    _put(c, 0, torch.arange(first, last), -INF)
    assert not _both_ways(c).isnan().any()


def test_one_head_of_minus_infinity():
    c = _case([(512, [300, 290, 1])], [400, 2000], seed=3)
    _put(c, 1, torch.arange(512, 640), -INF, head=1)
    _put(c, 3, torch.arange(0, 256), -INF, head=0)
    _put(c, 4, torch.arange(0, 1999), -INF, head=1)      # the last key alone is left
    assert not _both_ways(c).isnan().any()


def test_a_long_request_cut_over_many_sms():
    c = _case([], [20000, 20000], 8, 1, seed=4)
    _put(c, 0, torch.arange(0, 9000), -INF)
    _put(c, 0, torch.arange(12000, 20000), -INF)
    assert not _both_ways(c).isnan().any()


@pytest.mark.parametrize("value", [INF, float("nan")])
@pytest.mark.parametrize("at", [0, 130, 511, 512, 700])
def test_what_is_not_a_number_shows(at, value):
    c = _case([(512, [300, 290, 1])], [400], seed=at)
    _put(c, 1, torch.tensor([at]), value)
    want = _both_ways(c)
    assert want[1].isnan().all() and not want[3].isnan().any() and bool(want[0].isnan().any()) == (at < 512)


def test_nothing_but_minus_infinity():
    """0 / 0 for a request without any weight, 0 for one without any key."""
    c = _case([(512, [30, 200, 5])], [150, 0, 300], seed=6)
    _put(c, 3, torch.arange(150), -INF)
    want = _both_ways(c)
    assert want[3].isnan().all() and bool((want[4] == 0).all()) and int(want.isnan().any(-1).any(-1).sum()) == 1
    c = _case([(512, [30, 200, 5])], [150], seed=7)
    _put(c, 0, torch.arange(512), -INF)
    _put(c, 0, torch.arange(512, 542), -INF)
    want = _both_ways(c)
    assert want[0].isnan().all() and not want[1:].isnan().any()
