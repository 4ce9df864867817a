"""attn_decode_shared where its plan gives a thread several batch rows, and at the rows and groups that it holds at most: unequal own
lengths, empty members, few SMs.  The counts passed make the call take the kernel that shares, which each test asserts."""
import pytest
import torch

from tests.test_gpu_attn_shared import D, check, device, make_case

pytestmark = pytest.mark.gpu
HQ, HK = 4, 2


def _run(c, sms=0, hq=HQ, hk=HK):
    from semi_pd_b200 import ops
    d = device(c)
    tokens = ops.SharedTokens(1 << 20, 1 << 24, 0, 1 << 20)
    ops.set_sm_budget(sms)
    try:
        assert ops.attn_shared_pays(len(c["lens"]), len(c["shared"]), 0, hq, hk, D, tokens)
        return ops.attn_decode_shared(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], 0, hq, hk, D,
                                      c["scale"], shared_tokens=tokens)
    finally:
        ops.set_sm_budget(0)


def _own(i):
    return (0, 1, 127, 128, 129, 40, 200, 3)[i * 5 % 8]


@pytest.mark.parametrize("sms", [0, 1, 7])
@pytest.mark.parametrize("rows", [384, 385, 768, 769, 1023, 1024])
def test_rows(rows, sms):
    """One large group, a few small ones, and requests of no group; every seventh request is empty."""
    big = rows - 60
    c = make_case([(256, [_own(i) for i in range(big)]), (130, [3, 200]), (0, [90]), (384, [_own(i + 1) for i in range(37)])],
                  [_own(i) for i in range(20)], HQ, HK, torch.bfloat16, seed=rows)
    assert len(c["lens"]) == rows
    c["lens"] = [0 if i % 7 == 3 else n for i, n in enumerate(c["lens"])]
    check(c, _run(c, sms))


@pytest.mark.parametrize("sms", [0, 5])
@pytest.mark.parametrize("members", [2, 4])
@pytest.mark.parametrize("groups", [255, 256])
def test_groups(groups, members, sms):
    c = make_case([(128 * (1 + g % 3) - (g % 2), [_own(g + i) for i in range(members)]) for g in range(groups)], [], HQ, HK,
                  torch.float16, seed=groups + members)
    if members == 2:    # some groups have one member left, some none
        c["lens"] = [0 if i % 11 in (4, 5) else n for i, n in enumerate(c["lens"])]
    check(c, _run(c, sms))


def test_many_members_behind_many_tiles():
    """All 1024 rows one group, 32 pairs of query tiles, with a token or two of their own."""
    c = make_case([(1024, [1 + i % 2 for i in range(1024)])], [], 8, 1, torch.bfloat16, seed=1)
    check(c, _run(c, 0, 8, 1))
