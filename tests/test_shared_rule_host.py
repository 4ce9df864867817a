"""Whether decode attention reads shared prefixes once, by the groups that a batch has: unequal ones, and requests of no group
beside them.  (Values in brackets: us saved a layer as measured, by request less shared.)"""
import pytest
import torch

from semi_pd_b200 import _lib, ops
from semi_pd_b200.attention_backend import SpdAttnBackend
from semi_pd_b200.forward_batch_info import SharedPrefix
from semi_pd_b200.memory_pool import ReqToTokenPool, TokenToKVPoolAllocator
from semi_pd_b200.schedule_batch import Req, SamplingParams, ScheduleBatch, _joined_alone

RUN = 128


def _saves(groups, alone, hq=32, hk=8, own=130):
    """groups: (members, shared tokens); alone: lengths of the requests of no group."""
    indptr, lens, seq = [0], [], []
    for members, shared in groups:
        indptr.append(indptr[-1] + members)
        lens.append(shared)
        seq += [shared + own] * members
    seq += alone
    return _lib.lib.spd_attn_decode_shared_saves_tokens(len(seq), len(lens), *ops.attn_shared_tokens(indptr, lens, seq), hq, hk, 128, 148)


@pytest.mark.parametrize("n,measured", [(0, 145), (64, 133), (100, 131), (400, 117)])
def test_unrelated_requests_do_not_end_sharing(n, measured):
    assert abs(_saves([(64, 8192)], [500] * n) - measured) < 30


def test_a_few_continuations_beside_others():
    assert 10 < _saves([(16, 8192)], [500] * 24) < 50     # (27)
    assert _saves([(64, 8192)], [4000] * 100) > 50        # (102)
    assert _saves([(8, 4096)], [2000] * 100) == 0         # (-27)
    assert _saves([(12, 2048), (12, 512)], [700] * 30) <= SpdAttnBackend.GRAPH_SAVES  # (-10)
    assert _saves([(64, 8192)], [1] * 900) > 50


def test_one_long_pair_does_not_count_for_all():
    assert 20 < _saves([(126, 128), (2, 16384)], []) < 120           # (55)
    assert 100 < _saves([(2, 128)] * 63 + [(2, 65536)], []) < 400    # (244)
    assert _saves([(2, 128)] * 63 + [(2, 1024)], []) == 0
    assert _saves([(64, 128)], []) == 0 and _saves([], [300] * 9) == 0


@pytest.mark.parametrize("members,groups,shared", [(64, 1, 8192), (2, 32, 4096), (8, 4, 1024), (2, 1, 4096), (16, 1, 256), (3, 60, 640)])
@pytest.mark.parametrize("hq,hk", [(32, 8), (32, 32), (16, 2)])
def test_equal_groups_are_judged_as_before(members, groups, shared, hq, hk):
    batch = members * groups
    known = _lib.lib.spd_attn_decode_shared_saves_tokens(batch, groups, groups * shared, batch * shared, 64 * batch, shared, hq, hk, 128, 148)
    assert known == _lib.lib.spd_attn_decode_shared_saves(batch, groups, shared, hq, hk, 128, 148)
    assert abs(known - _saves([(members, shared)] * groups, [], hq, hk, 64)) <= 1 + known // 20


def test_counts_that_make_no_sense():
    f = _lib.lib.spd_attn_decode_shared_saves_tokens
    assert f(64, 1, 8192, 64 * 8192, 0, 9000, 32, 8, 128, 148) > 0
    for bad in ((64, 0, 8192, 64 * 8192), (64, 257, 8192, 64 * 8192), (1, 1, 8192, 8192), (1025, 1, 8192, 64 * 8192), (64, 1, 127, 64 * 127),
                (64, 1, 8192, 100)):
        assert f(*bad, 0, 9000, 32, 8, 128, 148) == 0
    assert f(64, 1, 8192, 64 * 8192, 0, 9000, 32, 8, 64, 148) == 0


@pytest.mark.parametrize("indptr,lens,want", [
    ([0, 3, 4, 6], [48, 0, 64], ([0, 3, 4, 6], [48, 0, 64])),
    ([0, 1, 2, 4], [0, 0, 48], ([2, 4], [48])),
    ([0, 2, 3, 4, 5], [32, 0, 0, 0], ([0, 2], [32])),
    ([0, 1, 3, 4, 5, 6, 9, 10], [0, 16, 0, 0, 0, 32, 0], ([1, 3, 6, 9], [16, 0, 32])),
    ([0, 2, 4], [16, 16], ([0, 2, 4], [16, 16]))])
def test_requests_of_no_group_are_joined(indptr, lens, want):
    assert _joined_alone(indptr, lens) == want


def test_a_batch_of_both(monkeypatch):
    """64 continuations in two places among 500 unrelated requests: four entries in the lists, and what they save."""
    monkeypatch.setattr(ScheduleBatch, "_h2d", lambda self, values, dtype: torch.tensor(values, dtype=dtype))
    alloc = TokenToKVPoolAllocator(2000 * RUN, torch.float16, "cpu", None, run_len=RUN)
    batch = ScheduleBatch.init_new([], ReqToTokenPool(600, 16384, "cpu"), alloc, "cpu")
    order, lens = [], []

    def place(n, count=1):
        for _ in range(count):
            idx = len(order)
            order.append(idx)
            lens.append(n)
            alloc.alloc_extend([idx], [0], [n])

    def forks(n, prefix):
        first = len(order)
        place(prefix)
        kids = list(range(first + 1, first + n))
        alloc.fork_req(first, kids)
        order.extend(kids)
        lens.extend([prefix] * (n - 1))

    place(200, 100)
    forks(40, 8200)
    place(300, 300)
    forks(24, 4100)
    place(100, 100)
    for idx in order:
        req = Req(str(idx), [1], SamplingParams())
        req.req_pool_idx = idx
        batch.reqs.append(req)
    batch.seq_lens_host = lens
    shared = batch._shared_prefix()
    assert shared.group_indptr.tolist() == [100, 140, 440, 464] and shared.shared_lens.tolist() == [8192, 0, 4096]
    assert shared.tokens == (8192 + 4096, 40 * 8192 + 24 * 4096, sum(lens) - 40 * 8192 - 24 * 4096, 8200)
    backend = SpdAttnBackend.__new__(SpdAttnBackend)
    backend.impl, backend.is_mla, backend.num_q_heads, backend.num_kv_heads, backend.head_dim = "tc", False, 32, 8, 128
    backend.graph_max_bs = 1024
    assert backend.shares_prefix(len(order), shared)
    # the lists are kept, the counts follow the lengths
    batch.seq_lens_host = [n + 1 for n in lens]
    again = batch._shared_prefix()
    assert again.group_indptr is shared.group_indptr and again.tokens.own == shared.tokens.own + len(order)
    assert again.tokens.longest == 8201


def test_the_lists_say_more_than_the_longest_prefix():
    """What the two forms answer for 64 continuations beside 100 unrelated requests."""
    lists = dict(batch_size=164)
    backend = SpdAttnBackend.__new__(SpdAttnBackend)
    backend.impl, backend.is_mla, backend.num_q_heads, backend.num_kv_heads, backend.head_dim = "tc", False, 32, 8, 128
    backend.graph_max_bs = 0
    plain = SharedPrefix(torch.zeros(102, dtype=torch.int32), torch.zeros(101, dtype=torch.int64), 8192)
    known = SharedPrefix(plain.group_indptr[:2], plain.shared_lens[:1], 8192, ops.SharedTokens(8192, 64 * 8192, 60000, 8400))
    assert not backend.shares_prefix(shared=plain, **lists) and backend.shares_prefix(shared=known, **lists)


def test_a_backend_without_such_a_form_reads_by_request():
    from semi_pd_b200.attention_backend import AttentionBackend

    class Plain(AttentionBackend):
        def init_forward_metadata(self, forward_batch):
            pass

    assert Plain().shares_prefix(64, SharedPrefix(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), 8192)) is False
