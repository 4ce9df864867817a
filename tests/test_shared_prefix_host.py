"""Forking and compacting on the host: which runs requests hold, share and give back; groups of neighbours; what the C ABI
refuses before any CUDA call."""
import ctypes as C

import numpy as np
import pytest
import torch

from semi_pd_b200 import _lib, ops
from semi_pd_b200.memory_pool import ReqToTokenPool, TokenToKVPoolAllocator

R = 16


def _alloc(runs=20):
    return TokenToKVPoolAllocator(runs * R, torch.float16, "cpu", None, run_len=R)


def _place(a, idx, n):
    out = a.alloc_extend([idx], [0], [n])
    assert out is not None and out.numel() == n
    return out


def test_children_share_whole_runs_and_get_a_partial_one():
    a = _alloc()
    slots = _place(a, 3, 40).numpy()     # two runs and eight tokens
    tails = a.fork_req(3, [5, 6])
    assert a.available_size() == (20 - 3 - 2) * R
    for child, tail in zip((5, 6), tails):
        mine = a.req_slots(child)
        assert (mine[:32] == slots[:32]).all()
        assert (mine[32:] == tail + np.arange(8)).all() and tail not in slots
        assert a.req_len(child) == 40
    assert tails[0] != tails[1]
    # every request goes on in a run of its own
    out = a.alloc_decode([3, 5, 6], [40, 40, 40]).numpy()
    assert out[0] == slots[-1] + 1 and (out[1:] == tails + 8).all()


def test_a_run_is_free_when_its_last_holder_lets_go():
    a = _alloc()
    _place(a, 0, 33)
    a.fork_req(0, [1, 2])
    assert a.free_req(0) == 33 and a.available_size() == (20 - 2 - 2) * R   # its own partial run alone
    a.free_req(1)
    assert a.available_size() == (20 - 2 - 1) * R
    a.free_req(2)
    assert a.available_size() == 20 * R and a.shared_prefix([0]) is None
    assert (a._held == 0).all() and (a._used == 0).all()
    _place(a, 0, 320)                    # all of it again
    assert a.available_size() == 0


def test_forks_of_forks():
    a = _alloc()
    _place(a, 0, 2 * R)
    a.fork_req(0, [1])
    assert a.available_size() == 18 * R  # whole runs only: nothing is copied
    a.alloc_decode([1], [2 * R])
    for i in range(1, R):
        a.alloc_decode([1], [2 * R + i])
    a.fork_req(1, [2, 3])                # three whole runs now
    assert a.shared_prefix([0, 1, 2, 3]) == ([0, 4], [2 * R])
    assert a.shared_prefix([1, 2, 3]) == ([0, 3], [3 * R])
    assert a.shared_prefix([0]) is None
    for r in (1, 0, 3):
        a.free_req(r)
    assert a.available_size() == (20 - 3) * R
    a.free_req(2)
    assert a.available_size() == 20 * R


def test_groups_are_neighbours():
    a = _alloc(40)
    _place(a, 0, 50)
    _place(a, 9, 70)
    _place(a, 4, 5)
    assert a.shared_prefix([0, 9, 4]) is None
    a.fork_req(0, [1, 2])
    a.fork_req(9, [8])
    assert a.shared_prefix([0, 1, 2, 4, 9, 8]) == ([0, 3, 4, 6], [48, 0, 64])
    assert a.shared_prefix([0, 4, 1, 2]) == ([0, 1, 2, 4], [0, 0, 48])
    assert a.shared_prefix([4, 0, 9]) is None
    a.fork_req(4, [5])                   # less than a run: nothing in common
    assert a.shared_prefix([4, 5]) is None


def test_nothing_is_taken_when_runs_do_not_suffice():
    a = _alloc(5)
    _place(a, 0, 40)
    assert a.fork_req(0, [1, 2, 3]) is None
    assert a.available_size() == 2 * R and (a._held[:3] == 1).all() and a.shared_prefix([0, 1]) is None
    assert a.rebuild_req(0, 40) is None and a.req_len(0) == 40


def test_bad_forks_are_refused():
    a = _alloc()
    _place(a, 0, 40)
    _place(a, 1, 4)
    for parent, children in ((7, [2]), (0, [0]), (0, [1]), (0, [2, 2])):
        with pytest.raises(RuntimeError):
            a.fork_req(parent, children)
    a.fork_req(0, [2])
    with pytest.raises(RuntimeError, match="several requests"):
        a.free(torch.from_numpy(a.req_slots(0)[:4].copy()))


def test_rebuild_gives_new_runs_and_keeps_the_old_until_released():
    a = _alloc()
    _place(a, 0, 40)
    a.fork_req(0, [1])
    before = a.req_slots(0)
    slots, old = a.rebuild_req(0, 20)
    assert len(slots) == 20 and not set(slots) & set(before) and a.req_len(0) == 20
    assert a.available_size() == (20 - 4 - 2) * R
    a.release_runs(old)
    assert a.available_size() == (20 - 3 - 2) * R   # the two shared runs are still the other request's
    assert a.req_len(1) == 40
    for n in (0, 21):
        with pytest.raises(RuntimeError, match="cannot keep"):
            a.rebuild_req(0, n)
    a.free_req(0)
    a.free_req(1)
    assert a.available_size() == 20 * R and (a._used == 0).all()


def test_what_the_allocator_did_before_stays():
    a = _alloc()
    ids = a.alloc(20)
    a.free(ids[:4])
    a.free(ids[4:])
    assert a.available_size() == 20 * R and (a._held == 0).all()
    with pytest.raises(RuntimeError, match="twice"):
        a.free(ids[:1])


def test_planes_are_grouped_by_shape_and_stride():
    slab = torch.zeros(6, 10, 2, 8, dtype=torch.float16)
    p = ops.KVPlanes(list(slab))
    assert [n for _, n in p.calls] == [1] and p.token_bytes == 6 * 32
    assert p._arrays[0][0].planes == 6 and p._arrays[0][0].plane_stride == 320
    p = ops.KVPlanes([slab[0], torch.zeros(10, 4), None, slab[0], slab[3], slab[5]])
    assert [s.planes for s in p._arrays[0]] == [1, 1, 2]
    p = ops.KVPlanes([torch.zeros(3, 1 + i % 2) for i in range(130)])
    assert sum(n for _, n in p.calls) >= 65 and len(p.calls) >= 2
    with pytest.raises(RuntimeError, match="no buffers"):
        ops.KVPlanes([None])
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.KVPlanes([slab[0][:, :1]])


def test_ops_need_cuda_tensors():
    planes = ops.KVPlanes([torch.zeros(8, 2)])
    i = torch.tensor([1])
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.kv_copy(planes, i, i)


def test_c_abi_refuses_before_any_cuda_call():
    lib = _lib.lib
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    good = _lib.KVPlaneSet(p, 64, 4, 16, 2)
    at = C.addressof(good)
    assert lib.spd_kv_copy(at, 0, p, p, 1, None) == -1
    assert lib.spd_kv_copy(at, 65, p, p, 1, None) == -1
    assert lib.spd_kv_copy(None, 1, p, p, 1, None) == -1
    assert lib.spd_kv_copy(at, 1, None, p, 1, None) == -1
    assert lib.spd_kv_copy(at, 1, p, p, -1, None) == -1
    assert lib.spd_kv_copy(at, 1, None, None, 0, None) == 0
    for bad, code in ((_lib.KVPlaneSet(None, 64, 4, 16, 2), -1), (_lib.KVPlaneSet(p, 64, 0, 16, 2), -1),
                      (_lib.KVPlaneSet(p, 64, 4, 0, 2), -1), (_lib.KVPlaneSet(p, 64, 4, 16, 0), -1),
                      (_lib.KVPlaneSet(p, 64, 4, 3, 2), -2), (_lib.KVPlaneSet(p + 1, 64, 4, 16, 2), -2),
                      (_lib.KVPlaneSet(p, 64, 4, 16, 70000), -3)):
        assert lib.spd_kv_copy(C.addressof(bad), 1, p, p, 1, None) == code
    assert lib.spd_kv_fork(at, 1, p, 8, 2, 9, p, p, p, p, 1, 128, None) == -1      # row shorter than its tokens
    assert lib.spd_kv_fork(at, 1, p, 8, 2, 8, p, p, p, p, 1, 0, None) == -1
    assert lib.spd_kv_fork(at, 1, p, 8, 2, 8, p, p, p, p, 70000, 128, None) == -3
    assert lib.spd_kv_compact(at, 1, p, 8, 2, 8, p, None, None, p, p, 1, 4, 1, None) == -1
    assert lib.spd_kv_compact(at, 1, p, 8, 2, 8, None, None, None, None, None, 0, 0, 1, None) == 0

    def shared(batch=4, groups=1, most=512, slots=64, hq=8, hk=2, d=128, stride=1024, scale=0.1, dtype=0, ws=p, ws_bytes=64,
               indptr=p, lens=p):
        return lib.spd_attn_decode_shared(p, p, p, p, p, p, p, indptr, lens, batch, groups, most, slots, hq, hk, d, stride, stride,
                                          8, scale, dtype, ws, ws_bytes, 0, None)
    assert shared(hq=9, hk=2) == -3 and shared(hq=18, hk=2) == -3
    assert shared(d=64) == -3 and shared(d=96) == -3
    assert shared(stride=1023) == -2
    assert shared(batch=-1) == -1 and shared(groups=-1) == -1 and shared(most=-1) == -1 and shared(slots=0) == -1
    assert shared(indptr=None) == -1 and shared(lens=None) == -1
    assert shared(ws=None) == -4 and shared() == -4
    assert shared(batch=0) == 0
    assert lib.spd_attn_decode_shared_workspace_bytes(0, 32, 8, 128) == 0
    assert lib.spd_attn_decode_shared_workspace_bytes(8, 32, 8, 64) == 0


@pytest.mark.parametrize("args,pays", [
    ((64, 1, 8192, 32, 8, 128, 148), 1),     # a batch behind one long prompt
    ((256, 1, 32768, 64, 8, 128, 148), 1),
    ((2, 1, 300, 32, 8, 128, 148), 0),       # too little to share
    ((64, 1, 256, 32, 8, 128, 148), 0),
    ((64, 32, 2048, 32, 8, 128, 148), 0),    # pairs of requests
    ((64, 32, 8192, 32, 8, 128, 148), 1),
    ((2, 1, 4096, 16, 2, 128, 148), 1),      # few requests, which would be cut over many SMs each
    ((1, 1, 8192, 32, 8, 128, 148), 0), ((64, 0, 8192, 32, 8, 128, 148), 0), ((64, 1, 127, 32, 8, 128, 148), 0),
    ((1025, 1, 8192, 32, 8, 128, 148), 0), ((1024, 257, 8192, 32, 8, 128, 148), 0), ((64, 1, 8192, 32, 8, 64, 148), 0)])
def test_when_sharing_pays(args, pays):
    assert _lib.lib.spd_attn_decode_shared_pays(*args) == pays
    assert (_lib.lib.spd_attn_decode_shared_saves(*args) > 0) == bool(pays)


def test_a_graph_is_given_up_only_for_more_than_it_saves():
    from semi_pd_b200 import ops
    from semi_pd_b200.attention_backend import SpdAttnBackend
    from semi_pd_b200.forward_batch_info import SharedPrefix
    backend = SpdAttnBackend.__new__(SpdAttnBackend)
    backend.impl, backend.is_mla, backend.num_q_heads, backend.num_kv_heads, backend.head_dim = "tc", False, 32, 8, 128
    shared = lambda n: SharedPrefix(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), n)  # noqa: E731
    few = next(n for n in range(128, 1 << 16, 128) if ops.attn_shared_pays(64, 1, n, 32, 8, 128))
    assert 0 < ops.attn_shared_saves(64, 1, few, 32, 8, 128) <= SpdAttnBackend.GRAPH_SAVES < ops.attn_shared_saves(64, 1, 8192, 32, 8, 128)
    for most, want in ((0, True), (63, True), (64, False)):
        backend.graph_max_bs = most
        assert backend.shares_prefix(64, shared(few)) is want
        assert backend.shares_prefix(64, shared(8192))


class _Event:
    def __init__(self):
        self.done, self.waited = False, False

    def query(self):
        return self.done

    def synchronize(self):
        self.done = self.waited = True


def test_what_a_copy_reads_is_free_when_it_has_run():
    """Runs and request slots that come back while a copy may still read them are not handed out before it has run."""
    pool = ReqToTokenPool(4, 64, "cpu")
    alloc = TokenToKVPoolAllocator(6 * 8, torch.float32, "cpu", None, run_len=8)
    (a,) = pool.alloc(1)
    alloc.alloc_extend([a], [0], [20])          # three of six runs
    held = set(alloc._req_runs[a])
    event = _Event()
    alloc._free_runs.copies.append(event)
    pool._free.copies.append(event)
    alloc.free_req(a)
    pool.free(a)
    assert alloc.available_size() == 48 and pool.available_size() == 4
    b = pool.alloc(3)
    assert a not in b
    alloc.alloc_extend(b[:1], [0], [24])        # the other three
    assert not held & set(alloc._req_runs[b[0]]) and not event.waited
    assert alloc.can_alloc_decode([8]) and event.waited   # a fourth one waits for the copy
    alloc.alloc_extend(b[1:2], [0], [24])
    assert set(alloc._req_runs[b[1]]) == held and alloc.available_size() == 0
    assert pool.alloc(1) == [a]
    alloc.free_req(b[0])                        # no copy runs any more
    assert alloc.alloc_extend([a], [0], [24]) is not None
    alloc.clear()
    pool.clear()
    assert alloc.available_size() == 48 and pool.available_size() == 4
    event = _Event()
    alloc._free_runs.copies.append(event)
    alloc.alloc_extend([a], [0], [20])
    alloc.free_req(a)
    event.done = True
    assert alloc.alloc_extend([a], [0], [48]) is not None and not event.waited
