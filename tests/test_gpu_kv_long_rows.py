"""Rows of a megabyte and more (a recurrent state of a request is one row): copied bit for bit, and forked through the pools."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

# elements of a row: 1 MB, one vector more, 2 MB, 4 MB and some odd bytes; and a mixture with short ones
ROWS = {
    "1 MB": [(1 << 18, torch.float32)],
    "1 MB + 16": [((1 << 18) + 4, torch.float32)],
    "2 MB": [(1 << 19, torch.float32)] * 3,
    "odd": [((1 << 21) + 12345, torch.float16)],
    "mixed": [(1 << 19, torch.float32), (8, torch.float16), (100003, torch.bfloat16), (1 << 20, torch.float32), (24, torch.float32)],
    "just over a part": [(8192 + 4, torch.float32), (8192, torch.float32), (8192 - 4, torch.float32)],
}


@pytest.mark.parametrize("kind", list(ROWS))
@pytest.mark.parametrize("n", [1, 3])
def test_copy(kind, n):
    from semi_pd_b200 import ops
    slots = 2 * n + 3
    g = torch.Generator(device=DEV).manual_seed(n)
    bufs = [torch.randn(slots, size, generator=g, device=DEV).to(dtype) for size, dtype in ROWS[kind]]
    perm = torch.randperm(slots, generator=torch.Generator().manual_seed(n))
    src, dst = perm[:n].to(DEV), perm[n:2 * n].to(DEV)
    src[-1:] = src[:1]      # one source twice
    want = [b.clone() for b in bufs]
    for w in want:
        w[dst] = w[src]
    ops.kv_copy(ops.KVPlanes(bufs), src, dst)
    for b, w in zip(bufs, want):
        assert torch.equal(b, w)


@pytest.mark.parametrize("kind", ["1 MB + 16", "odd", "mixed"])
def test_fork_and_compact(kind):
    """Pools of such rows: the partial run of a fork, and what a compaction keeps."""
    from semi_pd_b200 import ops
    run, slots = 4, 25
    g = torch.Generator(device=DEV).manual_seed(3)
    bufs = [torch.randn(slots, size, generator=g, device=DEV).to(dtype) for size, dtype in ROWS[kind]]
    planes = ops.KVPlanes(bufs)
    table = torch.zeros(4, 12, dtype=torch.int32, device=DEV)
    table[1, :7] = torch.tensor([5, 6, 7, 8, 13, 14, 15], dtype=torch.int32, device=DEV)
    i64 = lambda *x: torch.tensor(x, device=DEV)  # noqa: E731
    want = [b.clone() for b in bufs]
    for w in want:
        w[17:20] = w[13:16]
        w[21:24] = w[13:16]
        w[1:4] = w[i64(5, 8, 15)]
    ops.kv_fork(planes, table, i64(1, 1), i64(0, 3), i64(7, 7), i64(17, 21), run)
    ops.kv_compact(planes, table, i64(1), i64(2), i64(0, 3, 6), i64(0, 3), i64(1, 2, 3))
    for b, w in zip(bufs, want):
        assert torch.equal(b, w)
    assert table[0, :7].tolist() == [5, 6, 7, 8, 17, 18, 19] and table[3, :7].tolist() == [5, 6, 7, 8, 21, 22, 23]
    assert table[2, :3].tolist() == [1, 2, 3]


@pytest.mark.parametrize("heads,dim,v_dim", [(32, 128, 128), (64, 64, 128), (5, 256, 259)])
def test_fork_of_large_states(heads, dim, v_dim):
    """States of 2 MB a request, and of an odd number of floats above 1 MB."""
    from semi_pd_b200.memory_pool import (HybridTokenToKVPool, RecurrentStatePool, ReqToTokenPool, TokenToKVPoolAllocator,
                                          fork_request)
    reqs, run_len = 6, 128
    states = RecurrentStatePool(reqs, [(heads, dim, v_dim), None, (heads, dim, v_dim)], DEV)
    pool = HybridTokenToKVPool(8 * run_len, 1, torch.bfloat16, [None, (2, 64, 64), None], DEV, state_pool=states)
    table, alloc = ReqToTokenPool(reqs, 1024, DEV), TokenToKVPoolAllocator(8 * run_len, torch.bfloat16, DEV, pool)
    for t in states.state:
        if t is not None:
            t.normal_()
    for b in pool.planes.buffers:
        b.normal_()
    (parent,) = table.alloc(1)
    table.req_to_token[parent, :200] = alloc.alloc_extend([parent], [0], [200]).int()
    before = [t.clone() for t in states.state if t is not None]
    children = fork_request(pool, table, alloc, parent, 3)
    for t, was in zip([t for t in states.state if t is not None], before):
        for r in range(t.shape[0]):
            assert torch.equal(t[r], was[parent if r in children else r])
    slots = table.req_to_token[parent, :200].long()
    for c in children:
        for b in pool.planes.buffers:
            assert torch.equal(b[table.req_to_token[c, :200].long()], b[slots])
