"""A compaction reads and writes its request's page-table row when its copy runs: the slot is handed out again only then."""
import pytest
import torch

from tests.test_gpu_fork import DEV, _place, _pools, _rows

pytestmark = pytest.mark.gpu


def test_the_slot_of_a_compacted_request_waits_for_the_copy():
    from semi_pd_b200.memory_pool import compact_request
    pool, table, alloc = _pools("mha", runs=12, reqs=3)
    req = _place(table, alloc, 500)
    warm = _place(table, alloc, 10)               # (a kernel's first launch waits for the device)
    assert compact_request(pool, table, alloc, warm, [1, 2])
    torch.cuda.synchronize()
    alloc.free_req(warm)
    table.free(warm)
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        torch.cuda._sleep(200_000_000)            # about 0.1 s
        assert compact_request(pool, table, alloc, req, list(range(3, 500, 2)))
        alloc.free_req(req)
        table.free(req)
    with torch.cuda.stream(other):                # the slot's next request
        slots = table.alloc(3)
        assert req in slots
        loc = alloc.alloc_extend([req], [0], [600])
        table.req_to_token[req, :600] = loc.int()
        for b in pool.planes.buffers:
            b[loc] = 3
    torch.cuda.synchronize()
    assert table.req_to_token[req, :600].tolist() == loc.tolist()
    assert all(bool((r == 3).all()) for r in _rows(pool, table.req_to_token, req, 600))
