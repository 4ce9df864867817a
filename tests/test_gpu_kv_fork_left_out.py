"""Children outside the page table are left out of a fork altogether: their page-table rows and the rows of their partial run."""
import pytest
import torch

from tests.test_gpu_kv_pages import _fork_case, _fork_want, _lists, _same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", [0, 1, 2, 3])
@pytest.mark.parametrize("child", [-1, "rows", 1 << 40, "parent"])
def test_children_outside_the_table(child, where):
    from semi_pd_b200 import ops
    bufs, table, rows = _fork_case([200, 77], 2, 128, "mha")
    good = rows[:where] + rows[where + 1:]
    want, want_table = _fork_want(bufs, table, good, 128)
    parent, _, n, base = rows[where]
    rows[where] = (parent, {"rows": table.shape[0], "parent": parent}.get(child, child), n, base)
    ops.kv_fork(ops.KVPlanes(bufs), table, *_lists(rows), 128)
    _same(bufs, want)
    assert torch.equal(table, want_table)
