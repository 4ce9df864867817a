"""A fork or a compaction whose copy is refused leaves requests, runs and slots as they were."""
import pytest
import torch

from semi_pd_b200 import memory_pool, ops
from semi_pd_b200.memory_pool import ReqToTokenPool, TokenToKVPoolAllocator, compact_request, fork_request

R = 16


class _Pool:
    """What fork_request and compact_request ask of a pool; its second copy is refused."""
    planes = None

    def buffers(self):
        return [torch.zeros(4, 1)]

    def fork_rows(self, *args):
        raise RuntimeError("refused behind the first copy")

    def compact_refusal(self):
        return None


def _setup(tokens=40, runs=20, reqs=6):
    table = ReqToTokenPool(reqs, 256, "cpu")
    alloc = TokenToKVPoolAllocator(runs * R, torch.float16, "cpu", None, run_len=R)
    (req,) = table.alloc(1)
    alloc.alloc_extend([req], [0], [tokens])
    return table, alloc, req


def _counts(table, alloc):
    return (table.available_size(), sorted(table._live), alloc.available_size(), alloc._held.tolist(), alloc._used.tolist(),
            {k: list(v) for k, v in alloc._req_runs.items()}, dict(alloc._req_len))


def _refuse(*args, **kw):
    raise RuntimeError("refused")


@pytest.mark.parametrize("where", ["first copy", "second copy"])
@pytest.mark.parametrize("tokens", [40, 2 * R, 3])
def test_fork(monkeypatch, where, tokens):
    table, alloc, parent = _setup(tokens)
    before = _counts(table, alloc)
    monkeypatch.setattr(ops, "kv_fork", _refuse if where == "first copy" else lambda *a: None)
    with pytest.raises(RuntimeError, match="refused"):
        fork_request(_Pool(), table, alloc, parent, 3)
    assert _counts(table, alloc) == before
    alloc.free_req(parent)              # the parent's runs are its own again
    assert alloc.available_size() == 20 * R and (alloc._held == 0).all() and (alloc._used == 0).all()


def test_what_was_launched_is_waited_for(monkeypatch):
    """The runs and slots of a refused fork are free when the copies launched before have run."""
    table, alloc, parent = _setup(40, runs=5, reqs=3)

    class Event:
        done = False

        def query(self):
            return self.done

        def synchronize(self):
            self.done = True

    events = []

    def copying(self):
        events.append(Event())
        self.copies.append(events[-1])

    monkeypatch.setattr(memory_pool._FreeList, "copying", copying)
    monkeypatch.setattr(ops, "kv_fork", lambda *a: None)
    with pytest.raises(RuntimeError, match="refused"):
        fork_request(_Pool(), table, alloc, parent, 2)
    assert len(events) == 2 and table.available_size() == 2 and alloc.available_size() == 2 * R
    assert table.alloc(2) is not None and alloc.alloc_extend([5], [0], [2 * R]) is not None
    assert all(e.done for e in events)


def test_compact(monkeypatch):
    table, alloc, req = _setup(40)
    alloc.fork_req(req, [5])
    before, slots = _counts(table, alloc), alloc.req_slots(req)
    monkeypatch.setattr(ops, "kv_compact", _refuse)
    with pytest.raises(RuntimeError, match="refused"):
        compact_request(_Pool(), table, alloc, req, [0, 1, 30])
    assert _counts(table, alloc) == before and (alloc.req_slots(req) == slots).all()
    monkeypatch.setattr(ops, "kv_compact", lambda *a: None)
    assert compact_request(_Pool(), table, alloc, req, [0, 1, 30]) and alloc.req_len(req) == 3
    alloc.free_req(req)
    alloc.free_req(5)
    assert alloc.available_size() == 20 * R and (alloc._held == 0).all() and (alloc._used == 0).all()


def test_a_model_without_cached_tokens_forks_its_states(monkeypatch):
    """All layers recurrent: there are no rows of tokens to copy, the states of the request slots are."""
    states = memory_pool.RecurrentStatePool(6, [(2, 4, 4), (1, 4, 8)], "cpu")
    pool = memory_pool.HybridTokenToKVPool(20 * R, 1, torch.float32, [None, None], "cpu", state_pool=states, run_len=R)
    table, alloc, parent = _setup(40)
    copied = []
    monkeypatch.setattr(ops, "kv_fork", _refuse)
    monkeypatch.setattr(ops, "kv_copy", lambda planes, src, dst: copied.append((planes is states.planes, src.tolist(), dst.tolist())))
    children = fork_request(pool, table, alloc, parent, 2)
    assert len(children) == 2 and copied == [(True, [parent] * 2, children)]
