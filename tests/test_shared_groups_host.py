"""How a batch is cut into groups that share a prefix: by what sharing saves, found again only when it may have changed."""
import itertools
import random
import time

import pytest
import torch

from semi_pd_b200 import memory_pool
from semi_pd_b200.memory_pool import TokenToKVPoolAllocator, _best_groups, _common_runs

R = 16


def _alloc(runs=4000):
    return TokenToKVPoolAllocator(runs * R, torch.float16, "cpu", None, run_len=R)


def _grow(a, idx, runs):
    """A request goes on for whole runs."""
    a.alloc_extend([idx], [a.req_len(idx)], [a.req_len(idx) + runs * R])


def test_a_shallow_relative_does_not_end_deep_sharing():
    a = _alloc()
    a.alloc_extend([0], [0], [R])
    a.fork_req(0, [9])
    _grow(a, 0, 10)
    a.fork_req(0, [1, 2, 3])
    assert a.shared_prefix([0, 1, 2, 3]) == ([0, 4], [11 * R])
    assert a.shared_prefix([0, 1, 2, 3, 9]) == ([0, 4, 5], [11 * R, 0])
    assert a.shared_prefix([9, 0, 1, 2, 3]) == ([0, 1, 5], [0, 11 * R])
    assert a.shared_prefix([0, 9]) == ([0, 2], [R])


def test_two_branches_behind_one_common_run():
    a = _alloc()
    a.alloc_extend([0], [0], [R])
    a.fork_req(0, [100])
    for root, first in ((0, 1), (100, 101)):
        _grow(a, root, 63)
        a.fork_req(root, list(range(first, first + 31)))
    rows = list(range(32)) + list(range(100, 132))
    assert a.shared_prefix(rows) == ([0, 32, 64], [64 * R, 64 * R])
    mixed = rows[::2] + rows[1::2]
    assert a.shared_prefix(mixed) == ([0, 16, 32, 48, 64], [64 * R] * 4)


def _value(n, shared):
    return (7 * n - 12) * shared if n > 1 else 0


def _exhaustive(common, start, end):
    """The best sum over all cuts of the rows."""
    top = 0
    for cuts in itertools.product((False, True), repeat=end - start - 1):
        at = [start] + [start + 1 + i for i, c in enumerate(cuts) if c] + [end]
        top = max(top, sum(_value(q - p, min(common[p + 1:q], default=0)) for p, q in zip(at, at[1:])))
    return top


@pytest.mark.parametrize("seed", range(60))
def test_the_cut_that_saves_most(seed):
    rng = random.Random(seed)
    n = rng.randint(1, 11)
    common = [0, 0] + [rng.choice([1, 1, 2, 3, 3, 8, 40]) for _ in range(n - 1)] + [0, 5]
    if seed % 3 == 0:       # stretches of equals
        common = [0, 0] + sorted(common[2:n + 1]) + [0, 5]
    start, end = 1, 1 + n
    groups = _best_groups(common, start, end)
    at = [start] + [e for e, _ in groups]
    assert at[-1] == end and all(p < q for p, q in zip(at, at[1:]))
    for p, (q, shared) in zip(at, groups):
        assert shared == min(common[p + 1:q], default=0)
    assert sum(_value(q - p, s) for p, (q, s) in zip(at, groups)) == _exhaustive(common, start, end)


def test_common_runs():
    for n, m, k in ((0, 3, 0), (5, 5, 5), (5, 9, 5), (7, 7, 0), (7, 7, 6), (100, 90, 31)):
        a = list(range(k)) + [1000 + i for i in range(n - k)]
        b = list(range(k)) + [5000 + i for i in range(m - k)]
        assert _common_runs(a, b) == k == _common_runs(b, a)


def test_groups_are_found_again_only_when_they_may_have_changed(monkeypatch):
    a = _alloc()
    found = []
    real = TokenToKVPoolAllocator._find_groups
    monkeypatch.setattr(TokenToKVPoolAllocator, "_find_groups", lambda self, rows: (found.append(1), real(self, rows))[1])
    a.alloc_extend([0], [0], [5 * R])
    assert a.shared_prefix([0]) is None and not found     # nothing was ever forked
    a.fork_req(0, [1, 2])
    want = ([0, 3], [5 * R])
    for step in range(3 * R):
        assert a.shared_prefix([0, 1, 2]) == want
        a.alloc_decode([0, 1, 2], [5 * R + step] * 3)
    assert len(found) == 1
    assert a.shared_prefix([0, 1]) == ([0, 2], [5 * R]) and len(found) == 2          # other members
    a.alloc_extend([7], [0], [R])
    assert a.shared_prefix([7, 0, 1]) == ([0, 1, 3], [0, 5 * R]) and len(found) == 3
    a.fork_req(0, [3])
    assert a.shared_prefix([0, 3, 1]) == ([0, 3], [5 * R])           # (0.7 x 3 - 1.2) x 5 runs, of two (0.7 x 2 - 1.2) x 8
    assert a.shared_prefix([0, 3]) == ([0, 2], [8 * R])
    a.rebuild_req(3, R)
    assert a.shared_prefix([0, 3, 1]) is None
    a.free_req(1)
    a.alloc_extend([1], [0], [5 * R])                                                 # the slot's next request
    assert a.shared_prefix([0, 1]) is None and a.shared_prefix([0, 2]) == ([0, 2], [5 * R])


def test_a_request_is_not_mistaken_for_its_slots_last_owner():
    a = _alloc()
    a.alloc_extend([0], [0], [4 * R])
    a.fork_req(0, [1, 2])
    assert a.shared_prefix([0, 1, 2]) == ([0, 3], [4 * R])
    a.free_req(2)
    a.alloc_extend([2], [0], [4 * R])
    assert a.shared_prefix([0, 1, 2]) == ([0, 2, 3], [4 * R, 0])
    a.clear()
    assert a.shared_prefix([0, 1, 2]) is None


def test_many_rows_do_not_take_long():
    """1024 rows, every fourth one a little deeper than its neighbours."""
    common = [0] + [60 + (i % 4 == 0) for i in range(1023)]
    t = time.perf_counter()
    memory_pool._best_groups(common, 0, 1024)
    assert time.perf_counter() - t < 1.0
