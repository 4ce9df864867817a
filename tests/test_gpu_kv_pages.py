"""kv_copy, kv_fork, kv_compact: rows of every layer's pool and page-table entries, bit for bit what indexing gives, in pools of
one kind and of several, with rows that no vector fits, skipped slots, several calls' worth of buffers, graphs and streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bits(t):
    return t.contiguous().view(torch.uint8).cpu()


# pools: (rows' shapes and dtypes of the buffers, all layers in one allocation)
POOLS = {
    "mha": ([(8, 128)] * 6, torch.bfloat16, True),
    "latent": ([(1, 576)] * 5, torch.float16, True),
    "f32": ([(2, 64)] * 4, torch.float32, True),
    "odd": ([(1, 3), (5, 7), (1, 1)], torch.bfloat16, False),       # 6, 70 and 2 bytes: pieces of two
    "mixed": ([(4, 96), (4, 64), (2, 32), (1, 8)], torch.float32, False),
    "many": ([(1, 8 + 2 * (i % 3)) for i in range(150)], torch.float16, False),  # more sets than a call takes
    "wide": ([(64, 512)], torch.float32, False),                    # rows of 128 KB
}


def _pool(kind, slots, seed=0):
    shapes, dtype, slab = POOLS[kind]
    g = torch.Generator(device=DEV).manual_seed(seed)
    if slab:
        one = torch.randn(len(shapes), slots, *shapes[0], generator=g, device=DEV).to(dtype)
        return list(one)
    return [torch.randn(slots, *s, generator=g, device=DEV).to(dtype) for s in shapes]


def _same(bufs, want):
    for i, (b, w) in enumerate(zip(bufs, want)):
        assert torch.equal(_bits(b), _bits(w)), f"buffer {i}"


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 300])
def test_copy(kind, n):
    from semi_pd_b200 import ops
    slots = 2 * n + 5
    bufs = _pool(kind, slots, n)
    planes = ops.KVPlanes(bufs)
    perm = torch.randperm(slots, generator=torch.Generator().manual_seed(n))
    src, dst = perm[:n].to(DEV), perm[n:2 * n].to(DEV)
    want = [b.clone() for b in bufs]
    for w in want:
        w[dst] = w[src]
    ops.kv_copy(planes, src, dst)
    _same(bufs, want)


def test_copy_one_source_many_times_and_slots_left_out():
    from semi_pd_b200 import ops
    bufs = _pool("mha", 40)
    planes = ops.KVPlanes(bufs)
    src = torch.tensor([7, 7, 7, -1, 3, 40, 1 << 40, 5], device=DEV)
    dst = torch.tensor([20, 21, 22, 23, -5, 24, 25, 40], device=DEV)
    want = [b.clone() for b in bufs]
    for w in want:
        w[20:23] = w[7]
    ops.kv_copy(planes, src, dst)
    _same(bufs, want)


def test_copy_past_32_bits():
    """Slots whose rows lie beyond 4 GB."""
    from semi_pd_b200 import ops
    rows = (5 << 30) // 2048
    buf = torch.zeros(rows, 8, 128, dtype=torch.bfloat16, device=DEV)
    buf[rows - 3] = 3.0
    buf[5] = 5.0
    ops.kv_copy(ops.KVPlanes([buf]), torch.tensor([rows - 3, 5], device=DEV), torch.tensor([9, rows - 1], device=DEV))
    assert bool((buf[9] == 3).all()) and bool((buf[rows - 1] == 5).all()) and bool((buf[10:rows - 3] == 0).all())


def test_copy_shared_buffer_counts_once():
    from semi_pd_b200 import ops
    bufs = _pool("mixed", 30)
    planes = ops.KVPlanes(bufs + [bufs[0], None, bufs[2]])
    assert len(planes.buffers) == len(bufs)
    assert planes.token_bytes == sum(b[0].numel() * b.element_size() for b in bufs)


def _fork_case(lens, kids, run, kind, seed=0):
    """Parents of these lengths in shuffled runs, `kids` children each, a fresh run per child."""
    g = torch.Generator().manual_seed(seed + sum(lens))
    need = sum(-(-n // run) for n in lens) + len(lens) * kids
    order = torch.randperm(max(need, 1), generator=g)
    ids = torch.randperm(len(lens) * (1 + kids) + 3, generator=g)
    table = torch.full((len(ids), max(lens) + 5), -7, dtype=torch.int32)
    at, rows = 0, []
    for i, n in enumerate(lens):
        runs = order[at:at + -(-n // run)]
        at += len(runs)
        pos = torch.arange(n)
        table[ids[i], :n] = (runs[pos // run] * run + 1 + pos % run).int() if n else pos.int()
        for c in range(kids):
            rows.append((int(ids[i]), int(ids[len(lens) + i * kids + c]), n, int(order[at]) * run + 1))
            at += 1
    return _pool(kind, need * run + 1, seed), table.to(DEV), rows


def _lists(rows):
    return [torch.tensor(x, dtype=torch.int64, device=DEV) for x in zip(*rows)]


def _fork_want(bufs, table, rows, run):
    bufs, table = [b.clone() for b in bufs], table.clone()
    for parent, child, n, base in rows:
        full = n // run * run
        table[child, :full] = table[parent, :full]
        table[child, full:n] = torch.arange(base, base + n - full, dtype=torch.int32, device=DEV)
        for b in bufs:
            b[base:base + n - full] = b[table[parent, full:n].long()]
    return bufs, table


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("lens,kids,run", [([1], 1, 128), ([128], 2, 128), ([0, 5], 3, 128), ([127, 129, 1000], 4, 128),
                                           ([77, 16, 31], 2, 16), ([9], 5, 1), ([300, 3], 40, 128), ([4000], 2, 128)])
def test_fork(kind, lens, kids, run):
    from semi_pd_b200 import ops
    if kind == "wide" and (max(lens) > 300 or kids > 5):
        pytest.skip("gigabytes of rows that show nothing else")
    bufs, table, rows = _fork_case(lens, kids, run, kind)
    want, want_table = _fork_want(bufs, table, rows, run)
    ops.kv_fork(ops.KVPlanes(bufs), table, *_lists(rows), run)
    _same(bufs, want)
    assert torch.equal(table, want_table)


@pytest.mark.parametrize("order", [0, 1, 2])
def test_fork_lengths_of_children_differ_and_parents_mix(order):
    """Children that take less of their parent than the next one does, and lists in which parents do not stand together."""
    from semi_pd_b200 import ops
    bufs, table, rows = _fork_case([300, 200, 90], 5, 128, "mha")
    rows = [(p, c, n - (7 * i) % 11 * (i % 3), base) for i, (p, c, n, base) in enumerate(rows)]
    rows = [rows[i] for i in torch.randperm(len(rows), generator=torch.Generator().manual_seed(order))] if order else rows
    want, want_table = _fork_want(bufs, table, rows, 128)
    ops.kv_fork(ops.KVPlanes(bufs), table, *_lists(rows), 128)
    _same(bufs, want)
    assert torch.equal(table, want_table)


def test_fork_leaves_bad_requests_alone():
    from semi_pd_b200 import ops
    bufs, table, rows = _fork_case([200], 1, 128, "mha")
    before, before_table = [b.clone() for b in bufs], table.clone()
    n = table.shape[0]
    bad = [(n, rows[0][1], 200, 300), (-1, rows[0][1], 200, 300), (rows[0][0], rows[0][1], table.shape[1] + 1, 300),
           (rows[0][0], rows[0][1], -4, 300)]
    ops.kv_fork(ops.KVPlanes(bufs), table, *_lists(bad), 128)
    _same(bufs, before)
    assert torch.equal(table, before_table)


def _compact_case(lens, kept, kind, seed=0, run=128):
    g = torch.Generator().manual_seed(seed + sum(lens))
    need = sum(-(-n // run) + -(-k // run) for n, k in zip(lens, kept))
    order = torch.randperm(max(need, 1), generator=g)
    ids = torch.randperm(2 * len(lens) + 2, generator=g)
    table = torch.full((len(ids), max(lens) + 3), -7, dtype=torch.int32)
    at, keep, loc, indptr = 0, [], [], [0]
    for i, (n, k) in enumerate(zip(lens, kept)):
        runs, pos = order[at:at + -(-n // run)], torch.arange(n)
        at += len(runs)
        table[ids[i], :n] = (runs[pos // run] * run + 1 + pos % run).int() if n else pos.int()
        keep.append(torch.randperm(n, generator=g)[:k].sort().values)
        runs, pos = order[at:at + -(-k // run)], torch.arange(k)
        at += len(runs)
        loc.append(runs[pos // run] * run + 1 + pos % run if k else pos)
        indptr.append(indptr[-1] + k)
    m = len(lens)
    return (_pool(kind, need * run + 1, seed), table.to(DEV), ids[:m].to(DEV), ids[m:2 * m].to(DEV), torch.cat(keep).to(DEV),
            torch.tensor(indptr, device=DEV), torch.cat(loc).to(DEV))


@pytest.mark.parametrize("kind", list(POOLS))
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,kept", [([1], [1]), ([10], [0]), ([0, 5, 0], [0, 5, 0]), ([300, 129, 64], [299, 1, 64]),
                                       ([700], [350]), ([40 + 7 * i for i in range(12)], [3 * i for i in range(12)])])
def test_compact(kind, lens, kept, in_place):
    from semi_pd_b200 import ops
    bufs, table, src, dst, keep, indptr, loc = _compact_case(lens, kept, kind)
    if in_place:
        dst = src
    want, want_table = [b.clone() for b in bufs], table.clone()
    p = indptr.tolist()
    for i in range(len(lens)):
        to, old = loc[p[i]:p[i + 1]], table[src[i], keep[p[i]:p[i + 1]]].long()
        for w in want:
            w[to] = w[old]
        want_table[dst[i], :len(to)] = to.int()
    ops.kv_compact(ops.KVPlanes(bufs), table, src, None if in_place else dst, keep, indptr, loc)
    _same(bufs, want)
    assert torch.equal(table, want_table)


def test_compact_keeps_any_order_and_leaves_bad_entries_out():
    from semi_pd_b200 import ops
    bufs, table, src, dst, _, _, _ = _compact_case([200, 200], [100, 100], "mha")
    keep = torch.tensor([150, 3, 77, -1, table.shape[1], 5], device=DEV)
    free = [s for s in range(1, bufs[0].shape[0]) if s not in set(table[src].flatten().tolist())][:6]
    loc = torch.tensor(free, device=DEV)
    indptr = torch.tensor([0, 3, 6], device=DEV)
    want, want_table = [b.clone() for b in bufs], table.clone()
    for j, (r, pos) in enumerate([(0, 150), (0, 3), (0, 77), (1, None), (1, None), (1, 5)]):
        if pos is not None:
            for w in want:
                w[free[j]] = w[table[src[r], pos].long()]
    want_table[dst[0], :3] = loc[:3].int()
    want_table[dst[1], :3] = loc[3:].int()
    ops.kv_compact(ops.KVPlanes(bufs), table, src, dst, keep, indptr, loc)
    _same(bufs, want)
    assert torch.equal(table, want_table)


@pytest.mark.parametrize("own_stream", [False, True])
def test_captured_calls_follow_their_lists(own_stream):
    """One graph, replayed with other slots and lengths in the same lists."""
    from semi_pd_b200 import ops
    bufs, table, rows = _fork_case([200, 300], 2, 128, "mha")
    planes = ops.KVPlanes(bufs)
    lists = _lists(rows)
    src, dst = torch.tensor([1, 2], device=DEV), torch.tensor([1, 2], device=DEV)  # onto themselves
    stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream if own_stream else None):
        ops.kv_fork(planes, table, *lists, 128)
        ops.kv_copy(planes, src, dst)
    torch.cuda.synchronize()
    free = rows[0][3] + 100  # inside the first child's run, behind its tokens
    src.fill_(rows[0][3])
    dst.copy_(torch.tensor([free, free + 1], device=DEV))
    lists[2].copy_(torch.tensor([150, 129, 256, 257], device=DEV))
    changed = [(a, b, n, d) for (a, b, _, d), n in zip(rows, (150, 129, 256, 257))]
    want, want_table = _fork_want(bufs, table, changed, 128)
    for w in want:
        w[[free, free + 1]] = w[rows[0][3]].clone()
    graph.replay()
    torch.cuda.synchronize()
    _same(bufs, want)
    assert torch.equal(table, want_table)


def test_refusals():
    from semi_pd_b200 import ops
    bufs = _pool("mha", 20)
    planes = ops.KVPlanes(bufs)
    i64 = torch.tensor([1, 2], device=DEV)
    table = torch.zeros(4, 10, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="int64"):
        ops.kv_copy(planes, i64.int(), i64)
    with pytest.raises(RuntimeError, match="as many"):
        ops.kv_copy(planes, i64, i64[:1])
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.kv_copy(planes, i64.cpu(), i64)
    with pytest.raises(RuntimeError, match="int32"):
        ops.kv_fork(planes, table.long(), i64, i64, i64, i64, 128)
    with pytest.raises(RuntimeError, match="per child"):
        ops.kv_fork(planes, table, i64, i64[:1], i64, i64, 128)
    with pytest.raises(RuntimeError, match="run_len"):
        ops.kv_fork(planes, table, i64, i64, i64, i64, 0)
    with pytest.raises(RuntimeError, match="one more offset"):
        ops.kv_compact(planes, table, i64, None, i64, i64, i64)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.KVPlanes([bufs[0][::2]])
    with pytest.raises(RuntimeError, match="even number"):
        ops.kv_copy(ops.KVPlanes([torch.zeros(20, 3, dtype=torch.uint8, device=DEV)]), i64, i64)
