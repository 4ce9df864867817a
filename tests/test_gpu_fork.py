"""Requests forked and compacted through the pools and the scheduler's batch: rows, states and page tables; decode steps over a
shared prefix against the same steps without it, and against requests that were never forked."""
import pytest
import torch

from tests.helpers import GpuSession, make_runner

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
           head_dim=128, vocab_size=1024, max_position_embeddings=4096)


def _rows(pool, table, req, n):
    slots = table[req, :n].long()
    return [b[slots].clone() for b in pool.planes.buffers]


def _pools(kind, runs=24, reqs=12, run_len=128):
    from semi_pd_b200.memory_pool import (HybridTokenToKVPool, MHATokenToKVPool, MLATokenToKVPool, RecurrentStatePool,
                                          ReqToTokenPool, TokenToKVPoolAllocator)
    size = runs * run_len
    if kind == "mha":
        pool = MHATokenToKVPool(size, 1, torch.bfloat16, 2, 128, 3, DEV)
    elif kind == "latent":
        pool = MLATokenToKVPool(size, 1, torch.float16, 512, 64, 3, DEV)
    else:
        states = RecurrentStatePool(reqs, [None, (2, 16, 24), None, (1, 8, 8)], DEV, shift_dims=[None, 48, None, None], token_state=True)
        pool = HybridTokenToKVPool(size, 1, torch.float32, [(2, 32, 48), None, (1, 64, 0), None], DEV, state_pool=states,
                                   block_sizes=[48, None, 32, None])
        for t in states.state + states.shift + [states.prev_token]:
            if t is not None:
                t.copy_(torch.randint(0, 1000, t.shape, device=DEV).to(t.dtype))
    for b in pool.planes.buffers:
        b.normal_()
    return pool, ReqToTokenPool(reqs, 2048, DEV), TokenToKVPoolAllocator(size, pool.dtype, DEV, pool)


def _place(table, alloc, n):
    (idx,) = table.alloc(1)
    table.req_to_token[idx, :n] = alloc.alloc_extend([idx], [0], [n]).int()
    return idx


@pytest.mark.parametrize("kind", ["mha", "latent", "hybrid"])
@pytest.mark.parametrize("n", [1, 128, 700])
def test_fork_through_the_pools(kind, n):
    from semi_pd_b200.memory_pool import fork_request
    pool, table, alloc = _pools(kind)
    parent = _place(table, alloc, n)
    before = _rows(pool, table.req_to_token, parent, n)
    children = fork_request(pool, table, alloc, parent, 3)
    assert len(children) == 3
    for c in [parent] + children:
        for a, b in zip(_rows(pool, table.req_to_token, c, n), before):
            assert torch.equal(a, b)
        assert table.req_to_token[c, :n].tolist() == alloc.req_slots(c).tolist()
    if kind == "hybrid":
        sp = pool.state_pool
        for t in sp.state + sp.shift + [sp.prev_token]:
            if t is not None:
                assert all(torch.equal(t[c], t[parent]) for c in children)
        for layer in (0, 2):
            size, run_len, base = pool.get_blocks(layer)
            per = -(-run_len // size)
            rows = lambda r: pool.k_buffer[layer][base + r * per:base + (r + 1) * per]
            for c in children:
                for mine, theirs in zip(alloc._req_runs[c], alloc._req_runs[parent]):
                    assert torch.equal(rows(mine), rows(theirs))
    # a child's next token does not touch the others
    slot = alloc.alloc_decode([children[0]], [n])
    for b in pool.planes.buffers:
        b[slot] = 7.0
    for c in (parent, children[1]):
        for a, b in zip(_rows(pool, table.req_to_token, c, n), before):
            assert torch.equal(a, b)


def test_fork_takes_nothing_when_slots_or_runs_do_not_suffice():
    from semi_pd_b200.memory_pool import fork_request
    pool, table, alloc = _pools("mha", runs=4, reqs=5)
    parent = _place(table, alloc, 300)
    for n in (2, 9):
        assert fork_request(pool, table, alloc, parent, n) is None
        assert table.available_size() == 4 and alloc.available_size() == 128
    assert fork_request(pool, table, alloc, parent, 0) == []
    with pytest.raises(RuntimeError):
        fork_request(pool, table, alloc, 99, 1)
    assert table.available_size() == 4


@pytest.mark.parametrize("kind", ["mha", "latent"])
def test_compact_through_the_pools(kind):
    from semi_pd_b200.memory_pool import compact_request, fork_request
    pool, table, alloc = _pools(kind)
    req = _place(table, alloc, 700)
    (other,) = fork_request(pool, table, alloc, req, 1)
    before = _rows(pool, table.req_to_token, req, 700)
    keep = list(range(4)) + list(range(300, 411)) + list(range(500, 700, 3))
    free = alloc.available_size()
    assert compact_request(pool, table, alloc, req, keep)
    n = len(keep)
    for a, b in zip(_rows(pool, table.req_to_token, req, n), before):
        assert torch.equal(a, b[torch.tensor(keep, device=DEV)])
    for a, b in zip(_rows(pool, table.req_to_token, other, 700), before):
        assert torch.equal(a, b)
    assert alloc.req_len(req) == n and table.req_to_token[req, :n].tolist() == alloc.req_slots(req).tolist()
    assert alloc.available_size() == free - 2 * 128 + 128   # two new runs, the partial one back
    for bad in ([], [3, 3], [5, 4], [-1, 2], [n]):
        with pytest.raises(RuntimeError, match="positions"):
            compact_request(pool, table, alloc, req, bad)


def test_compact_refuses_pools_that_hold_more_than_rows():
    from semi_pd_b200.memory_pool import compact_request
    pool, table, alloc = _pools("hybrid")
    req = _place(table, alloc, 200)
    with pytest.raises(NotImplementedError, match="states"):
        compact_request(pool, table, alloc, req, [0, 1])


def test_steps_over_a_shared_prefix(monkeypatch):
    """One prompt, 61 continuations: five decode steps with the prefix shared, without, and some of them unforked."""
    from semi_pd_b200.attention_backend import SpdAttnBackend
    from semi_pd_b200 import ops
    mr, _, _ = make_runner(CFG, torch.float16, kv_slots=24 * 1024, max_reqs=150, ctx=4096)
    prompt = [(11 + 29 * i) % 1024 for i in range(2500)]
    steps = [[(5 + 7 * i + 131 * s) % 1024 for i in range(61)] for s in range(5)]
    calls = []
    real = ops.attn_decode_shared
    monkeypatch.setattr(ops, "attn_decode_shared", lambda *a, **k: (calls.append(1), real(*a, **k))[1])

    def run(share):
        monkeypatch.setattr(SpdAttnBackend, "shares_prefix", shares if share else lambda *a: False)
        gs = GpuSession(mr)
        reqs, _, _ = gs.extend([prompt])
        children = gs.batch.fork_req(0, 60)
        assert len(children) == 60 and len({r.req_pool_idx for r in gs.batch.reqs}) == 61
        reqs = list(gs.batch.reqs)
        out = [gs.decode(reqs, toks)[0] for toks in steps]
        for r in reqs:
            mr.token_to_kv_pool_allocator.free_req(r.req_pool_idx)
            mr.req_to_token_pool.free(r.req_pool_idx)
        return torch.stack(out)

    shares = SpdAttnBackend.shares_prefix
    free = mr.token_to_kv_pool_allocator.available_size()
    with_it = run(True)
    assert len(calls) == 5 * CFG["num_hidden_layers"]  # the rule takes it for this batch
    without = run(False)
    assert len(calls) == 5 * CFG["num_hidden_layers"]
    assert mr.token_to_kv_pool_allocator.available_size() == free
    # both sides round alike but sum in another order; logits of the session's size are within 1e-2 of the oracle's
    assert (with_it - without).abs().max().item() < 1e-2
    gs = GpuSession(mr)
    some = [0, 17, 60]
    reqs, _, _ = gs.extend([prompt] * 3)
    for s, toks in enumerate(steps):
        lg, _ = gs.decode(reqs, [toks[i] for i in some])
        assert (lg - with_it[s][some]).abs().max().item() < 1e-2
    for r in reqs:
        mr.token_to_kv_pool_allocator.free_req(r.req_pool_idx)
        mr.req_to_token_pool.free(r.req_pool_idx)


def test_attention_over_a_compacted_request():
    """Decode attention of a request that went on with a part of its tokens is attention over those tokens."""
    from semi_pd_b200 import ops
    from semi_pd_b200.memory_pool import compact_request
    pool, table, alloc = _pools("mha")
    req = _place(table, alloc, 900)
    k, v = pool.k_buffer[1], pool.v_buffer[1]
    slots = table.req_to_token[req, :900].long()
    keep = list(range(8)) + list(range(450, 900))
    kk, vv = k[slots][keep].double(), v[slots][keep].double()
    assert compact_request(pool, table, alloc, req, keep)
    q = torch.randn(1, 4 * 128, device=DEV).to(torch.bfloat16)
    out = ops.attn_decode(q, k, v, table.req_to_token, torch.tensor([req], device=DEV), torch.tensor([len(keep)], device=DEV), 4, 2,
                          128, 128 ** -0.5)
    s = torch.einsum("hd,nhd->hn", q.double().view(4, 128), kk.repeat_interleave(2, 1)) * 128 ** -0.5
    p = torch.softmax(s, -1)
    want = torch.einsum("hn,nhd->hd", p, vv.repeat_interleave(2, 1))
    spread = torch.einsum("hn,nhd->hd", p, (vv.repeat_interleave(2, 1) - want).abs())
    u = 2.0 ** -8   # weights and output rounded to bf16, half a step each
    assert bool(((out.double().view(4, 128) - want).abs() <= 1.02 * u * (spread + want.abs()) + 1e-4).all())


@pytest.mark.parametrize("what", ["fork", "compact"])
def test_what_a_copy_reads_is_not_written_by_another_stream(what):
    """A request that is let go right after it was forked (or compacted), its runs and slots asked for on another stream while the
    copy has not begun."""
    from semi_pd_b200.memory_pool import compact_request, fork_request
    pool, table, alloc = _pools("mha", runs=8, reqs=3)
    parent = _place(table, alloc, 500)            # four of eight runs
    before = _rows(pool, table.req_to_token, parent, 500)
    torch.cuda.synchronize()
    one, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        torch.cuda._sleep(200_000_000)            # about 0.1 s
        if what == "fork":
            (req,) = fork_request(pool, table, alloc, parent, 1)
            alloc.free_req(parent)
            table.free(parent)
            keep = list(range(500))
        else:
            keep = list(range(3, 500, 2))
            assert compact_request(pool, table, alloc, parent, keep)
            req = parent
    with torch.cuda.stream(other):
        while table.available_size() and alloc.available_size():
            (idx,) = table.alloc(1)
            n = min(alloc.available_size(), 256)
            slots = alloc.alloc_extend([idx], [0], [n])
            table.req_to_token[idx] = -1
            for b in pool.planes.buffers:
                b[slots] = 0
    torch.cuda.synchronize()
    for a, b in zip(_rows(pool, table.req_to_token, req, len(keep)), before):
        assert torch.equal(a, b[keep])
