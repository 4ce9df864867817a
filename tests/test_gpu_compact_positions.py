"""Decode steps of a request whose cache was compacted, against the oracle over the same rows: the keys that are left are rotated
for their old positions, so the next query stands where it would have stood."""
import pytest
import torch

from oracle import llama_oracle as O
from tests.helpers import GpuSession, make_runner

pytestmark = pytest.mark.gpu
CFG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
           head_dim=128, vocab_size=1024, max_position_embeddings=2048)
TOL = 1e-2      # of fp16 logits against the oracle's, as for every model of this size


def _compact_oracle(session, oracle, rid, keep):
    keep = torch.tensor(keep)
    oracle.req_to_token[rid, :len(keep)] = oracle.req_to_token[rid, keep].clone()
    session.lens[rid] = len(keep)


@pytest.mark.parametrize("graph", [False, True])
def test_steps_after_a_compaction(monkeypatch, graph):
    mr, oracle, _ = make_runner(CFG, torch.float16, cuda_graph=graph, cuda_graph_bs=[1, 2, 4] if graph else None)
    gs, os_ = GpuSession(mr), O.OracleSession(oracle, 4096, 17)
    prompts = [[(7 + 13 * i + 31 * j * i * i) % 1024 for i in range(n)] for j, n in enumerate((700, 300))]
    reqs, lg, _ = gs.extend(prompts)
    rids, lc, _ = os_.extend(prompts)
    clamp, offsets = O.clamp_position, [0, 0]
    monkeypatch.setattr(O, "clamp_position", lambda seq: clamp(seq) + torch.tensor(offsets))

    def steps(n):
        for s in range(n):
            toks = [(17 + 5 * s + 101 * i) % 1024 for i in range(len(rids))]
            lg, _ = gs.decode(list(gs.batch.reqs), toks)
            lc, _ = os_.decode(rids, toks)
            assert (lg - lc).abs().max().item() < TOL

    steps(2)
    keep = list(range(4)) + list(range(351, 702))
    free = mr.token_to_kv_pool_allocator.available_size()
    assert gs.batch.compact_req(0, keep)
    assert gs.batch.seq_lens_host == [355, 302] == gs.batch.seq_lens.tolist() and gs.batch.seq_lens_sum == 657
    assert mr.token_to_kv_pool_allocator.available_size() == free + 3 * 128
    _compact_oracle(os_, oracle, rids[0], keep)
    # the other positions give other logits, by more than the tolerance: a wrong one would be seen
    toks = [3, 5]
    lens = dict(os_.lens)
    wrong, _ = os_.decode(rids, toks)
    os_.lens = lens
    offsets[0] = 702 - 355
    right, _ = os_.decode(rids, toks)
    assert (right[0] - wrong[0]).abs().max().item() > 5 * TOL
    lg, _ = gs.decode(list(gs.batch.reqs), toks)
    assert (lg - right).abs().max().item() < TOL
    steps(3)
    # again, the other one too, and a fork of the first
    for i, keep in ((0, list(range(0, 359, 2))), (1, list(range(100, 306)))):
        offsets[i] += gs.batch.seq_lens_host[i] - len(keep)
        assert gs.batch.compact_req(i, keep)
        _compact_oracle(os_, oracle, rids[i], keep)
    steps(2)
    gs.batch.fork_req(0, 1)
    n = os_.lens[rids[0]]
    child = os_.free_reqs.pop(0)
    oracle.req_to_token[child, :n] = oracle.req_to_token[rids[0], :n]
    os_.lens[child] = n
    rids.insert(1, child)
    offsets.insert(1, offsets[0])
    steps(2)
    # what is left of the batch
    gs.batch.filter_batch(keep_indices=[2])
    del rids[:2], offsets[:2]
    steps(1)
    # a fresh request beside it has no offset, and alone its batch has none
    fresh = GpuSession(mr)
    fresh.extend([[(9 * i) % 1024 for i in range(50)]])
    fresh.batch.output_ids = torch.zeros(1, dtype=torch.int64, device=mr.device)
    gs.batch.output_ids = torch.zeros(len(gs.batch.reqs), dtype=torch.int64, device=mr.device)
    gs.batch.merge_batch(fresh.batch)
    offsets = gs.batch._position_offsets()
    assert offsets.tolist() == [gs.batch.reqs[0].dropped_tokens, 0]
    gs.batch.filter_batch(keep_indices=[1])
    assert gs.batch._position_offsets() is None


def test_refusals():
    mr, _, _ = make_runner(CFG, torch.float16)
    gs = GpuSession(mr)
    reqs, _, _ = gs.extend([[1, 2, 3, 4, 5, 6]])
    for bad in ([], [2, 1], [0, 6]):
        with pytest.raises(RuntimeError, match="positions"):
            gs.batch.compact_req(0, bad)
    assert gs.batch.compact_req(0, [0, 5]) and gs.batch.seq_lens_host == [2]
    with pytest.raises(NotImplementedError, match="compacted"):
        gs.extend([[7, 8]], reqs)
    reqs[0].finished_reason = "length"
    with pytest.raises(RuntimeError, match="finished"):
        gs.batch.compact_req(0, [0])
