"""Requests forked while the engine decodes: the loop keeps a launched step unread, whose token must reach the children too."""
import pytest
import torch

from oracle import llama_oracle as O
from tests.test_gpu_engine import CFG, _build_engine

pytestmark = pytest.mark.gpu


def test_continuations_of_a_running_request():
    ocfg = O.OracleLlamaConfig(**CFG)
    eng = _build_engine(torch.float16, O.make_weights(ocfg, torch.float16, seed=5), 4096)
    decode, new = eng.decode, 24
    plain, seen = decode.get_next_batch_to_run, {}

    def hooked():
        batch = decode.running_batch
        parent = next((r for r in batch.reqs if r.rid == seen.get("rid")), None)
        if parent is not None and not parent.finished():
            if "first" not in seen and len(parent.output_ids) >= 6:
                assert parent.launched_tokens == len(parent.output_ids) + 1 and decode.result_queue
                free = (decode.token_to_kv_pool_allocator.available_size(), decode.req_to_token_pool.available_size())
                try:
                    batch.fork_req(batch.reqs.index(parent), 2)
                except RuntimeError as e:
                    seen["refused"] = str(e)
                seen["kept"] = free == (decode.token_to_kv_pool_allocator.available_size(), decode.req_to_token_pool.available_size())
                seen["first"] = decode.fork_running(parent.rid, 2)
                seen["at"] = len(parent.output_ids)
            elif "second" not in seen and "first" in seen and len(parent.output_ids) >= 14:
                seen["second"] = decode.fork_running(parent.rid, 1)
                seen["none"] = decode.fork_running("nobody", 1)
                seen["too many"] = decode.fork_running(parent.rid, 99)
        return plain()

    decode.get_next_batch_to_run = hooked
    try:
        prompt = [(5 + 7 * i) % 1024 for i in range(200)]
        others = [eng.submit([(3 + i + j) % 1024 for i in range(40)], 40) for j in range(2)]
        seen["rid"] = eng.submit(prompt, new)
        done = {r.rid: r for r in eng.wait(3 + 3, timeout=60)}
        pools = eng.d_worker.model_runner.token_to_kv_pool_allocator, eng.d_worker.model_runner.req_to_token_pool
    finally:
        eng.shutdown()
    assert "unread" in seen["refused"] and seen["kept"] and seen["none"] is None and seen["too many"] is None
    parent = done[seen["rid"]]
    children = seen["first"] + seen["second"]
    assert sorted(done) == sorted(others + [parent.rid] + [c.rid for c in children]) and len({c.rid for c in children}) == 3
    for c, n in zip(children, (seen["at"], seen["at"], 14)):
        assert done[c.rid] is c and len(c.output_ids) == new == len(c.token_times) and c.finished_reason == "length"
        # greedy and of the same tokens: alike, at least to the token behind the fork
        assert c.output_ids[:n + 1] == parent.output_ids[:n + 1]
    assert pools[0].available_size() == pools[0].num_runs * pools[0].run_len and pools[1].available_size() == pools[1].size
    assert (pools[0]._held == 0).all() and (pools[0]._used == 0).all()


def test_a_finished_request_is_not_forked():
    from tests.helpers import GpuSession, make_runner
    mr, _, _ = make_runner(CFG, torch.float16)
    gs = GpuSession(mr)
    reqs, _, _ = gs.extend([[1, 2, 3, 4, 5, 6]])
    first, second = gs.batch.fork_req(0, 2), gs.batch.fork_req(0, 1)
    assert len({r.rid for r in reqs + first + second}) == 4 and len({r.rid for r in gs.batch.fork_req(1, 2)} | {r.rid for r in gs.batch.reqs}) == 6
    assert gs.batch.fork_req(0, 0) == [] and len(gs.batch.reqs) == 6
    reqs[0].finished_reason = "stop"
    with pytest.raises(RuntimeError, match="finished"):
        gs.batch.fork_req(0, 1)
