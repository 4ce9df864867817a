"""Log-probabilities of a prompt's tokens chunk by chunk through one ScheduleBatch, up to its decode steps."""
import pytest
import torch

from oracle import llama_oracle as O
from semi_pd_b200.forward_batch_info import ForwardBatch
from tests.helpers import GpuSession
from tests.test_gpu_w8a8_model import TINY, prompts, runner

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("quantization", [None, "w8a8_int8"])
def test_chunks(quantization):
    """Every row against the log-softmax of its own logits (rounded to 16 bits: half a step of the largest, 2^-9 of 8 at most, twice); the
    last row of a chunk has the token that the next chunk begins with."""
    mr = runner(TINY, torch.bfloat16, O.make_weights(O.OracleLlamaConfig(**TINY), torch.bfloat16), quantization)
    gs = GpuSession(mr)
    p = prompts([40, 7, 150], 1000)
    reqs = [gs.Req(f"r{i}", x, gs.SP()) for i, x in enumerate(p)]
    sb = gs.SB.init_new(reqs, mr.req_to_token_pool, mr.token_to_kv_pool_allocator, mr.device)
    sb.return_logprob = True
    seen = [0, 0, 0]
    for ends in ([16, 3, 64], [32, 6, 128], [40, 7, 150]):
        for r, pre, end in zip(reqs, seen, ends):
            r.init_next_round_input(prefix_len=pre)
            r.fill_ids = r.fill_ids[:end]
            r.extend_input_len = end - pre
        T = sum(ends) - sum(seen)
        if ends[0] == 16:  # of one chunk the caller's own tokens
            sb.extend_input_logprob_token_ids = own = torch.arange(T, device=DEV) * 11 % 1000
        sb.prepare_for_extend()
        sb.extend_logit_rows = torch.arange(T, device=DEV)
        out = mr.forward(ForwardBatch.init_new(sb.get_model_worker_batch(), mr))
        logits = out.next_token_logits.double()
        assert logits.abs().max() < 8
        nexts = [t for x, pre, end in zip(p, seen, ends) for t in (x + [-1])[pre + 1:end + 1]]
        targets = own if ends[0] == 16 else torch.tensor(nexts, device=DEV)
        want = torch.log_softmax(logits, 1).gather(1, targets.clamp(min=0)[:, None])[:, 0] * (targets >= 0)
        got = out.input_token_logprobs
        assert got.shape == (T,) and ((got.double() - want).abs() <= 2 * 8 * 2.0 ** -9).all()
        assert torch.equal(got == 0, targets < 0)
        seen = ends
    for r in reqs:
        r.output_ids.append(5)
    sb.output_ids = torch.full((3,), 5, dtype=torch.int64, device=DEV)
    sb.prepare_for_decode()
    out = mr.forward(ForwardBatch.init_new(sb.get_model_worker_batch(), mr))
    assert out.next_token_logits.shape == (3, 1000) and out.input_token_logprobs is None
