"""return_logprob of OPT (tied embeddings) and DeepSeek-V2, in two chunks, against the log-softmax of the same rows' logits."""
import pytest
import torch

from semi_pd_b200.forward_batch_info import ForwardBatch
from tests.helpers import GpuSession

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("family", ["opt", "deepseek"])
def test_input_token_logprobs(family):
    if family == "opt":
        from tests.test_gpu_opt import _runner
        mr, dtype = _runner(False)[0], torch.float16
    else:
        from tests.test_gpu_deepseek import _runner
        mr, dtype = _runner(None, torch.bfloat16)[0], torch.bfloat16
    vocab = mr.model_config.vocab_size
    p = [[(7 + 13 * i + 31 * j) % vocab for i in range(n)] for j, n in enumerate([5, 60, 33])]
    gs = GpuSession(mr)
    reqs = [gs.Req(f"r{i}", x, gs.SP()) for i, x in enumerate(p)]
    sb = gs.SB.init_new(reqs, mr.req_to_token_pool, mr.token_to_kv_pool_allocator, mr.device)
    sb.return_logprob = True
    seen = [0, 0, 0]
    for ends in ([2, 40, 16], [5, 60, 33]):
        for r, pre, end in zip(reqs, seen, ends):
            r.init_next_round_input(prefix_len=pre)
            r.fill_ids = r.fill_ids[:end]
            r.extend_input_len = end - pre
        T = sum(ends) - sum(seen)
        sb.prepare_for_extend()
        sb.extend_logit_rows = torch.arange(T, device=DEV)
        out = mr.forward(ForwardBatch.init_new(sb.get_model_worker_batch(), mr))
        logits = out.next_token_logits.double()
        targets = torch.tensor([t for x, pre, end in zip(p, seen, ends) for t in (x + [-1])[pre + 1:end + 1]], device=DEV)
        want = torch.log_softmax(logits, 1).gather(1, targets.clamp(min=0)[:, None])[:, 0] * (targets >= 0)
        # the logits here are rounded to 16 bits, those of the log-probabilities are not: half a step of the largest for the target's
        # and for the sum's, and 2^-13 of it for sums in fp32 of 2048 products at most
        tol = logits.abs().max().item() * (torch.finfo(dtype).eps + 2.0 ** -12)
        got = out.input_token_logprobs
        assert got.shape == (T,) and got.dtype == torch.float32
        assert ((got.double() - want).abs() <= tol).all() and (got[targets < 0] == 0).all()
        seen = ends
