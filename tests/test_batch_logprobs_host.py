"""Which tokens an extend batch's log-probabilities are asked of (ScheduleBatch.return_logprob): the requests' next ones, chunk by chunk, or
the caller's own for one batch."""
import pytest
import torch

from semi_pd_b200.forward_batch_info import ForwardMode
from semi_pd_b200.schedule_batch import Req, SamplingParams, ScheduleBatch


class Refuses:
    device = "cpu"

    def alloc(self, n):
        return None


@pytest.fixture
def batch(monkeypatch):
    monkeypatch.setattr(ScheduleBatch, "_h2d", lambda self, values, dtype: torch.tensor(values, dtype=dtype))

    def make(*prompts):
        reqs = [Req(f"r{i}", p, SamplingParams()) for i, p in enumerate(prompts)]
        sb = ScheduleBatch.init_new(reqs, Refuses(), None, "cpu")
        assert sb.return_logprob is False and sb.extend_input_logprob_token_ids is None
        return sb

    return make


def chunk(sb, ends):
    """Every request's tokens up to `ends`, behind what it had: what prepare_for_extend notes of them, without a device."""
    for r, end in zip(sb.reqs, ends):
        r.init_next_round_input(prefix_len=len(r.fill_ids))
        r.fill_ids = r.fill_ids[:end]
        r.extend_input_len = end - len(r.prefix_indices)
    with pytest.raises(RuntimeError, match="max-running-requests"):  # past the list's upkeep, the first thing that needs a pool
        sb.prepare_for_extend()
    sb.prefix_lens = [len(r.prefix_indices) for r in sb.reqs]
    sb.extend_lens = [r.extend_input_len for r in sb.reqs]


def asked(sb):
    b = sb.get_model_worker_batch()
    return b.return_logprob, None if b.extend_input_logprob_token_ids is None else b.extend_input_logprob_token_ids.tolist()


def test_next_tokens_of_every_chunk(batch):
    sb = batch([10, 11, 12, 13, 14], [20], [30, 31, 32])
    sb.return_logprob = True
    chunk(sb, [2, 1, 3])
    assert asked(sb) == (True, [11, 12, -1, 31, 32, -1])
    chunk(sb, [4, 1, 3])       # nothing more of the others
    assert asked(sb) == (True, [13, 14])
    chunk(sb, [5, 1, 3])
    assert asked(sb) == (True, [-1])
    assert sb._next_input_tokens().dtype == torch.int64


def test_output_is_known_too(batch):
    sb = batch([1, 2])
    sb.return_logprob = True
    sb.reqs[0].output_ids = [3, 4]   # retracted: its output is prompt now
    chunk(sb, [3])
    assert asked(sb) == (True, [2, 3, 4])
    chunk(sb, [4])
    assert asked(sb) == (True, [-1])


@pytest.mark.parametrize("late", [False, True])
def test_tokens_of_the_callers_own_are_for_one_batch(batch, late):
    sb = batch([1, 2, 3, 4, 5, 6])
    sb.return_logprob = True
    own = torch.tensor([7, -1, 9])
    if not late:
        sb.extend_input_logprob_token_ids = own
    chunk(sb, [3])
    if late:
        sb.extend_input_logprob_token_ids = own
    assert asked(sb) == (True, [7, -1, 9]) and asked(sb) == (True, [7, -1, 9])
    chunk(sb, [6])                  # as many tokens: the last batch's would fit
    assert asked(sb) == (True, [5, 6, -1])
    sb.extend_input_logprob_token_ids = own     # the same list again, said again
    chunk(sb, [6])
    sb.return_logprob = False
    assert asked(sb)[0] is False


def test_not_asked(batch):
    sb = batch([1, 2, 3])
    chunk(sb, [3])
    assert asked(sb) == (False, None)


def test_a_decode_batch_has_no_input_tokens(batch, monkeypatch):
    sb = batch([1, 2, 3])
    sb.return_logprob = True
    chunk(sb, [3])
    assert asked(sb)[0]
    sb.forward_mode = ForwardMode.DECODE
    monkeypatch.setattr(ScheduleBatch, "_shared_prefix", lambda self: None)
    assert asked(sb) == (False, None)
