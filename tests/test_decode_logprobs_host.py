"""return_logprob where there are no input tokens' log-probabilities is refused, not passed over."""
from types import SimpleNamespace

import pytest

from semi_pd_b200.forward_batch_info import ForwardMode
from semi_pd_b200.model_runner import ModelRunner


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("asked", [False, True])
def test_decode(graphs, asked):
    ran = []
    runner = SimpleNamespace(
        tp_comm=None, forward_decode=lambda fb: ran.append("eager"),
        cuda_graph_runner=SimpleNamespace(can_run=lambda fb: True, replay=lambda fb, skip_attn_backend_init: ran.append("graph"))
        if graphs else None)
    batch = SimpleNamespace(forward_mode=ForwardMode.DECODE, return_logprob=asked)
    if asked:
        with pytest.raises(NotImplementedError, match="decode"):
            ModelRunner.forward(runner, batch)
    else:
        ModelRunner.forward(runner, batch)
    assert ran == ([] if asked else ["graph" if graphs else "eager"])
